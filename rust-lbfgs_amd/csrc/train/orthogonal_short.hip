// rust-lbfgs_amd/csrc/train/orthogonal_short.hip -- orthogonalised updates whose shorter side is 64 or less: in 64 bits, on the
// Gram matrix alone.
//
// With S = G G^T / |G|^2 and Q = I, repeat  P = a I + b S + c S S,  Q <- Q P,  S <- S P P;  the result is  Q G / |G|.
// |G|^2 is the trace of G G^T.  G is read twice, whatever the number of steps, and what happens in between is small enough for
// the LDS of one compute unit.  An error of S grows by up to a^2 in each step and by b in the last: 2^16 in five of the usual ones,
// which 64 bits have room for -- the only rounding that shows is that of the result -- and 32 bits do not.  (More than 7 of the
// usual steps would be too many even so: they go by products of the whole matrix, as larger updates do.)
//
// Such updates are bound by latency: products of whole matrices, one launch each, take 4 to 5 us apiece, three a step.  Here there
// are three launches in all: sums over slices of the long side, the steps, the result.  Measured, five steps, in us, with the
// launches' own time, against products of the whole matrix: 32 x 64 27 (70), 64 x 128 48 (77), 64 x 1000 53 (100; bf16 83),
// 64 x 4000 59 (179; bf16 107), 16 of 64 x 64 47 (75).  At 64 the steps alone take 30 us, 17 products of 64^3 at 1.1 to 1.3 us
// of the matrix units and half as much for reads of LDS, sums and barriers; at 32 10, at 16 5.  Sides beyond 64 would not fit the
// LDS, and 128 x 128 in one compute unit would take 8 times as long.  The slices take 3 us at 16 x 64, 6 at 64 x 64, 15 at 64 x 5000, the
// result 3, 9 and 10: both wait for memory and for each other's launches.
#include "orthogonal.h"

#include <algorithm>

namespace lt {

typedef double double4_ __attribute__((ext_vector_type(4)));

// v_mfma_f64_16x16x4: lane l has row (column) l % 16 of L (of R), K = l / 16; of the result column l % 16, rows l / 16 + 4 r
__device__ __forceinline__ double4_ mfma(double l, double r, double4_ c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(l, r, c, 0, 0, 0); }

// a symmetric matrix of 16 MB rows as blocks of 16 x 16, the lower triangle's in the order (0,0) (1,0) (1,1) (2,0) ...
template <int MB>
constexpr int blocks_of() {
    return MB * (MB + 1) / 2;
}
struct Block {
    int i, j;
};
__device__ __forceinline__ Block block_of(int t) {
    const int i = t >= 6 ? 3 : t >= 3 ? 2 : t >= 1 ? 1 : 0;
    return {i, t - i * (i + 1) / 2};
}

// 64 columns of G (from column j0) to registers, four adjacent elements at a time -- of a row of G or, tall, of G^T --, and from
// there to LDS; zeros where G has ended
template <int MB>
__device__ __forceinline__ void whose(int e, int tall, int* i, int* j) {
    const int k = threadIdx.x + e * 256;
    *i = tall ? k % (MB * 4) * 4 : k / 16, *j = tall ? k / (MB * 4) : k % 16 * 4;
}
template <class T, int MB>
__device__ __forceinline__ void fetch(const T* g, int m, int n, int tall, int64_t j0, float4_ (&v)[MB]) {
#pragma unroll
    for (int e = 0; e < MB; e++) {
        int i, j;
        whose<MB>(e, tall, &i, &j);
        v[e] = float4_{0, 0, 0, 0};
        if (i >= m || j0 + j >= n) continue;
        const T* x = g + (tall ? (j0 + j) * m + i : i * (int64_t)n + j0 + j);
        const int64_t left = tall ? m - i : n - j0 - j;
        if (left >= 4) {
            const Pack<T, 4> w = *(const Pack<T, 4>*)x;
            v[e] = float4_{(float)w.v[0], (float)w.v[1], (float)w.v[2], (float)w.v[3]};
        } else {
            v[e][0] = (float)x[0];
            if (left > 1) v[e][1] = (float)x[1];
            if (left > 2) v[e][2] = (float)x[2];
        }
    }
}
template <int MB, int LINE>
__device__ __forceinline__ void keep(float* tile, int tall, const float4_ (&v)[MB]) {
#pragma unroll
    for (int e = 0; e < MB; e++) {
        int i, j;
        whose<MB>(e, tall, &i, &j);
        if (!tall)
            *(float4_*)&tile[i * LINE + j] = v[e];
        else
#pragma unroll
            for (int k = 0; k < 4; k++) tile[(i + k) * LINE + j] = v[e][k];
    }
}

// part[matrix][slice] = the sum of g g^T over a slice's columns g of G.  A wave has a quarter of the columns and all blocks, so
// that what it reads from LDS, the same for rows and columns, feeds MB (MB + 1) / 2 products for MB reads.
template <class T, int MB>
__global__ __launch_bounds__(256) void short_gram_kernel(const T* g, int m, int n, int tall, double* part) {
    constexpr int LINE = 68, B = blocks_of<MB>();  // (4 rows on: 16 banks on)
    __shared__ __attribute__((aligned(16))) float tile[MB * 16 * LINE];
    __shared__ double4_ join[B * WAVE];
    const int slices = gridDim.x, lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int64_t chunks = (n + 63) / 64, from = chunks * blockIdx.x / slices, to = chunks * (blockIdx.x + 1) / slices;
    g += (int64_t)blockIdx.y * m * n;
    double4_ acc[B];
#pragma unroll
    for (int t = 0; t < B; t++) acc[t] = double4_{0, 0, 0, 0};
    float4_ v[MB];
    fetch<T, MB>(g, m, n, tall, from * 64, v);
    for (int64_t c = from; c < to; c++) {
        __syncthreads();
        keep<MB, LINE>(tile, tall, v);
        __syncthreads();
        if (c + 1 < to) fetch<T, MB>(g, m, n, tall, (c + 1) * 64, v);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            double x[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) x[i] = (double)tile[(i * 16 + lane % 16) * LINE + wave * 16 + k * 4 + lane / 16];
#pragma unroll
            for (int i = 0, t = 0; i < MB; i++)
#pragma unroll
                for (int j = 0; j <= i; j++, t++) acc[t] = mfma(x[i], x[j], acc[t]);
        }
    }
    for (int w = 0; w < 4; w++) {
        if (wave == w)
#pragma unroll
            for (int t = 0; t < B; t++) join[t * WAVE + lane] = w ? join[t * WAVE + lane] + acc[t] : acc[t];
        __syncthreads();
    }
    double4_* o = (double4_*)part + ((int64_t)blockIdx.y * slices + blockIdx.x) * B * WAVE;
    for (int k = threadIdx.x; k < B * WAVE; k += 256) o[k] = join[k];
}

// The steps, a workgroup to a matrix: S, P and Q in LDS, all of them symmetric, so that the lower triangle's blocks are all that
// is multiplied -- dealt to the waves in turn -- and rows may be read as columns.  q[matrix] = Q / |G|.
template <int MB>
__global__ __launch_bounds__(512) void short_steps_kernel(const double* part, int slices, int steps, double a, double b, double c, double* q) {
    constexpr int M = MB * 16, LINE = M + 2, B = blocks_of<MB>(), EACH = (B + 7) / 8, BOTH = (2 * B + 7) / 8;
    __shared__ double S[M * LINE], P[M * LINE], Q[M * LINE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    auto put = [&](double* to, Block at, double4_ v) {
        const int j = at.j * 16 + lane % 16;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = at.i * 16 + lane / 16 + 4 * r;
            to[i * LINE + j] = v[r];
            if (at.i != at.j) to[j * LINE + i] = v[r];
        }
    };
    auto get = [&](const double* from, Block at) {
        double4_ v;
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = from[(at.i * 16 + lane / 16 + 4 * r) * LINE + at.j * 16 + lane % 16];
        return v;
    };
    auto product = [&](const double* l, const double* r, Block at) {
        double4_ v = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < M / 4; k++) {
            const int row = (k * 4 + lane / 16) * LINE;
            v = mfma(l[row + at.i * 16 + lane % 16], r[row + at.j * 16 + lane % 16], v);
        }
        return v;
    };
    const double4_* from = (const double4_*)part + (int64_t)blockIdx.x * slices * B * WAVE;
    double4_ sum[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const int t = wave + e * 8;
        sum[e] = double4_{0, 0, 0, 0};
        if (t >= B) continue;
#pragma unroll 8
        for (int k = 0; k < slices; k++) sum[e] += from[((int64_t)k * B + t) * WAVE + lane];
        put(S, block_of(t), sum[e]);
    }
    __syncthreads();
    const double trace = wave_sum(lane < M ? S[lane * LINE + lane] : 0.0);
    const double f = trace > 0 && trace < INFINITY ? 1 / trace : trace == 0 ? 0.0 : NAN;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; e++)
        if (wave + e * 8 < B) put(S, block_of(wave + e * 8), sum[e] * f);
    __syncthreads();
    for (int step = 0; step < steps; step++) {
        const bool more = step + 1 < steps;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int t = wave + e * 8;
            if (t >= B) continue;
            const Block at = block_of(t);
            double4_ v = c * product(S, S, at) + b * get(S, at);
            if (at.i == at.j)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (lane / 16 + 4 * r == lane % 16) v[r] += a;
            put(P, at, v);
            if (!step) put(Q, at, v);
        }
        __syncthreads();
        // Q P and S P; both take the place of their left operands once all have read them
        double4_ w[BOTH];
#pragma unroll
        for (int e = 0; e < BOTH; e++) {
            const int t = wave + e * 8;
            if (t < B && more) w[e] = product(S, P, block_of(t));
            if (t >= B && t < 2 * B && step) w[e] = product(Q, P, block_of(t - B));
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < BOTH; e++) {
            const int t = wave + e * 8;
            if (t < B && more) put(S, block_of(t), w[e]);
            if (t >= B && t < 2 * B && step) put(Q, block_of(t - B), w[e]);
        }
        __syncthreads();
        if (!more) break;
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (wave + e * 8 < B) w[e] = product(S, P, block_of(wave + e * 8));
        __syncthreads();
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (wave + e * 8 < B) put(S, block_of(wave + e * 8), w[e]);
        __syncthreads();
    }
    const double scale = f == 0 ? 0.0 : sqrt(f);
    q += (int64_t)blockIdx.x * M * M;
    for (int k = threadIdx.x; k < M * M; k += 512) q[k] = Q[k / M * LINE + k % M] * scale;
}

// out = Q G, 64 columns to a workgroup, 16 to a wave; tall: out^T = G^T Q, so that adjacent lanes store adjacent elements in either case
template <class T, int MB>
__global__ __launch_bounds__(256) void short_apply_kernel(const T* g, int m, int n, int tall, const double* q, T* out) {
    constexpr int M = MB * 16, LINE = 80, Q_LINE = M + 2;  // (a row on: 16 banks on)
    __shared__ double Q[M * Q_LINE];
    __shared__ __attribute__((aligned(16))) float tile[M * LINE];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int64_t j0 = (int64_t)blockIdx.x * 64, at = (int64_t)blockIdx.y * m * n;
    float4_ v[MB];
    fetch<T, MB>(g + at, m, n, tall, j0, v);
    q += (int64_t)blockIdx.y * M * M;
#pragma unroll
    for (int k = 0; k < M * M / 256; k++) Q[(k * 256 + threadIdx.x) / M * Q_LINE + (k * 256 + threadIdx.x) % M] = q[k * 256 + threadIdx.x];
    keep<MB, LINE>(tile, tall, v);
    __syncthreads();
    out += at;
    double4_ acc[MB];
#pragma unroll
    for (int i = 0; i < MB; i++) acc[i] = double4_{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < MB * 4; k++) {
        const int row = k * 4 + lane / 16;
        const double x = (double)tile[row * LINE + wave * 16 + lane % 16];
#pragma unroll
        for (int i = 0; i < MB; i++) {
            const double y = Q[row * Q_LINE + i * 16 + lane % 16];
            acc[i] = tall ? mfma(x, y, acc[i]) : mfma(y, x, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int down = lane / 16 + 4 * r, across = lane % 16;
            const int row = i * 16 + (tall ? across : down);
            const int64_t col = j0 + wave * 16 + (tall ? down : across);
            if (row < m && col < n) out[tall ? col * m + row : row * (int64_t)n + col] = (T)acc[i][r];
        }
}

// Slices: a chunk of 64 columns takes some 1.5 us of a workgroup, adding up a slice 0.2 us; and no more than the device has use for.
// Measured, the three kernels at 64 x n, in us, with 8, 32 and 79 slices and with the rule's: n = 1000 51, 50, 50, 52; 5000 72, 59, 67, 60;
// 100000 747, 252, 165, 155.
static int slices_of(int64_t batch, int n) {
    const double chunks = (n + 63) / 64;
    return (int)std::max(1.0, std::min({chunks, std::sqrt(7.5 * chunks), 256.0, std::ceil(1024.0 / batch)}));
}
static int side_of(int m) { return (m + 15) / 16 * 16; }

uint64_t short_workspace(int64_t batch, int m, int n) {
    const uint64_t side = side_of(m), blocks = side / 16 * (side / 16 + 1) / 2;
    return (uint64_t)batch * sizeof(double) * (slices_of(batch, n) * blocks * 256 + side * side);
}

template <class T, int MB>
static void launch(const Short& p, hipStream_t s) {
    const int slices = slices_of(p.batch, p.n);
    double* part = (double*)p.workspace;
    double* q = part + (int64_t)p.batch * slices * blocks_of<MB>() * 256;
    short_gram_kernel<T, MB><<<dim3(slices, p.batch), 256, 0, s>>>((const T*)p.update, p.m, p.n, p.tall, part);
    short_steps_kernel<MB><<<p.batch, 512, 0, s>>>(part, slices, p.steps, p.a, p.b, p.c, q);
    short_apply_kernel<T, MB><<<dim3((p.n + 63) / 64, p.batch), 256, 0, s>>>((const T*)p.update, p.m, p.n, p.tall, q, (T*)p.out);
}
template <class T>
void short_orthogonalize(const Short& p, hipStream_t s) {
    if (p.m <= 16)
        launch<T, 1>(p, s);
    else if (p.m <= 32)
        launch<T, 2>(p, s);
    else if (p.m <= 48)
        launch<T, 3>(p, s);
    else
        launch<T, 4>(p, s);
}
template void short_orthogonalize<float>(const Short&, hipStream_t);
template void short_orthogonalize<bf16>(const Short&, hipStream_t);
template void short_orthogonalize<f16>(const Short&, hipStream_t);

}  // namespace lt
