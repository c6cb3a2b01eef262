// rust-lbfgs_amd/csrc/train/orthogonal_panel.hip -- orthogonalised updates whose shorter side is 65 to 128 and whose longer one is
// not much more: one launch a step.
//
//   S = sum over panels of X_w X_w^T,   P = a I + b S + c S S,   X_w <- P X_w,   the panel's share of the next S
//
// A workgroup has a panel X_w of 64 or 128 columns for good.  All that the workgroups of a matrix need of each other are their shares of S, so
// that a step is one launch where products of whole matrices take three of 5 us each; the price is that every workgroup adds up the
// shares and makes P for itself.  Products as in orthogonal.hip: three of f16 for 22 bits, the small ones summed apart.
#include "orthogonal.h"

namespace lt {

// Blocks of 16 x 16 of a symmetric matrix of MB block rows (MB even), dealt to MB waves: wave w has (w, w + d mod MB), d = 0 .. MB/2 -- the
// last for the first half of the waves --, which are all of one triangle or the other, with the same left operand.
template <int MB>
constexpr int slots_of() {
    return MB * (MB + 1) / 2;
}
template <int MB>
__device__ __forceinline__ bool has(int wave, int d) {
    return d < MB / 2 || wave < MB / 2;
}

// hi and lo of a matrix in LDS, K adjacent, 16 bytes between the rows' ends and the next: 16 rows' chunks lie in different banks
template <int K>
struct Operand {
    static constexpr int LINE = K + 8;
    f16 *hi, *lo;
    __device__ __forceinline__ half8 get(const f16* p, int row, int k) const {  // a fragment: 16 rows, 32 of K
        const int lane = threadIdx.x % WAVE;
        return *(const half8*)&p[(row + lane % 16) * LINE + k * 32 + lane / 16 * 8];
    }
    __device__ __forceinline__ void put(int row, int k, float v) {
        const Halves h = split(v);
        hi[row * LINE + k] = h.hi, lo[row * LINE + k] = h.lo;
    }
    __device__ __forceinline__ void put4(int row, int k, const float4_& v) {  // four of K
        half4 a, b;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const Halves h = split(v[e]);
            a[e] = h.hi, b[e] = h.lo;
        }
        *(half4*)&hi[row * LINE + k] = a, *(half4*)&lo[row * LINE + k] = b;
    }
};
// L R^T, 16 rows of L (its fragments are in registers) and 16 of R
template <int K>
struct Left {
    half8 hi[K / 32], lo[K / 32];
    __device__ __forceinline__ void get(const Operand<K>& x, int row) {
#pragma unroll
        for (int k = 0; k < K / 32; k++) hi[k] = x.get(x.hi, row, k), lo[k] = x.get(x.lo, row, k);
    }
    __device__ __forceinline__ float4_ times(const Operand<K>& x, int row) const {
        float4_ acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < K / 32; k++) {
            const half8 h = x.get(x.hi, row, k), l = x.get(x.lo, row, k);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[k], h, acc, 0, 0, 0);
            low = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[k], l, low, 0, 0, 0);
            low = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[k], h, low, 0, 0, 0);
        }
        return acc + low;
    }
};

// a panel's share of S: X X^T over its columns, as the waves hold it
template <int MB, int COLS>
__device__ __forceinline__ void share(const Operand<COLS>& x, float4_* o) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    Left<COLS> l;
    l.get(x, wave * 16);
#pragma unroll
    for (int d = 0; d <= MB / 2; d++)
        if (has<MB>(wave, d)) o[(d * MB + wave) * WAVE + lane] = l.times(x, (wave + d) % MB * 16);
}
// block (wave, wave + d) into both halves of a symmetric matrix; on the diagonal what is below it
template <int MB>
__device__ __forceinline__ void put_block(Operand<MB * 16>& s, int d, const float4_& v) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const int i = wave * 16 + lane / 16 * 4, j = (wave + d) % MB * 16 + lane % 16;
    if (d) {
        s.put4(j, i, v);
#pragma unroll
        for (int e = 0; e < 4; e++) s.put(i + e, j, v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (i + e >= j) {
                s.put(i + e, j, v[e]);
                s.put(j, i + e, v[e]);
            }
    }
}

// G / |G| -> X^T of the panel (columns adjacent to K of P X), and its share of S
template <class T, int MB, int COLS>
__global__ __launch_bounds__(MB * WAVE) void panel_first_kernel(const T* g, int m, int n, int tall, const double* norms, int parts, double scale, f16* xt, float* shares) {
    constexpr int M = MB * 16, THREADS = MB * WAVE;
    __shared__ __attribute__((aligned(16))) f16 x_pool[2 * M * Operand<COLS>::LINE], t_pool[2 * COLS * Operand<M>::LINE];
    __shared__ double sums[MB];
    const int64_t b = blockIdx.y, w = b * gridDim.x + blockIdx.x;
    double norm = 0;
    for (int k = threadIdx.x; k < parts; k += THREADS) norm += norms[b * NORM_BLOCKS + k];
    norm = wave_sum(norm);
    if (threadIdx.x % WAVE == 0) sums[threadIdx.x / WAVE] = norm;
    Operand<COLS> x = {x_pool, x_pool + M * Operand<COLS>::LINE};
    Operand<M> t = {t_pool, t_pool + COLS * Operand<M>::LINE};
    g += b * (int64_t)m * n;
    xt += w * 2 * COLS * M;
    const int j0 = blockIdx.x * COLS;
    constexpr int EACH = M * COLS / THREADS;
    float v[EACH];
#pragma unroll
    for (int k = 0; k < EACH; k++) {  // (adjacent threads read adjacent elements of G in either case)
        const int at = k * THREADS + threadIdx.x, i = tall ? at % M : at / COLS, j = tall ? at / M : at % COLS;
        v[k] = i < m && j0 + j < n ? (float)g[tall ? (int64_t)(j0 + j) * m + i : (int64_t)i * n + j0 + j] : 0.0f;
    }
    __syncthreads();
    norm = 0;
    for (int k = 0; k < MB; k++) norm += sums[k];
    norm = sqrt(norm);
    const double f = norm > 0 && norm < INFINITY ? scale / norm : norm == 0 ? 0.0 : NAN;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        const int at = k * THREADS + threadIdx.x, i = tall ? at % M : at / COLS, j = tall ? at / M : at % COLS;
        const Halves h = split((float)((double)v[k] * f));
        x.hi[i * Operand<COLS>::LINE + j] = t.hi[j * Operand<M>::LINE + i] = h.hi;
        x.lo[i * Operand<COLS>::LINE + j] = t.lo[j * Operand<M>::LINE + i] = h.lo;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH / 4; k++) {
        const int at = (k * THREADS + threadIdx.x) * 8, part = at / (COLS * M), j = at % (COLS * M) / M, i = at % M;
        *(half8*)&xt[at] = *(const half8*)&(part ? t.lo : t.hi)[j * Operand<M>::LINE + i];
    }
    share<MB, COLS>(x, (float4_*)shares + w * slots_of<MB>() * WAVE);
}

// One step of a panel.  shares: of S, by all panels of the matrix; next: of the next S.  The last step leaves out = X instead.
template <class T, int MB, int COLS, bool LAST>
__global__ __launch_bounds__(MB * WAVE) void panel_step_kernel(const float* shares, f16* xt, float* next, T* out, int m, int n, int tall, float a, float b, float c,
                                                               float s_scale, float x_scale) {
    constexpr int M = MB * 16, THREADS = MB * WAVE, EACH = MB / 2 + 1;
    constexpr int OLD = COLS * Operand<M>::LINE, NEW = M * Operand<COLS>::LINE;
    constexpr bool SHARED = COLS > 64;  // (the new X in the place of the old one's transpose: LDS has no room for both)
    __shared__ __attribute__((aligned(16))) f16 s_pool[2 * M * Operand<M>::LINE], x_pool[SHARED ? 2 * (OLD > NEW ? OLD : NEW) : 2 * (OLD + NEW)];
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE, panels = gridDim.x;
    const int64_t matrix = blockIdx.y, w = matrix * panels + blockIdx.x;
    Operand<M> s = {s_pool, s_pool + M * Operand<M>::LINE}, t = {x_pool, x_pool + OLD};
    Operand<COLS> x = {x_pool + (SHARED ? 0 : 2 * OLD), x_pool + (SHARED ? 0 : 2 * OLD) + NEW};
    xt += w * 2 * COLS * M;
    // the panel, on its way while S is added up
    constexpr int PACKS = 2 * COLS * M / 8 / THREADS;
    half8 mine[PACKS];
#pragma unroll
    for (int k = 0; k < PACKS; k++) mine[k] = ((const half8*)xt)[k * THREADS + threadIdx.x];
    const float4_* from = (const float4_*)shares + matrix * panels * slots_of<MB>() * WAVE;
    float4_ sum[EACH];
#pragma unroll
    for (int d = 0; d < EACH; d++) sum[d] = float4_{0, 0, 0, 0};
#pragma unroll 4
    for (int p = 0; p < panels; p++)
#pragma unroll
        for (int d = 0; d < EACH; d++)
            if (has<MB>(wave, d)) sum[d] += from[((int64_t)p * slots_of<MB>() + d * MB + wave) * WAVE + lane];
#pragma unroll
    for (int d = 0; d < EACH; d++)
        if (has<MB>(wave, d)) put_block<MB>(s, d, sum[d] * s_scale);
#pragma unroll
    for (int k = 0; k < PACKS; k++) {
        const int at = (k * THREADS + threadIdx.x) * 8, part = at / (COLS * M), j = at % (COLS * M) / M, i = at % M;
        *(half8*)&(part ? t.lo : t.hi)[j * Operand<M>::LINE + i] = mine[k];
    }
    __syncthreads();
    Left<M> l;
    l.get(s, wave * 16);
#pragma unroll
    for (int d = 0; d < EACH; d++) {
        if (!has<MB>(wave, d)) continue;
        sum[d] = c * l.times(s, (wave + d) % MB * 16) + b * (sum[d] * s_scale);
        const int i = wave * 16 + lane / 16 * 4, j = (wave + d) % MB * 16 + lane % 16;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (i + e == j && j < m) sum[d][e] += a;
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < EACH; d++)
        if (has<MB>(wave, d)) put_block<MB>(s, d, sum[d]);
    __syncthreads();
    l.get(s, wave * 16);
    const int i = wave * 16 + lane / 16 * 4, j0 = blockIdx.x * COLS;
    float4_ v[COLS / 16];
#pragma unroll
    for (int q = 0; q < COLS / 16; q++) v[q] = l.times(t, q * 16) * x_scale;
    if (LAST) {
        T* o = out + matrix * m * n;
#pragma unroll
        for (int q = 0; q < COLS / 16; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = i + e, col = j0 + q * 16 + lane % 16;
                if (row < m && col < n) o[tall ? (int64_t)col * m + row : (int64_t)row * n + col] = (T)v[q][e];
            }
        return;
    }
    if (SHARED) __syncthreads();
#pragma unroll
    for (int q = 0; q < COLS / 16; q++) {
        const int j = q * 16 + lane % 16;
        half4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const Halves h = split(v[q][e]);
            hi[e] = h.hi, lo[e] = h.lo;
            x.hi[(i + e) * Operand<COLS>::LINE + j] = h.hi, x.lo[(i + e) * Operand<COLS>::LINE + j] = h.lo;
        }
        *(half4*)&xt[j * M + i] = hi, *(half4*)&xt[COLS * M + j * M + i] = lo;
    }
    __syncthreads();
    share<MB, COLS>(x, (float4_*)next + w * slots_of<MB>() * WAVE);
}

static int side_of(int m) { return m <= 96 ? 96 : 128; }

// Columns of a panel: few, so that more workgroups share the work, while there are not too many shares of S to add up.  In us at 128 x n,
// five steps, 64 and 128 columns: n = 256 66, 79; 512 88, 89; 1000 122, 109; 30 of 100 x 500 124, 108.
static int cols_of(int64_t batch, int n) { return n <= 512 && batch * ((n + 63) / 64) <= 128 ? 64 : 128; }
static int64_t panels_of(int64_t batch, int n) { return (n + cols_of(batch, n) - 1) / cols_of(batch, n); }

// Measured against products of the whole matrix (in brackets; those of 16-bit updates are fewer), in us, five steps, f32: 80 x 80 44 (87),
// 128 x 256 67 (93), 128 x 1000 108 (115), 128 x 2000 142 (150), 128 x 4000 208 (253), 16 of 128 x 1000 131 (159); bf16: 80 x 80 44 (94), 128 x 256
// 67 (96), 128 x 512 88 (98), 128 x 1000 109 (102), 90 x 500 69 (97), 90 x 2000 112 (111).
bool panel_fits(int dtype, int64_t batch, int m, int n) {
    return m > SHORT && m <= 128 && n <= (dtype == LBFGS_TRAIN_F32 ? 4096 : m <= 96 ? 1536 : 768) && panels_of(batch, n) * batch <= 256;
}
uint64_t panel_workspace(int64_t batch, int m, int n) {
    const uint64_t side = side_of(m), panels = (uint64_t)batch * panels_of(batch, n), blocks = side / 16 * (side / 16 + 1) / 2;
    return (uint64_t)batch * NORM_BLOCKS * sizeof(double) + panels * (2 * blocks * 256 * sizeof(float) + 2 * cols_of(batch, n) * side * sizeof(f16));
}

template <class T, int MB, int COLS>
static void launch(const Panel& p, hipStream_t s) {
    const int panels = (int)panels_of(p.batch, p.n);
    const int64_t all = (int64_t)p.batch * panels, each = all * slots_of<MB>() * 256;
    double* norms = (double*)p.workspace;
    float* shares[2] = {(float*)(norms + (int64_t)p.batch * NORM_BLOCKS), nullptr};
    shares[1] = shares[0] + each;
    f16* xt = (f16*)(shares[1] + each);
    const dim3 grid(panels, p.batch);
    panel_first_kernel<T, MB, COLS><<<grid, MB * WAVE, 0, s>>>((const T*)p.update, p.m, p.n, p.tall, norms, p.norms, p.sx, xt, shares[0]);
    const float a = (float)(p.a * p.sp), b = (float)(p.b * p.sp / p.ss), c = (float)(p.c * p.sp / (p.ss * p.ss)), s_scale = (float)(p.ss / (p.sx * p.sx));
    for (int k = 0; k < p.steps; k++)
        if (k + 1 < p.steps)
            panel_step_kernel<T, MB, COLS, false><<<grid, MB * WAVE, 0, s>>>(shares[k & 1], xt, shares[~k & 1], nullptr, p.m, p.n, p.tall, a, b, c, s_scale, (float)(1 / p.sp));
        else
            panel_step_kernel<T, MB, COLS, true><<<grid, MB * WAVE, 0, s>>>(shares[k & 1], xt, nullptr, (T*)p.out, p.m, p.n, p.tall, a, b, c, s_scale, (float)(1 / (p.sp * p.sx)));
}
template <class T>
void panel_orthogonalize(const Panel& p, hipStream_t s) {
    const bool wide = cols_of(p.batch, p.n) == 128;
    if (side_of(p.m) == 96)
        wide ? launch<T, 6, 128>(p, s) : launch<T, 6, 64>(p, s);
    else
        wide ? launch<T, 8, 128>(p, s) : launch<T, 8, 64>(p, s);
}
template void panel_orthogonalize<float>(const Panel&, hipStream_t);
template void panel_orthogonalize<bf16>(const Panel&, hipStream_t);
template void panel_orthogonalize<f16>(const Panel&, hipStream_t);

}  // namespace lt
