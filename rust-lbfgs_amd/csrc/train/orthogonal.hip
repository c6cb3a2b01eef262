// rust-lbfgs_amd/csrc/train/orthogonal.hip -- a matrix update brought near its polar factor by products.
//
//   X <- G / |G|_F          repeat:  S = X X^T,  P = a I + b S + c S S,  X <- P X
//
// maps every singular value s of X to a s + b s^3 + c s^5 and leaves the singular vectors alone.  All of the work is matrix
// products, so all of it is on the matrix cores, in f16 with 32-bit accumulation.  What 11 bits of significand would lose is
// kept by splitting: a value v is held as  hi + lo, hi = f16(v), lo = f16(v - hi)  -- 22 bits --, and a product of two such is
// hi hi + hi lo + lo hi, three matrix instructions instead of one (lo lo is below the accumulator's own rounding).  That is as
// good as a product of 32-bit values (measured against 64 bits) at the rate of 16-bit ones over three.  A power of two puts the
// largest value that can occur near the top of f16's range, so that lo stays a normal number.
// Only the last steps of a bf16 update use hi alone: what is rounded away early is multiplied by up to `a` in every step that
// follows, and a gradient's small singular values would end as noise.
#include "common.h"

#include <algorithm>

namespace lt {

typedef f16 half8 __attribute__((ext_vector_type(8)));
typedef f16 half4 __attribute__((ext_vector_type(4)));
typedef float float4_ __attribute__((ext_vector_type(4)));

constexpr int TILE = 128, BK = 32, PAD = 8;  // (PAD: halves between the rows of a tile in LDS)
constexpr int NORM_BLOCKS = 64;

struct Split {  // hi and lo parts, dense, padded with zeros to multiples of TILE
    f16 *hi, *lo;
};

// ------------------------------------------------------------------------------------ norm, normalise, split
template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* g, int64_t n, double* part) {
    constexpr int N = vec_len<T>();
    const T* x = g + (int64_t)blockIdx.y * n;
    double s = 0;
    const int64_t packs = n / N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += (int64_t)gridDim.x * 256) {
        const Pack<T, N> p = ((const Pack<T, N>*)x)[i];
#pragma unroll
        for (int k = 0; k < N; k++) s += (double)p.v[k] * (double)p.v[k];
    }
    if (blockIdx.x == 0)
        for (int64_t i = packs * N + threadIdx.x; i < n; i += 256) s += (double)x[i] * (double)x[i];
    __shared__ double w[4];
    s = wave_sum(s);
    if (threadIdx.x % WAVE == 0) w[threadIdx.x / WAVE] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = w[0] + w[1] + w[2] + w[3];
}

__device__ __forceinline__ void split(float v, f16& hi, f16& lo) {
    hi = (f16)v;
    lo = (f16)(v - (float)hi);
}

// X (m x n, K = n adjacent) and its transpose, scaled and split, from G or, tall, from G^T
template <class T>
__global__ __launch_bounds__(256) void split_kernel(const T* g, int m, int n, int mp, int np, int tall, const double* part, int parts, float scale, Split x, Split xt) {
    __shared__ float tile[64][65];
    const int64_t b = blockIdx.z;
    double norm = wave_sum(threadIdx.x % WAVE < parts ? part[b * NORM_BLOCKS + threadIdx.x % WAVE] : 0.0);
    norm = sqrt(norm);
    const double f = norm > 0 ? (double)scale / norm : norm == 0 ? 0.0 : NAN;
    const int i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    g += b * (int64_t)m * n;
    const int64_t at = b * (int64_t)mp * np;
    for (int k = threadIdx.x; k < 64 * 64; k += 256) {  // (adjacent threads read adjacent elements of G in either case)
        const int r = k / 64, c = k % 64;
        const int i = tall ? c : r, j = tall ? r : c;
        float v = 0;
        if (i0 + i < m && j0 + j < n) v = (float)((double)(float)g[tall ? (int64_t)(j0 + j) * m + i0 + i : (int64_t)(i0 + i) * n + j0 + j] * f);
        tile[i][j] = v;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 64 * 64; k += 256) {
        const int r = k / 64, c = k % 64;
        f16 hi, lo;
        split(tile[r][c], hi, lo);
        const int64_t o = at + (int64_t)(i0 + r) * np + j0 + c;
        x.hi[o] = hi, x.lo[o] = lo;
        split(tile[c][r], hi, lo);
        const int64_t t = at + (int64_t)(j0 + r) * mp + i0 + c;
        xt.hi[t] = hi, xt.lo[t] = lo;
    }
}

// ------------------------------------------------------------------------------------ products
enum { GRAM, POLY, STEP, LAST };

struct Product {
    Split l, r;          // C = L R^T, both with K adjacent
    int64_t l_batch, r_batch, o_batch;
    int k, ld;           // K (a multiple of BK), the row length of both
    float scale;         // of the accumulated product
    // GRAM, POLY: C is symmetric, m x m; POLY: scale * C + b * L + a on the diagonal (L itself is S)
    float a, b;
    int m, n;            // real rows and columns of C
    int o_ld, t_ld;      // row lengths of o and its transpose t
    Split o, t;
    void* out;           // LAST: the result, in the caller's type and orientation
    int tall;
};

template <class T, int WHAT, int PARTS>
__global__ __launch_bounds__(256) void product_kernel(Product p) {
    constexpr bool SYM = WHAT == GRAM || WHAT == POLY;
    constexpr int LD = BK + PAD, SPLITS = PARTS == 3 ? 2 : 1;
    __shared__ f16 lds[2 * SPLITS][TILE * LD];
    int ti = blockIdx.y, tj = blockIdx.x;
    if (SYM && tj > ti) return;  // the mirror image writes it
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int wi = (wave / 2) * 64, wj = (wave % 2) * 64;
    const int64_t b = blockIdx.z;
    const f16* src[2 * SPLITS];
    src[0] = p.l.hi + b * p.l_batch + (int64_t)ti * TILE * p.ld;
    src[1] = p.r.hi + b * p.r_batch + (int64_t)tj * TILE * p.ld;
    if (SPLITS == 2) {
        src[2] = p.l.lo + b * p.l_batch + (int64_t)ti * TILE * p.ld;
        src[3] = p.r.lo + b * p.r_batch + (int64_t)tj * TILE * p.ld;
    }
    float4_ acc[4][4];
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) acc[x][y] = float4_{0, 0, 0, 0};
    const int row = tid / 4, col = (tid % 4) * 8;  // 64 rows of 32 halves at a time
    for (int k0 = 0; k0 < p.k; k0 += BK) {
        half8 in[2 * SPLITS][2];
#pragma unroll
        for (int s = 0; s < 2 * SPLITS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) in[s][h] = *(const half8*)(src[s] + (int64_t)(row + h * 64) * p.ld + k0 + col);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2 * SPLITS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) *(half8*)&lds[s][(row + h * 64) * LD + col] = in[s][h];
        __syncthreads();
        half8 l[SPLITS][4], r[SPLITS][4];
#pragma unroll
        for (int s = 0; s < SPLITS; s++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                l[s][x] = *(const half8*)&lds[2 * s][(wi + x * 16 + lane % 16) * LD + (lane / 16) * 8];
                r[s][x] = *(const half8*)&lds[2 * s + 1][(wj + x * 16 + lane % 16) * LD + (lane / 16) * 8];
            }
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0][x], r[0][y], acc[x][y], 0, 0, 0);
                if (PARTS == 3) {
                    acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[0][x], r[SPLITS - 1][y], acc[x][y], 0, 0, 0);
                    acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[SPLITS - 1][x], r[0][y], acc[x][y], 0, 0, 0);
                }
            }
    }
    // a lane holds rows i .. i+3 of column j of each 16 x 16 block
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const int i = ti * TILE + wi + x * 16 + (lane / 16) * 4, j = tj * TILE + wj + y * 16 + lane % 16;
            half4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float v = acc[x][y][e] * p.scale;
                if (WHAT == POLY) {
                    const int64_t at = b * p.l_batch + (int64_t)j * p.ld + i + e;  // (S is symmetric)
                    v += p.b * ((float)p.l.hi[at] + (float)p.l.lo[at]);
                    if (i + e == j && j < p.m) v += p.a;
                }
                if (WHAT == LAST) {
                    if (i + e < p.m && j < p.n) ((T*)p.out)[b * (int64_t)p.m * p.n + (p.tall ? (int64_t)j * p.m + i + e : (int64_t)(i + e) * p.n + j)] = (T)v;
                } else {
                    f16 h, l;
                    split(v, h, l);
                    hi[e] = h, lo[e] = l;
                    const int64_t o = b * p.o_batch + (int64_t)(i + e) * p.o_ld + j;
                    p.o.hi[o] = h, p.o.lo[o] = l;
                }
            }
            if (WHAT != LAST && !(SYM && ti == tj)) {
                const int64_t t = b * p.o_batch + (int64_t)j * p.t_ld + i;
                *(half4*)(p.t.hi + t) = hi, *(half4*)(p.t.lo + t) = lo;
            }
        }
}

// ------------------------------------------------------------------------------------ launches
static int64_t up(int64_t n) { return (n + TILE - 1) / TILE * TILE; }

struct Plan {
    int m, n, mp, np, batch, steps;
    float sx, ss, sp;    // what X, S and P are multiplied by
    double a, b, c;
};
struct Buffers {
    Split x[2], xt[2], s, p;
    double* part;
};

static uint64_t lay_out(Buffers* out, void* base, int64_t batch, int64_t rows, int64_t cols) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        void* p = (char*)base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const uint64_t m = (uint64_t)up(std::min(rows, cols)), n = (uint64_t)up(std::max(rows, cols)), bt = (uint64_t)batch;
    Buffers f;
    for (int k = 0; k < 2; k++) {
        f.x[k] = {(f16*)take(2 * bt * m * n), (f16*)take(2 * bt * m * n)};
        f.xt[k] = {(f16*)take(2 * bt * m * n), (f16*)take(2 * bt * m * n)};
    }
    f.s = {(f16*)take(2 * bt * m * m), (f16*)take(2 * bt * m * m)};
    f.p = {(f16*)take(2 * bt * m * m), (f16*)take(2 * bt * m * m)};
    f.part = (double*)take(bt * NORM_BLOCKS * sizeof(double));
    if (out) *out = f;
    return at;
}

// The largest value of X, S and P that singular values in [0, 1] can lead to, and from them the powers of two that keep f16
// in range.  false: the polynomial leaves it.
static bool ranges(Plan* q) {
    double x_most = 1.0, p_most = 0.0;
    for (int k = 0; k <= 1000; k++) {
        double s = k / 1000.0;
        for (int j = 0; j < q->steps; j++) {
            const double l = s * s, p = q->a + q->b * l + q->c * l * l;
            p_most = std::max(p_most, std::fabs(p));
            s *= p;
            if (!(std::fabs(s) < 64 && p_most < 1024)) return false;
            x_most = std::max(x_most, std::fabs(s));
        }
    }
    auto scale = [](double most) { return (float)std::exp2(std::floor(std::log2(48000.0 / most))); };
    q->sx = scale(x_most * 1.01);
    q->ss = scale(x_most * x_most * 1.02);
    q->sp = scale(std::max(p_most, 1.0) * 1.01);
    return true;
}

template <class T, int WHAT>
static void launch_product(const Product& p, int parts, dim3 grid, hipStream_t s) {
    if (parts == 1)
        product_kernel<T, WHAT, 1><<<grid, 256, 0, s>>>(p);
    else
        product_kernel<T, WHAT, 3><<<grid, 256, 0, s>>>(p);
}

template <class T>
static void launch_orthogonalize(const Plan& q, const void* g, void* out, const Buffers& f, int tall, hipStream_t s) {
    const int64_t size = (int64_t)q.m * q.n, X = (int64_t)q.mp * q.np, S = (int64_t)q.mp * q.mp;
    const int blocks = (int)std::min<int64_t>(NORM_BLOCKS, (size + 4095) / 4096);
    norm_kernel<T><<<dim3(blocks, q.batch), 256, 0, s>>>((const T*)g, size, f.part);
    split_kernel<T><<<dim3(q.np / 64, q.mp / 64, q.batch), 256, 0, s>>>((const T*)g, q.m, q.n, q.mp, q.np, tall, f.part, blocks, q.sx, f.x[0], f.xt[0]);
    const dim3 square(q.mp / TILE, q.mp / TILE, q.batch), wide(q.np / TILE, q.mp / TILE, q.batch);
    for (int k = 0; k < q.steps; k++) {
        const int at = k & 1, parts = sizeof(T) == 2 && std::is_same<T, bf16>::value && std::pow(std::fabs(q.a), q.steps - k) <= 12 ? 1 : 3;
        Product p = {};
        p.m = q.m, p.n = q.n, p.tall = tall;
        p.l = p.r = f.x[at], p.l_batch = p.r_batch = X, p.o_batch = S, p.k = p.ld = q.np;
        p.scale = q.ss / (q.sx * q.sx), p.o = p.t = f.s, p.o_ld = p.t_ld = q.mp;
        launch_product<T, GRAM>(p, parts, square, s);
        p.l = p.r = f.s, p.l_batch = p.r_batch = S, p.k = p.ld = q.mp;
        p.scale = (float)(q.c * q.sp / ((double)q.ss * q.ss)), p.b = (float)(q.b * q.sp / q.ss), p.a = (float)(q.a * q.sp), p.o = p.t = f.p;
        launch_product<T, POLY>(p, parts, square, s);
        p.l = f.p, p.r = f.xt[at], p.r_batch = p.o_batch = X;
        p.o = f.x[at ^ 1], p.t = f.xt[at ^ 1], p.o_ld = q.np, p.t_ld = q.mp;
        p.scale = k + 1 < q.steps ? 1 / q.sp : (float)(1 / ((double)q.sp * q.sx));
        if (k + 1 < q.steps) {
            launch_product<T, STEP>(p, parts, wide, s);
        } else {
            p.out = out;
            launch_product<T, LAST>(p, parts, wide, s);
        }
    }
}

}  // namespace lt

using namespace lt;

extern "C" uint64_t lbfgs_train_orthogonalize_workspace(int64_t batch, int64_t rows, int64_t cols) {
    if (batch < 1 || rows < 1 || cols < 1 || batch > 65535 || rows > (1 << 20) || cols > (1 << 20)) return 0;
    return lay_out(nullptr, nullptr, batch, rows, cols);
}

extern "C" int lbfgs_train_orthogonalize(int32_t dtype, int64_t batch, int64_t rows, int64_t cols, const void* update, void* out, int32_t steps, double a, double b,
                                         double c, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* who = "lbfgs_train_orthogonalize";
    if (dtype < LBFGS_TRAIN_F32 || dtype > LBFGS_TRAIN_F16)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: element type %d: float32, bfloat16 and float16 are offered", who, dtype);
    if (batch < 0 || rows < 0 || cols < 0 || batch > 65535 || rows > (1 << 20) || cols > (1 << 20))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld matrices of %lld x %lld", who, (long long)batch, (long long)rows, (long long)cols);
    if (steps < 1 || steps > 64) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %d steps: 1 to 64 are offered", who, steps);
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: coefficients %g, %g, %g", who, a, b, c);
    Plan q = {(int)std::min(rows, cols), (int)std::max(rows, cols), 0, 0, (int)batch, steps, 0, 0, 0, a, b, c};
    if (!ranges(&q)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %d steps of %g, %g, %g lead singular values out of range", who, steps, a, b, c);
    if (!batch || !rows || !cols) return LBFGS_HIP_OK;
    if (!update || !out) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: update and out are needed", who);
    q.mp = (int)up(q.m), q.np = (int)up(q.n);
    const uint64_t need = lay_out(nullptr, nullptr, batch, rows, cols);
    if (!workspace || workspace_bytes < need)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    Buffers f;
    lay_out(&f, workspace, batch, rows, cols);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case LBFGS_TRAIN_F32: launch_orthogonalize<float>(q, update, out, f, rows > cols, s); break;
        case LBFGS_TRAIN_BF16: launch_orthogonalize<bf16>(q, update, out, f, rows > cols, s); break;
        default: launch_orthogonalize<f16>(q, update, out, f, rows > cols, s);
    }
    return lt_launched(who);
}
