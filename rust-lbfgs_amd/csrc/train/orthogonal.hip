// rust-lbfgs_amd/csrc/train/orthogonal.hip -- a matrix update brought near its polar factor by products.
//
//   X <- G / |G|_F          repeat:  S = X X^T,  P = a I + b S + c S S,  X <- P X
//
// maps every singular value s of X to a s + b s^3 + c s^5 and leaves the singular vectors alone.  All of the work is matrix
// products, so all of it is on the matrix cores, in f16 with 32-bit accumulation.  What 11 bits of significand would lose is
// kept by splitting: a value v is held as  hi + lo, hi = f16(v), lo = f16(v - hi)  -- 22 bits --, and a product of two such is
// hi hi + hi lo + lo hi, three matrix instructions instead of one (lo lo is below the accumulator's own rounding).  That is as
// good as a product of 32-bit values (measured against 64 bits) at the rate of 16-bit ones over three.  Powers of two put the
// largest value that can occur near the top of f16's range, so that lo stays a normal number.  11 bits alone will not do, not
// even for 16-bit updates: what is rounded away early is multiplied by up to `a` in every step that follows, and the small
// singular values of a gradient would end as noise (4 % of the result for one of rank 8).
//
// Updates of 32 bits go through the steps as written.  Those of 16 bits are exact in hi alone at first (they are scaled by a
// power of two, the rest of 1/|G| is carried along as a number), and their last few steps work on the Gram matrix: with
// S = X X^T of the X that they begin with,
//   P = a I + b S + c S S,   Q <- Q P,   S <- S P P          and in the end   X <- Q X,
// all symmetric and all of the short side, which for a matrix m x 4 m is a third less work.  The price: an error of S is
// multiplied by up to a^2 in every such step.  Measured with gradients of low rank and noise, 16 x 16 to 400 x 401, five steps in
// all, against 64 bits and in the Frobenius norm: the last 4 on S add up to 1e-3 to the result (bf16 rounds by 1.7e-3: taken), the
// last 3 a tenth of that (f16 rounds by 2.1e-4: taken); all 5 would add 2e-3, and in 32 bits not even 2 would do.
#include "common.h"

#include <algorithm>

namespace lt {

typedef f16 half8 __attribute__((ext_vector_type(8)));
typedef f16 half2 __attribute__((ext_vector_type(2)));
typedef f16 half4 __attribute__((ext_vector_type(4)));
typedef float float4_ __attribute__((ext_vector_type(4)));

constexpr int EDGE = 64;     // sides are padded to multiples of it, with zeros ...
constexpr int SPARE = 256;  // ... and so many rows behind a matrix are memory, with whatever they hold: tiles reach beyond the last row
constexpr int NORM_BLOCKS = 256;

struct Split {  // hi and lo parts, dense, padded with zeros to multiples of EDGE
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

// (by value: halves of a vector are no lvalues to refer to)
struct Halves {
    f16 hi, lo;
};
__device__ __forceinline__ Halves split(float v) {
    const f16 hi = (f16)v;
    return {hi, (f16)(v - (float)hi)};
}

// X (m x n, K = n adjacent) and its transpose from G or, tall, from G^T: X = G * factor, and *inv what X has to be multiplied by
// to be G / |G|.  Split: factor = scale / |G|; else the power of two below it, which leaves 16-bit values as they are (lo unused).
template <class T>
__global__ __launch_bounds__(256) void split_kernel(const T* g, int m, int n, int mp, int np, int tall, const double* part, int parts, double scale, Split x, Split xt,
                                                    float* inv) {
    constexpr bool WHOLE = sizeof(T) == 2;
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    const int64_t b = blockIdx.z;
    double norm = wave_sum((int)threadIdx.x < parts ? part[b * NORM_BLOCKS + threadIdx.x] : 0.0);
    if (threadIdx.x % WAVE == 0) sums[threadIdx.x / WAVE] = norm;
    __syncthreads();
    norm = sqrt(sums[0] + sums[1] + sums[2] + sums[3]);
    double f = norm > 0 && norm < INFINITY ? scale / norm : norm == 0 ? 0.0 : NAN;
    if (WHOLE && f > 0) f = ldexp(1.0, ilogb(f));
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) inv[b] = f > 0 ? (float)(1.0 / (f * norm)) : (float)f;
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
    for (int k = threadIdx.x; k < 64 * 32; k += 256) {
        const int r = k / 32, c = k % 32 * 2;
        half2 hi, lo;
        const int64_t o = at + (int64_t)(i0 + r) * np + j0 + c, t = at + (int64_t)(j0 + r) * mp + i0 + c;
        const Halves a0 = split(tile[r][c]), a1 = split(tile[r][c + 1]), b0 = split(tile[c][r]), b1 = split(tile[c + 1][r]);
        hi[0] = a0.hi, hi[1] = a1.hi, lo[0] = a0.lo, lo[1] = a1.lo;
        *(half2*)(x.hi + o) = hi;
        if (!WHOLE) *(half2*)(x.lo + o) = lo;
        hi[0] = b0.hi, hi[1] = b1.hi, lo[0] = b0.lo, lo[1] = b1.lo;
        *(half2*)(xt.hi + t) = hi;
        if (!WHOLE) *(half2*)(xt.lo + t) = lo;
    }
}
// ------------------------------------------------------------------------------------ products
enum { SYM, POLY, STEP, LAST };

struct Product {
    Split l, r;          // C = L R^T, both with K adjacent
    int64_t l_batch, r_batch, o_batch;
    int k, ld;           // K (a multiple of 64), the row length of both
    float scale;         // of the accumulated product, times inv[batch] `inv_power` times
    const float* inv;
    int inv_power;
    // SYM, POLY: C is symmetric, m x m; POLY: scale * C + b * L + a on the diagonal (L itself is S)
    float a, b;
    int m, n;            // real rows and columns of C ...
    int rows, cols;      // ... and padded ones
    int o_ld, t_ld;      // row lengths of o and its transpose t
    Split o, t;
    void* out;           // LAST: the result, in the caller's type and orientation
    int tall;
};

// Which tile a workgroup has.  Workgroups go to the eight dies in turn, each with an L2 of its own: a die gets adjacent tiles,
// and they are numbered down GROUP rows, then across, so that its tiles share rows and columns.  Lower triangle alone if SYM.
struct Place {
    int i, j;
};
__device__ __forceinline__ Place place_of(int id, int tiles, int rows, int cols, bool sym) {
    constexpr int GROUP = 4, DIES = 8;
    const int die = id % DIES, each = tiles / DIES, more = tiles % DIES;
    int t = die * each + (die < more ? die : more) + id / DIES;
    for (int g = 0;; g += GROUP) {
        const int h = rows - g < GROUP ? rows - g : GROUP;  // rows g .. g + h
        if (!sym) {
            if (t < h * cols) return {g + t % h, t / h};
            t -= h * cols;
            continue;
        }
        if (t < h * g) return {g + t % h, t / h};           // columns left of the diagonal's blocks
        t -= h * g;
        if (t < h * (h + 1) / 2) {
            int c = 0;
            while (t >= h - c) t -= h - c, c++;
            return {g + c + t, g + c};
        }
        t -= h * (h + 1) / 2;
    }
}

// One K-step of a tile's operands, as the matrix instructions read them: rows of BK halves, in 16-byte chunks whose places
// within a row are exchanged by the row's number, so that the 16 rows a fragment reads lie in different banks.  The copy goes
// from global memory to LDS directly: an instruction's 64 lanes fill 1024 adjacent bytes, and which chunk a lane asks for
// makes the exchange.
template <int BK>
__device__ __forceinline__ int place(int row, int chunk) {
    return chunk ^ (BK == 32 ? (row >> 1) & 3 : row & 7);
}

// One such copy: 16 bytes a lane from base + off to 1024 adjacent bytes of LDS.  Written out, because the compiler takes any LDS
// read behind its own form of it as one that has to wait for all copies; the waits are the kernel's (ready()).
__device__ __forceinline__ void copy_to_lds(const f16* from, uint32_t off, uint32_t lds) {
    const uint64_t a = (uint64_t)from;  // (the same in all lanes)
    const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a);
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base));
}

struct Sources {  // the first rows of a tile's operands: hi of L, hi of R, lo of L, lo of R
    const f16 *a, *b, *c, *d;
};
template <int TILE, int BK, int ARRAYS>
__device__ __forceinline__ void stage(uint32_t lds, const Sources& src, int ld, int k0) {
    constexpr int CPR = BK / 8, RPI = 64 / CPR, EACH = ARRAYS * TILE / RPI / 4;  // chunks to a row, rows to an instruction, instructions to a wave
    const int lane = threadIdx.x % WAVE, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int row = lane / CPR, chunk = place<BK>(row, lane % CPR);
    const uint32_t off = (uint32_t)(row * ld + chunk * 8) * 2;
#pragma unroll
    for (int u = 0; u < EACH; u++) {
        const int t = wave * EACH + u, array = t / (TILE / RPI), part = t % (TILE / RPI);
        const f16* s = array == 0 ? src.a : array == 1 ? src.b : array == 2 ? src.c : src.d;
        copy_to_lds(s + (int64_t)part * RPI * ld + k0, off, lds + t * 1024);
    }
}

// fragments of one operand: NF blocks of 16 rows, 32 halves of K
template <int BK, int NF>
__device__ __forceinline__ void fragments(const f16* lds, int first, int kk, half8 (&f)[NF]) {
    const int lane = threadIdx.x % WAVE;
#pragma unroll
    for (int x = 0; x < NF; x++) {
        const int row = first + x * 16 + lane % 16;
        f[x] = *(const half8*)&lds[row * BK + place<BK>(row, kk * 4 + lane / 16) * 8];
    }
}
// all products of two operands' fragments, with `READS` LDS reads of the next ones spread between them
template <int NF, int READS>
__device__ __forceinline__ void products(const half8 (&l)[NF], const half8 (&r)[NF], float4_ (&acc)[NF][NF]) {
#pragma unroll
    for (int x = 0; x < NF; x++)
#pragma unroll
        for (int y = 0; y < NF; y++) acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[x], r[y], acc[x][y], 0, 0, 0);
    constexpr int GAP = NF * NF / (READS + 1) > 0 ? NF * NF / (READS + 1) : 1;
#pragma unroll
    for (int k = 0; k < READS; k++) {
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // a read ...
        __builtin_amdgcn_sched_group_barrier(0x008, GAP, 0);  // ... and some products
    }
}

// The second product of a launch, if there is one, is that of the workgroups with the higher numbers along z.
template <class T, int WHAT, int PARTS, int TILE, int STAGES>
__global__ __launch_bounds__(256, TILE <= 128 && STAGES * TILE <= 256 ? 2 : 1) void product_kernel(Product first, Product second, int batch) {
    constexpr int BK = PARTS == 1 ? 64 : 32, ARRAYS = PARTS == 1 ? 2 : PARTS + 1, NF = TILE / 32, ARRAY = TILE * BK;
    constexpr int EACH = ARRAYS * ARRAY / 512 / 4;  // copies of a stage to a wave
    __shared__ __attribute__((aligned(1024))) f16 s0[ARRAYS * ARRAY], s1[ARRAYS * ARRAY], s2[STAGES > 2 ? ARRAYS * ARRAY : 8], s3[STAGES > 3 ? ARRAYS * ARRAY : 8];
    const Product& p = (int)blockIdx.z < batch ? first : second;
    const int64_t b = blockIdx.z % batch;
    const Place at = place_of(blockIdx.x, gridDim.x, (p.rows + TILE - 1) / TILE, (p.cols + TILE - 1) / TILE, WHAT == SYM || WHAT == POLY);
    const int ti = at.i, tj = at.j;
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int wi = (wave / 2) * (TILE / 2), wj = (wave % 2) * (TILE / 2);
    const int64_t l_first = b * p.l_batch + (int64_t)ti * TILE * p.ld, r_first = b * p.r_batch + (int64_t)tj * TILE * p.ld;
    const Sources src = {p.l.hi + l_first, p.r.hi + r_first, p.l.lo + l_first, p.r.lo + r_first};
    float4_ acc[NF][NF];
#pragma unroll
    for (int x = 0; x < NF; x++)
#pragma unroll
        for (int y = 0; y < NF; y++) acc[x][y] = float4_{0, 0, 0, 0};
    // The copies of STAGES - 1 K-steps are under way while one is multiplied.  ready(): the oldest stage's copies of this wave
    // have arrived (the younger ones may still be out), then everybody's have, and nobody reads the stage that is filled next.
    const int steps = p.k / BK;
    auto ready = [&]() {
        constexpr int out = EACH * (STAGES - 2);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | (out & 15) | ((out >> 4) << 14));  // (and this wave's LDS reads are through)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto ask = [&](const f16* buf, int k) {  // (behind the last step the first is copied once more: the count of copies stays)
        stage<TILE, BK, ARRAYS>((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)buf, src, p.ld, k < steps ? k * BK : 0);
    };
    half8 l[NF], r[NF], u[NF], v[NF];  // the step's first fragments; those that follow them
    auto step = [&](f16* now, f16* next, f16* fill, int k) {
        if (PARTS == 1) {
            fragments<BK, NF>(now, wi, 1, u);
            fragments<BK, NF>(now + ARRAY, wj, 1, v);
            products<NF, 2 * NF>(l, r, acc);
            ready();
            ask(fill, k + STAGES);
            fragments<BK, NF>(next, wi, 0, l);
            fragments<BK, NF>(next + ARRAY, wj, 0, r);
            products<NF, 2 * NF>(u, v, acc);
        } else {
            if (PARTS == 3) {
                fragments<BK, NF>(now + 3 * ARRAY, wj, 0, v);  // lo of R
                products<NF, NF>(l, r, acc);                   // hi hi
                fragments<BK, NF>(now + 2 * ARRAY, wi, 0, u);  // lo of L
                products<NF, NF>(l, v, acc);                   // hi lo
            } else {
                fragments<BK, NF>(now + 2 * ARRAY, wi, 0, u);
                products<NF, NF>(l, r, acc);
            }
            ready();
            ask(fill, k + STAGES);
            fragments<BK, NF>(next, wi, 0, l);
            fragments<BK, NF>(next + ARRAY, wj, 0, v);
            products<NF, 2 * NF>(u, r, acc);                   // lo hi
#pragma unroll
            for (int x = 0; x < NF; x++) r[x] = v[x];
        }
    };
    f16* const buf[4] = {s0, s1, s2, s3};
#pragma unroll
    for (int k = 0; k < STAGES; k++) ask(buf[k], k);
    {
        constexpr int out = EACH * (STAGES - 1);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0f70 | (out & 15) | ((out >> 4) << 14));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    fragments<BK, NF>(s0, wi, 0, l);
    fragments<BK, NF>(s0 + ARRAY, wj, 0, r);
    for (int k = 0; k < steps; k += STAGES) {
#pragma unroll
        for (int h = 0; h < STAGES; h++)
            if (k + h < steps) step(buf[h], buf[(h + 1) % STAGES], buf[h], k + h);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the copies behind the last step: none may outlive the workgroup
    float scale = p.scale;
    if (p.inv_power) scale *= p.inv_power == 1 ? p.inv[b] : p.inv[b] * p.inv[b];
    // a lane holds rows i .. i+3 of column j of each 16 x 16 block
#pragma unroll
    for (int x = 0; x < NF; x++)
#pragma unroll
        for (int y = 0; y < NF; y++) {
            const int i = ti * TILE + wi + x * 16 + (lane / 16) * 4, j = tj * TILE + wj + y * 16 + lane % 16;
            if (WHAT != LAST && (i >= p.rows || j >= p.cols)) continue;
            half4 hi, lo, s_hi, s_lo;
            if (WHAT == POLY) {  // (S is symmetric)
                const int64_t at = b * p.l_batch + (int64_t)j * p.ld + i;
                s_hi = *(const half4*)(p.l.hi + at), s_lo = *(const half4*)(p.l.lo + at);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float v = acc[x][y][e] * scale;
                if (WHAT == POLY) {
                    v += p.b * ((float)s_hi[e] + (float)s_lo[e]);
                    if (i + e == j && j < p.m) v += p.a;
                }
                if (WHAT == LAST) {
                    if (i + e < p.m && j < p.n) ((T*)p.out)[b * (int64_t)p.m * p.n + (p.tall ? (int64_t)j * p.m + i + e : (int64_t)(i + e) * p.n + j)] = (T)v;
                } else {
                    const Halves h = split(v);
                    hi[e] = h.hi, lo[e] = h.lo;
                    const int64_t o = b * p.o_batch + (int64_t)(i + e) * p.o_ld + j;
                    p.o.hi[o] = h.hi, p.o.lo[o] = h.lo;
                }
            }
            if (WHAT == STEP || (WHAT != LAST && ti != tj)) {
                const int64_t t = b * p.o_batch + (int64_t)j * p.t_ld + i;
                *(half4*)(p.t.hi + t) = hi, *(half4*)(p.t.lo + t) = lo;
            }
        }
}

// ------------------------------------------------------------------------------------ launches
static int64_t up(int64_t n) { return (n + EDGE - 1) / EDGE * EDGE; }

struct Plan {
    int m, n, mp, np, batch, steps, gram, tall;  // gram: so many of the steps, the last, work on the Gram matrix
    double sx, ss, sp, st, sq;  // what X, S, P, P P and Q are multiplied by
    double a, b, c;
};
struct Buffers {
    Split x[2], xt[2], s[2], p, t, q[2];
    double* part;
    float* inv;
};

static uint64_t lay_out(Buffers* out, void* base, int dtype, int64_t batch, int64_t rows, int64_t cols) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        void* p = (char*)base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const uint64_t m = (uint64_t)up(std::min(rows, cols)), n = (uint64_t)up(std::max(rows, cols)), bt = (uint64_t)batch;
    auto half = [&](uint64_t rows_, uint64_t ld) { return (f16*)take(2 * (bt * rows_ + SPARE) * ld); };
    auto matrix = [&](uint64_t rows_, uint64_t ld) {
        f16* hi = half(rows_, ld);
        return Split{hi, half(rows_, ld)};
    };
    Buffers f = {};
    for (int k = 0; k < 2; k++) f.x[k] = matrix(m, n), f.xt[k] = matrix(n, m);
    f.s[0] = matrix(m, m);
    if (dtype != LBFGS_TRAIN_F32) {
        f.s[1] = matrix(m, m), f.t = matrix(m, m);
        for (int k = 0; k < 2; k++) f.q[k] = matrix(m, m);
    }
    f.p = matrix(m, m);
    f.part = (double*)take(bt * NORM_BLOCKS * sizeof(double));
    f.inv = (float*)take(bt * sizeof(float));
    if (out) *out = f;
    return at;
}

// The largest value of X, S, P and Q that singular values in [0, 1] can lead to, and from them the powers of two that keep f16
// in range.  false: the polynomial leaves it.
static bool ranges(Plan* q) {
    double x_most = 1.0, p_most = 1.0, q_most = 1.0;
    for (int k = 0; k <= 1000; k++) {
        double s = k / 1000.0, all = 1.0;
        for (int j = 0; j < q->steps; j++) {
            const double l = s * s, p = q->a + q->b * l + q->c * l * l;
            s *= p;
            if (j >= q->steps - q->gram) all *= p;
            x_most = std::max(x_most, std::fabs(s));
            p_most = std::max(p_most, std::fabs(p));
            q_most = std::max(q_most, std::fabs(all));
            if (!(x_most < 64 && p_most < 128 && q_most < 16384)) return false;
        }
    }
    auto scale = [](double most) { return std::exp2(std::floor(std::log2(48000.0 / (most * 1.02)))); };
    q->sx = scale(x_most);
    q->ss = scale(x_most * x_most);
    q->sp = scale(p_most);
    q->st = scale(p_most * p_most);
    q->sq = scale(q_most);
    return true;
}

template <class T, int WHAT, int PARTS, int TILE, int STAGES>
static void launch_tiles(const Product& p, const Product* second, int batch, hipStream_t s) {
    const int rows = (p.rows + TILE - 1) / TILE, cols = (p.cols + TILE - 1) / TILE;
    const int tiles = WHAT == SYM || WHAT == POLY ? rows * (rows + 1) / 2 : rows * cols;
    product_kernel<T, WHAT, PARTS, TILE, STAGES><<<dim3(tiles, 1, second ? 2 * batch : batch), 256, 0, s>>>(p, second ? *second : p, batch);
}
// The tile: what the compute unit with the most of them takes, from the time of a K-step of each (three products, all units
// busy, measured at 4000 x 4100): 64: 0.35 us, 128: 0.95, 192: 1.55.
template <class T, int WHAT, int PARTS>
static void launch_product(const Product& p, const Product* second, int batch, hipStream_t s) {
    auto rounds = [&](int tile) {
        const int64_t rows = (p.rows + tile - 1) / tile, cols = (p.cols + tile - 1) / tile;
        const int64_t tiles = (WHAT == SYM || WHAT == POLY ? rows * (rows + 1) / 2 : rows * cols) * batch * (second ? 2 : 1);
        return (tiles + 255) / 256;
    };
    const double t64 = 0.35 * rounds(64), t128 = 0.95 * rounds(128), t192 = 1.55 * rounds(192);
    if (t192 < t128 && t192 < t64)
        launch_tiles<T, WHAT, PARTS, 192, 3>(p, second, batch, s);
    else if (t128 < t64 && rounds(128) == 1)
        launch_tiles<T, WHAT, PARTS, 128, 4>(p, second, batch, s);
    else if (t128 < t64)
        launch_tiles<T, WHAT, PARTS, 128, 2>(p, second, batch, s);
    else
        launch_tiles<T, WHAT, PARTS, 64, 4>(p, second, batch, s);
}

static Product square(const Plan& q, Split l, Split r, Split o) {
    Product p = {};
    p.m = p.n = q.m, p.rows = p.cols = p.k = p.ld = p.o_ld = p.t_ld = q.mp;
    p.l = l, p.r = r, p.o = p.t = o, p.l_batch = p.r_batch = p.o_batch = (int64_t)q.mp * q.mp;
    return p;
}

template <class T>
static void launch_orthogonalize(const Plan& q, const void* g, void* out, const Buffers& f, hipStream_t s) {
    constexpr bool WHOLE = sizeof(T) == 2;
    const int64_t size = (int64_t)q.m * q.n, X = (int64_t)q.mp * q.np;
    const int blocks = (int)std::min<int64_t>(NORM_BLOCKS, (size + 4095) / 4096);
    norm_kernel<T><<<dim3(blocks, q.batch), 256, 0, s>>>((const T*)g, size, f.part);
    split_kernel<T><<<dim3(q.np / 64, q.mp / 64, q.batch), 256, 0, s>>>((const T*)g, q.m, q.n, q.mp, q.np, q.tall, f.part, blocks, q.sx, f.x[0], f.xt[0], f.inv);
    auto gram = [&](int at) {  // S = X X^T
        Product p = square(q, f.x[at], f.x[at], f.s[0]);
        p.l_batch = p.r_batch = X, p.k = p.ld = q.np, p.scale = (float)(q.ss / (q.sx * q.sx));
        return p;
    };
    auto poly = [&](Split from, Split to, double to_scale) {  // a I + b S + c S S
        Product p = square(q, from, from, to);
        p.scale = (float)(q.c * to_scale / (q.ss * q.ss)), p.b = (float)(q.b * to_scale / q.ss), p.a = (float)(q.a * to_scale);
        return p;
    };
    auto wide = [&](Split l, int at, double scale) {  // L X
        Product p = square(q, l, f.xt[at], f.x[at ^ 1]);
        p.r_batch = p.o_batch = X, p.cols = q.np, p.n = q.n, p.t = f.xt[at ^ 1], p.o_ld = q.np, p.tall = q.tall, p.out = out, p.scale = (float)scale;
        return p;
    };
    // of a whole first X: one part, and inv for its scale
    auto first = [&](Product p, int power) {
        p.scale *= (float)std::pow(q.sx, power), p.inv = f.inv, p.inv_power = power;
        return p;
    };
    const int plain = q.steps - q.gram;
    for (int k = 0; k < plain; k++) {
        const int at = k & 1;
        if (WHOLE && k == 0)
            launch_product<float, SYM, 1>(first(gram(at), 2), nullptr, q.batch, s);
        else
            launch_product<float, SYM, 3>(gram(at), nullptr, q.batch, s);
        launch_product<float, POLY, 3>(poly(f.s[0], f.p, q.sp), nullptr, q.batch, s);
        if (WHOLE && k == 0)
            launch_product<float, STEP, 2>(first(wide(f.p, at, 1 / q.sp), 1), nullptr, q.batch, s);
        else if (k + 1 < q.steps)
            launch_product<float, STEP, 3>(wide(f.p, at, 1 / q.sp), nullptr, q.batch, s);
        else
            launch_product<T, LAST, 3>(wide(f.p, at, 1 / (q.sp * q.sx)), nullptr, q.batch, s);
    }
    if (!WHOLE) return;
    const int at = plain & 1;
    if (plain)
        launch_product<float, SYM, 3>(gram(at), nullptr, q.batch, s);
    else
        launch_product<float, SYM, 1>(first(gram(at), 2), nullptr, q.batch, s);
    for (int k = 0; k < q.gram; k++) {
        const int now = k & 1;
        const bool more = k + 1 < q.gram;
        if (k == 0) launch_product<float, POLY, 3>(poly(f.s[0], f.q[0], q.sq), nullptr, q.batch, s);  // Q = P
        if (k || more) launch_product<float, POLY, 3>(poly(f.s[now], f.p, q.sp), nullptr, q.batch, s);
        Product pp = square(q, f.p, f.p, f.t), qp = square(q, f.q[now ^ 1], f.p, f.q[now]);
        pp.scale = (float)(q.st / (q.sp * q.sp)), qp.scale = (float)(1 / q.sp);
        if (more) {
            launch_product<float, SYM, 3>(pp, k ? &qp : nullptr, q.batch, s);
            Product next = square(q, f.s[now], f.t, f.s[now ^ 1]);
            next.scale = (float)(1 / q.st);
            launch_product<float, SYM, 3>(next, nullptr, q.batch, s);
        } else if (k) {
            launch_product<float, SYM, 3>(qp, nullptr, q.batch, s);
        }
    }
    const Product p = wide(f.q[(q.gram - 1) & 1], at, 1 / (q.sq * q.sx));
    if (plain)
        launch_product<T, LAST, 3>(p, nullptr, q.batch, s);
    else
        launch_product<T, LAST, 2>(first(p, 1), nullptr, q.batch, s);
}

}  // namespace lt

using namespace lt;

extern "C" uint64_t lbfgs_train_orthogonalize_workspace(int32_t dtype, int64_t batch, int64_t rows, int64_t cols) {
    if (dtype < LBFGS_TRAIN_F32 || dtype > LBFGS_TRAIN_F16 || batch < 1 || rows < 1 || cols < 1 || batch > 65535 || rows > (1 << 20) || cols > (1 << 20)) return 0;
    return lay_out(nullptr, nullptr, dtype, batch, rows, cols);
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
    Plan q = {(int)std::min(rows, cols), (int)std::max(rows, cols), 0, 0, (int)batch, steps, std::min(steps, dtype == LBFGS_TRAIN_BF16 ? 4 : dtype == LBFGS_TRAIN_F16 ? 3 : 0), rows > cols, 0, 0, 0, 0, 0, a, b, c};
    if (!ranges(&q)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %d steps of %g, %g, %g lead singular values out of range", who, steps, a, b, c);
    if (!batch || !rows || !cols) return LBFGS_HIP_OK;
    if (!update || !out) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: update and out are needed", who);
    q.mp = (int)up(q.m), q.np = (int)up(q.n);
    const uint64_t need = lay_out(nullptr, nullptr, dtype, batch, rows, cols);
    if (!workspace || workspace_bytes < need)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    Buffers f;
    lay_out(&f, workspace, dtype, batch, rows, cols);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case LBFGS_TRAIN_F32: launch_orthogonalize<float>(q, update, out, f, s); break;
        case LBFGS_TRAIN_BF16: launch_orthogonalize<bf16>(q, update, out, f, s); break;
        default: launch_orthogonalize<f16>(q, update, out, f, s);
    }
    return lt_launched(who);
}
