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
//   P = a I + b S + c S S,   Q <- Q P,   S <- (S P) P        and in the end   X <- Q X,
// all symmetric and all of the short side, which for a matrix m x 4 m is a third less work.  The price: an error of S is
// multiplied by up to a^2 in every such step, and by b where it enters P: of g steps, a rounding of 2^-23 becomes
// |b| a^(2 g - 2) 2^-23 of the result, which with the usual polynomial is 9.5e-4 for 4 steps and 8e-5 for 3.  So many are taken,
// of any polynomial, as keep that below 2^-10 for bf16 (which rounds by up to 2^-9) and 2^-13 for f16 (2^-12); in 32 bits not even
// 2 would do.  Measured against 64 bits with gradients of rank 1, 4 and 32 and noise of 1e-2 to 1e-4, 150 x 200 to 512 x 4000, five
// steps, in the Frobenius norm: 1.6e-3 to 1.7e-3 for bf16 and 2.1e-4 to 2.2e-4 for f16, which is what rounding the result takes alone;
// 1.1e-5 to 6.4e-5 for updates of 32 bits.
#include "orthogonal.h"

#include <algorithm>

namespace lt {

constexpr int EDGE = 64;     // sides are padded to multiples of it, with zeros ...
constexpr int SPARE = 256;  // ... and so many rows behind a matrix are memory, with whatever they hold: tiles reach beyond the last row

struct Split {  // hi and lo parts, dense, padded with zeros to multiples of EDGE
    f16 *hi, *lo;
};

// ------------------------------------------------------------------------------------ norm, normalise, split
// (bound by HBM: 4000 x 4100 in 32 bits 22 us, 3.0 TB/s, and 47 us, 4.2 TB/s read and written, of 3390 in all)
template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* g, int64_t n, double* part) {
    constexpr int N = vec_len<T>();
    const T* x = g + (int64_t)blockIdx.y * n;
    double s = 0;
    const int64_t packs = n / N;
    constexpr int U = 4;  // (loads under way at once)
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < packs; i += U * stride) {
        Pack<T, N> p[U];
#pragma unroll
        for (int u = 0; u < U; u++) p[u] = ((const Pack<T, N>*)x)[i + u * stride < packs ? i + u * stride : i];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i + u * stride < packs)
#pragma unroll
                for (int k = 0; k < N; k++) s += (double)p[u].v[k] * (double)p[u].v[k];
    }
    if (blockIdx.x == 0)
        for (int64_t i = packs * N + threadIdx.x; i < n; i += 256) s += (double)x[i] * (double)x[i];
    __shared__ double w[4];
    s = wave_sum(s);
    if (threadIdx.x % WAVE == 0) w[threadIdx.x / WAVE] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = w[0] + w[1] + w[2] + w[3];
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

// One such copy: 16 bytes a lane from base + off to 1024 bytes of LDS.  Written out, because the compiler takes
// any LDS read behind its own form of it as one that has to wait for all copies; the waits are the kernel's (ready()).
__device__ __forceinline__ void copy_to_lds(const f16* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0");
}
__device__ __forceinline__ const f16* uniform(const f16* p) {  // (the same in all lanes: to scalar registers)
    const uint64_t a = (uint64_t)p;
    return (const f16*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a));
}

// A K-step's copies are dealt to four waves in turn (of eight, each four have half of the arrays), so that copy u of a wave belongs to an array that is known when this is
// compiled, and its rows to one of OFFS byte offsets that stay the same throughout: what is left to do is a scalar addition each.
// (With the addresses made from the copy's number a step of 108 products spent as long on 400 scalar instructions.)
struct Sources {  // the first rows of a tile's operands: hi of L, hi of R, lo of L, lo of R
    const f16 *a, *b, *c, *d;
};
template <int TILE, int BK>
constexpr int offsets_of() {
    return TILE * BK / 512 / 4;
}
template <int TILE, int BK>
__device__ __forceinline__ void offsets(int ld, uint32_t (&off)[offsets_of<TILE, BK>()]) {
    constexpr int CPR = BK / 8, RPI = 64 / CPR;  // chunks to a row, rows to a copy
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE % 4, row = lane / CPR, chunk = place<BK>(row, lane % CPR);
#pragma unroll
    for (int u = 0; u < offsets_of<TILE, BK>(); u++) off[u] = (uint32_t)(((u * 4 + wave) * RPI + row) * ld + chunk * 8) * 2;
}
// copies [from, to) of a K-step
template <int TILE, int BK>
__device__ __forceinline__ void stage(uint32_t lds, const Sources& src, const uint32_t (&off)[offsets_of<TILE, BK>()], int k0, int from, int to) {
    constexpr int OFFS = offsets_of<TILE, BK>();
#pragma unroll
    for (int u = from; u < to; u++) {
        const int array = u / OFFS;
        copy_to_lds((array == 0 ? src.a : array == 1 ? src.b : array == 2 ? src.c : src.d) + k0, off[u % OFFS], lds + u * 4096);
    }
}

// fragment x of one operand: 16 rows, 32 halves of K
template <int BK>
__device__ __forceinline__ half8 fragment(const f16* lds, int first, int kk, int x) {
    const int lane = threadIdx.x % WAVE, row = first + x * 16 + lane % 16;
    return *(const half8*)&lds[row * BK + place<BK>(row, kk * 4 + lane / 16) * 8];
}
// All products of two operands' fragments, a column at a time: before each, slot(n) asks for what is needed later -- reads of LDS
// and copies to it, a few at a time, so that the matrix unit always has products to work on while they are served.
template <int NI, int NJ, class F>
__device__ __forceinline__ void products(const half8 (&l)[NI], const half8 (&r)[NJ], float4_ (&acc)[NI][NJ], F slot) {
#pragma unroll
    for (int n = 0; n < NJ; n++) {
        slot(n);
#pragma unroll
        for (int x = 0; x < NI; x++) acc[x][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[x], r[n], acc[x][n], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// C = L R^T by tiles of TILE x TILE.  Bound by the matrix units: 4000 x 4100 in 32 bits takes 165 us for S, 170 for P and 331 for P X, each
// 1.19 PFLOP/s of f16 products (a library's product of 8192^3 in f16, 1.21 on this card).  Small ones are bound by the launch: 5 us at
// 128 x 256, whatever is in it; in between by what one compute unit takes in, 37 bytes a cycle (K = 2000 on three units 16 us; two
// groups of waves to a tile, each with half of K, took as long).
// The second product of a launch, if there is one, is that of the workgroups with the higher numbers along z.
template <class T, int WHAT, int PARTS, int TILE, int STAGES, int WAVES>
__global__ __launch_bounds__(WAVES * WAVE, TILE <= 128 && STAGES * TILE <= 256 ? 2 : WAVES / 4) void product_kernel(Product first, Product second, int batch) {
    constexpr int BK = PARTS == 1 ? 64 : 32, ARRAYS = PARTS == 1 ? 2 : PARTS + 1, ARRAY = TILE * BK;
    constexpr int NI = TILE / 32, NJ = TILE / 16 / (WAVES / 2);  // a wave's blocks: the waves lie 2 x WAVES / 2
    constexpr int TEAMS = WAVES / 4, EACH = ARRAYS * ARRAY / 512 / WAVES;  // four waves copy every TEAMS-th part of the arrays; copies of a stage to a wave
    static_assert(ARRAYS % TEAMS == 0, "a team's arrays");
    constexpr int LINE = TILE + 4;  // of the 32-bit result in LDS
    constexpr int STAGED = STAGES * ARRAYS * ARRAY * 2, RESULT = TILE * LINE * 4;
    __shared__ __attribute__((aligned(1024))) char pool[STAGED > RESULT ? STAGED : RESULT];
    const Product& p = (int)blockIdx.z < batch ? first : second;
    const int64_t b = blockIdx.z % batch;
    const Place at = place_of(blockIdx.x, gridDim.x, (p.rows + TILE - 1) / TILE, (p.cols + TILE - 1) / TILE, WHAT == SYM || WHAT == POLY);
    const int ti = at.i, tj = at.j;
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int wi = wave / (WAVES / 2) * (TILE / 2), wj = wave % (WAVES / 2) * (NJ * 16);
    const int64_t l_first = b * p.l_batch + (int64_t)ti * TILE * p.ld, r_first = b * p.r_batch + (int64_t)tj * TILE * p.ld;
    const bool later = TEAMS == 2 && wave >= 4;  // the second team: the second half of the arrays
    const Sources src = {uniform(!later ? p.l.hi + l_first : ARRAYS == 2 ? p.r.hi + r_first : p.l.lo + l_first),
                         uniform(!later ? p.r.hi + r_first : p.r.lo + r_first), uniform(p.l.lo + l_first), uniform(p.r.lo + r_first)};
    uint32_t off[offsets_of<TILE, BK>()];
    offsets<TILE, BK>(p.ld, off);
    float4_ acc[NI][NJ], low[NI][NJ];  // of hi hi, and (three parts) of the others, 2^-11 of it: added to it one by one they would be cut off
#pragma unroll
    for (int x = 0; x < NI; x++)
#pragma unroll
        for (int y = 0; y < NJ; y++) acc[x][y] = low[x][y] = float4_{0, 0, 0, 0};
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
    // A stage's copies are spread over the products that follow its becoming free: SLOTS columns of them, the last NJ of a
    // step and, where there are stages enough, all of the next step's before it waits.
    constexpr bool SPREAD = STAGES > 2;
    constexpr int SLOTS = (!SPREAD ? 1 : PARTS == 3 ? 3 : 2) * NJ;
    const uint32_t pool_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)pool;
    auto ask = [&](int buf, int k, int from, int to) {  // (behind the last step that one is copied once more: the count of copies stays)
        const uint32_t lds = __builtin_amdgcn_readfirstlane(pool_at + (uint32_t)(wave % 4 * 1024 + wave / 4 * (ARRAYS / TEAMS * ARRAY * 2))) + buf * (ARRAYS * ARRAY * 2);
        stage<TILE, BK>(lds, src, off, (k < steps ? k : steps - 1) * BK, from * EACH / SLOTS, to * EACH / SLOTS);
    };
    // The products go column by column: a fragment of R is done with then, and the next step's takes its registers.
    constexpr int LOT = (NI + NJ - 1) / NJ + (NJ > 3);  // fragments of L to a column, so that the last come before they are needed
    half8 l[NI], r[NJ], u[NI], v[NJ];  // the step's first fragments; those that follow them
    auto step = [&](int h, int k) {
        const f16* now = (const f16*)pool + h * ARRAYS * ARRAY;
        const f16* next = (const f16*)pool + (h + 1) % STAGES * ARRAYS * ARRAY;
        const int prev = (h + STAGES - 1) % STAGES;
        if (PARTS == 1) {
            products(l, r, acc, [&](int n) {
                if (SPREAD) ask(prev, k + STAGES - 1, NJ + n, NJ + n + 1);
#pragma unroll
                for (int q = n * LOT; q < NI && q < n * LOT + LOT; q++) u[q] = fragment<BK>(now, wi, 1, q);
                v[n] = fragment<BK>(now + ARRAY, wj, 1, n);
            });
            ready();
            products(u, v, acc, [&](int n) {
                ask(h, k + STAGES, n, n + 1);
#pragma unroll
                for (int q = n * LOT; q < NI && q < n * LOT + LOT; q++) l[q] = fragment<BK>(next, wi, 0, q);
                r[n] = fragment<BK>(next + ARRAY, wj, 0, n);
            });
        } else {
            if (PARTS == 3) {
                products(l, r, acc, [&](int n) {  // hi hi
                    if (SPREAD) ask(prev, k + STAGES - 1, NJ + n, NJ + n + 1);
                    v[n] = fragment<BK>(now + 3 * ARRAY, wj, 0, n);  // lo of R
                });
                products(l, v, low, [&](int n) {  // hi lo
                    if (SPREAD) ask(prev, k + STAGES - 1, 2 * NJ + n, 2 * NJ + n + 1);
#pragma unroll
                    for (int q = n * LOT; q < NI && q < n * LOT + LOT; q++) u[q] = fragment<BK>(now + 2 * ARRAY, wi, 0, q);  // lo of L
                });
            } else {
                products(l, r, acc, [&](int n) {
                    if (SPREAD) ask(prev, k + STAGES - 1, NJ + n, NJ + n + 1);
#pragma unroll
                    for (int q = n * LOT; q < NI && q < n * LOT + LOT; q++) u[q] = fragment<BK>(now + 2 * ARRAY, wi, 0, q);
                });
            }
            ready();
            products(u, r, PARTS == 3 ? low : acc, [&](int n) {  // lo hi
                ask(h, k + STAGES, n, n + 1);
#pragma unroll
                for (int q = n * LOT; q < NI && q < n * LOT + LOT; q++) l[q] = fragment<BK>(next, wi, 0, q);
                if (n) r[n - 1] = fragment<BK>(next + ARRAY, wj, 0, n - 1);
            });
            r[NJ - 1] = fragment<BK>(next + ARRAY, wj, 0, NJ - 1);
        }
    };
#pragma unroll
    for (int k = 0; k < STAGES - 1; k++) ask(k, k, 0, SLOTS);
    ask(STAGES - 1, STAGES - 1, 0, NJ);
    {
        constexpr int out = EACH * (STAGES - 2) + NJ * EACH / SLOTS;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0f70 | (out & 15) | ((out >> 4) << 14));
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int x = 0; x < NI; x++) l[x] = fragment<BK>((const f16*)pool, wi, 0, x);
#pragma unroll
    for (int y = 0; y < NJ; y++) r[y] = fragment<BK>((const f16*)pool + ARRAY, wj, 0, y);
    for (int k = 0; k < steps; k += STAGES) {
#pragma unroll
        for (int h = 0; h < STAGES; h++)
            if (k + h < steps) step(h, k + h);
    }
    // The result goes through LDS, in 32 bits: a lane has 4 adjacent rows of a column, and what is stored are rows, of C and of
    // its transpose, 16 bytes a lane.  (Stored from the registers, 2 bytes a lane, the code for it alone -- 20 KB in a straight
    // line, fetched once -- took 14 us for a tile of 192.)  A column's rows are turned by 16 in every other 8 columns: the reads
    // across columns then find other banks.
    __builtin_amdgcn_s_waitcnt(0x0070);  // the copies behind the last step, and this wave's LDS reads
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    float* const res = (float*)pool;
    auto spot = [](int i, int j) { return j * LINE + (i + 16 * (j >> 3 & 1)) % TILE; };
    // A symmetric result is exactly so, on the diagonal too: a difference between its halves, as the factors' own roundings make
    // it where they should commute, grows by more than ten with every step on the Gram matrix (to 8e-3 of a result of bf16).
    const bool diagonal = (WHAT == SYM || WHAT == POLY) && ti == tj;
#pragma unroll
    for (int x = 0; x < NI; x++)
#pragma unroll
        for (int y = 0; y < NJ; y++) {
            const float4_ v = PARTS == 3 ? acc[x][y] + low[x][y] : acc[x][y];
            const int i = wi + x * 16 + (lane / 16) * 4, j = wj + y * 16 + lane % 16;
            const int below = wi + x * 16 - (wj + y * 16);
            if (!diagonal || below > 0) *(float4_*)&res[spot(i, j)] = v;
            if (diagonal && below > 0) {
#pragma unroll
                for (int e = 0; e < 4; e++) res[spot(j, i + e)] = v[e];
            } else if (diagonal && below == 0) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (i + e >= j) res[spot(i + e, j)] = res[spot(j, i + e)] = v[e];
            }
        }
    __syncthreads();
    float scale = p.scale;
    if (p.inv_power) scale *= p.inv_power == 1 ? p.inv[b] : p.inv[b] * p.inv[b];
    // 8 adjacent values of one row of C (or of its transpose): row `first`, columns `second` ...
    auto emit = [&](const float (&v)[8], int first, int second, bool transposed) {
        if constexpr (WHAT == LAST) {
            const int rows = transposed ? p.n : p.m, cols = transposed ? p.m : p.n;
            if (first >= rows || second >= cols) return;
            T* o = (T*)p.out + b * (int64_t)p.m * p.n + (int64_t)first * cols + second;
            Pack<T, 8> w;
#pragma unroll
            for (int e = 0; e < 8; e++) w.v[e] = (T)(v[e] * scale);
            if (second + 8 <= cols)
                *(Pack<T, 8>*)o = w;
            else
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (second + e < cols) o[e] = w.v[e];
        } else {
            if (first >= (transposed ? p.cols : p.rows) || second >= (transposed ? p.rows : p.cols)) return;
            half8 hi, lo, s_hi, s_lo;
            if (WHAT == POLY) {  // (S is symmetric)
                const int64_t from = b * p.l_batch + (int64_t)first * p.ld + second;
                s_hi = *(const half8*)(p.l.hi + from), s_lo = *(const half8*)(p.l.lo + from);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float w = v[e] * scale;
                if (WHAT == POLY) {
                    w += p.b * ((float)s_hi[e] + (float)s_lo[e]);
                    if (first == second + e && first < p.m) w += p.a;
                }
                const Halves h = split(w);
                hi[e] = h.hi, lo[e] = h.lo;
            }
            const int64_t to = b * p.o_batch + (int64_t)first * (transposed ? p.t_ld : p.o_ld) + second;
            *(half8*)((transposed ? p.t.hi : p.o.hi) + to) = hi;
            *(half8*)((transposed ? p.t.lo : p.o.lo) + to) = lo;
        }
    };
    if (WHAT == STEP || (WHAT == LAST && p.tall) || ((WHAT == SYM || WHAT == POLY) && ti != tj)) {
#pragma unroll 2
        for (int k = tid; k < TILE * TILE / 8; k += WAVES * WAVE) {
            const int j = k / (TILE / 8), i = k % (TILE / 8) * 8;
            float v[8];
            *(float4_*)v = *(const float4_*)&res[spot(i, j)], *(float4_*)(v + 4) = *(const float4_*)&res[spot(i, j) + 4];
            emit(v, tj * TILE + j, ti * TILE + i, true);
        }
    }
    if (WHAT != LAST || !p.tall) {
#pragma unroll 2
        for (int k = tid; k < TILE * TILE / 8; k += WAVES * WAVE) {
            const int g = k / WAVE, i = g % (TILE / 16) * 16 + lane % 16, j = g / (TILE / 16) * 32 + lane / 16 * 8;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = res[spot(i, j + e)];
            emit(v, ti * TILE + i, tj * TILE + j, false);
        }
    }
}

// ------------------------------------------------------------------------------------ launches
static int64_t up(int64_t n) { return (n + EDGE - 1) / EDGE * EDGE; }

struct Plan {
    int m, n, mp, np, batch, steps, tall;
    int gram;    // so many of the steps, the last, work on the Gram matrix
    bool brief;  // all of them, in 64 bits (orthogonal_short.hip)
    double sx, ss, sp, sq;  // what X, S (and S P), P and Q are multiplied by
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

// How many steps, the last, may work on the Gram matrix: an error of S is multiplied by up to p^2 in each that follows (p: what a
// step multiplies a singular value by at most) and then by b, and may reach `most`.
static int gram_steps(const Plan& q, double p, double error, double most) {
    const double growth = std::max(1.0, p * p);
    error *= std::max(1.0, std::fabs(q.b));
    int g = 1;
    while (g < q.steps && error * growth <= most) error *= growth, g++;
    return g;
}
// The largest values of X, S, P and Q that singular values in [0, 1] can lead to.  From them: how many steps work on the Gram
// matrix, and the powers of two that keep f16 in range.  false: the polynomial leaves it.
static bool ranges(Plan* q, int dtype) {
    double x_most = 1.0, p_most = 1.0, q_most = 1.0;
    for (int k = 0; k <= 1000; k++) {
        double s = k / 1000.0;
        for (int j = 0; j < q->steps; j++) {
            const double l = s * s, p = q->a + q->b * l + q->c * l * l;
            s *= p;
            x_most = std::max(x_most, std::fabs(s));
            p_most = std::max(p_most, std::fabs(p));
            if (!(x_most < 64 && p_most < 128)) return false;
        }
    }
    q->brief = q->m <= SHORT && gram_steps(*q, p_most, 0x1p-52, 0x1p-26) == q->steps;
    q->gram = dtype == LBFGS_TRAIN_F32 ? 0 : gram_steps(*q, p_most, 0x1p-23, dtype == LBFGS_TRAIN_BF16 ? 0x1p-10 : 0x1p-13);
    for (int j = 0; j < q->gram; j++) q_most *= p_most;  // (2^13.5 at most: p_most^(gram - 1) has passed, < 2^6.5, times 2^7)
    auto scale = [](double most) { return std::exp2(std::floor(std::log2(48000.0 / (most * 1.02)))); };
    q->sx = scale(x_most);
    q->ss = scale(x_most * x_most);
    q->sp = scale(p_most);
    q->sq = scale(q_most);
    return true;
}

template <class T, int WHAT, int PARTS, int TILE, int STAGES, int WAVES>
static void launch_tiles(const Product& p, const Product* second, int batch, hipStream_t s) {
    const int rows = (p.rows + TILE - 1) / TILE, cols = (p.cols + TILE - 1) / TILE;
    const int tiles = WHAT == SYM || WHAT == POLY ? rows * (rows + 1) / 2 : rows * cols;
    product_kernel<T, WHAT, PARTS, TILE, STAGES, WAVES><<<dim3(tiles, 1, second ? 2 * batch : batch), WAVES * WAVE, 0, s>>>(p, second ? *second : p, batch);
}
// The tile: the one with which the compute unit that has the most of them is done first.  What a tile takes, in us, measured with
// three products a K-step at 4000 x 4100 (all units busy) and 128 x 256 (a few steps): 64: 0.31 a step and 1.5 beside, 128: 0.72 and 4,
// 192: 1.32 and 8.  (64 and 128 in two stages: two workgroups a unit.)
template <class T, int WHAT, int PARTS>
static void launch_product(const Product& p, const Product* second, int batch, hipStream_t s) {
    const double steps = p.k / 32 * (PARTS / 3.0);
    auto rounds = [&](int tile) {
        const int64_t rows = (p.rows + tile - 1) / tile, cols = (p.cols + tile - 1) / tile;
        const int64_t tiles = (WHAT == SYM || WHAT == POLY ? rows * (rows + 1) / 2 : rows * cols) * batch * (second ? 2 : 1);
        return (tiles + 255) / 256;
    };
    const double t64 = rounds(64) * (0.31 * steps + 1.5), t128 = rounds(128) * (0.72 * steps + 4), t192 = rounds(192) * (1.32 * steps + 8);
    if (t192 < t128 && t192 < t64)
        launch_tiles<T, WHAT, PARTS, 192, 3, PARTS == 2 ? 4 : 8>(p, second, batch, s);
    else if (t128 < t64 && rounds(128) == 1)
        launch_tiles<T, WHAT, PARTS, 128, 4, 4>(p, second, batch, s);
    else if (t128 < t64)
        launch_tiles<T, WHAT, PARTS, 128, 2, 4>(p, second, batch, s);
    else
        launch_tiles<T, WHAT, PARTS, 64, 4, 4>(p, second, batch, s);
}

static Product square(const Plan& q, Split l, Split r, Split o) {
    Product p = {};
    p.m = p.n = q.m, p.rows = p.cols = p.k = p.ld = p.o_ld = p.t_ld = q.mp;
    p.l = l, p.r = r, p.o = p.t = o, p.l_batch = p.r_batch = p.o_batch = (int64_t)q.mp * q.mp;
    return p;
}

static int norm_blocks(const Plan& q) { return (int)std::min<int64_t>(NORM_BLOCKS, ((int64_t)q.m * q.n + 4095) / 4096); }
template <class T>
static void launch_norm(const Plan& q, const void* g, double* part, hipStream_t s) {
    norm_kernel<T><<<dim3(norm_blocks(q), q.batch), 256, 0, s>>>((const T*)g, (int64_t)q.m * q.n, part);
}
template <class T>
static void launch_panels(const Plan& q, const Panel& p, hipStream_t s) {
    launch_norm<T>(q, p.update, (double*)p.workspace, s);
    panel_orthogonalize<T>(p, s);
}

template <class T>
static void launch_orthogonalize(const Plan& q, const void* g, void* out, const Buffers& f, hipStream_t s) {
    constexpr bool WHOLE = sizeof(T) == 2;
    const int64_t X = (int64_t)q.mp * q.np;
    const int blocks = norm_blocks(q);
    launch_norm<T>(q, g, f.part, s);
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
        const Split step = k ? f.p : f.q[0];  // (Q = P at first)
        const double step_scale = k ? q.sp : q.sq;
        launch_product<float, POLY, 3>(poly(f.s[now], step, step_scale), nullptr, q.batch, s);
        Product sp = square(q, f.s[now], step, f.t), qp = square(q, f.q[now ^ 1], f.p, f.q[now]);
        sp.scale = (float)(1 / step_scale), qp.scale = (float)(1 / q.sp);
        if (more) {
            launch_product<float, SYM, 3>(sp, k ? &qp : nullptr, q.batch, s);
            Product next = square(q, f.t, step, f.s[now ^ 1]);
            next.scale = (float)(1 / step_scale);
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
    if (dtype < LBFGS_TRAIN_F32 || dtype > LBFGS_TRAIN_F16 || batch < 1 || rows < 1 || cols < 1 || batch > 32767 || rows > (1 << 20) || cols > (1 << 20)) return 0;
    const uint64_t size = lay_out(nullptr, nullptr, dtype, batch, rows, cols);
    const int m = (int)std::min(rows, cols), n = (int)std::max(rows, cols);
    if (m <= SHORT) return std::max(size, short_workspace(batch, m, n));  // (which of the two it is depends on the steps)
    return panel_fits(dtype, batch, m, n) ? panel_workspace(batch, m, n) : size;
}

extern "C" int lbfgs_train_orthogonalize(int32_t dtype, int64_t batch, int64_t rows, int64_t cols, const void* update, void* out, int32_t steps, double a, double b,
                                         double c, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* who = "lbfgs_train_orthogonalize";
    if (dtype < LBFGS_TRAIN_F32 || dtype > LBFGS_TRAIN_F16)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: element type %d: float32, bfloat16 and float16 are offered", who, dtype);
    if (batch < 0 || rows < 0 || cols < 0 || batch > 32767 || rows > (1 << 20) || cols > (1 << 20))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld matrices of %lld x %lld", who, (long long)batch, (long long)rows, (long long)cols);
    if (steps < 1 || steps > 64) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %d steps: 1 to 64 are offered", who, steps);
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: coefficients %g, %g, %g", who, a, b, c);
    Plan q = {(int)std::min(rows, cols), (int)std::max(rows, cols), 0, 0, (int)batch, steps, rows > cols, 0, false, 0, 0, 0, 0, a, b, c};
    if (!ranges(&q, dtype)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %d steps of %g, %g, %g lead singular values out of range", who, steps, a, b, c);
    if (!batch || !rows || !cols) return LBFGS_HIP_OK;
    if (!update || !out) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: update and out are needed", who);
    q.mp = (int)up(q.m), q.np = (int)up(q.n);
    const uint64_t need = lbfgs_train_orthogonalize_workspace(dtype, batch, rows, cols);
    if (!workspace || workspace_bytes < need)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    if ((uintptr_t)workspace % 256) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: the workspace is not aligned to 256 bytes", who);
    hipStream_t s = (hipStream_t)stream;
    if (q.brief) {
        const Short p = {update, out, workspace, q.m, q.n, q.tall, q.batch, q.steps, a, b, c};
        switch (dtype) {
            case LBFGS_TRAIN_F32: short_orthogonalize<float>(p, s); break;
            case LBFGS_TRAIN_BF16: short_orthogonalize<bf16>(p, s); break;
            default: short_orthogonalize<f16>(p, s);
        }
        return lt_launched(who);
    }
    if (panel_fits(dtype, batch, q.m, q.n)) {
        const Panel p = {update, out, workspace, q.m, q.n, q.tall, q.batch, q.steps, a, b, c, q.sx, q.ss, q.sp, norm_blocks(q)};
        switch (dtype) {
            case LBFGS_TRAIN_F32: launch_panels<float>(q, p, s); break;
            case LBFGS_TRAIN_BF16: launch_panels<bf16>(q, p, s); break;
            default: launch_panels<f16>(q, p, s);
        }
        return lt_launched(who);
    }
    Buffers f;
    lay_out(&f, workspace, dtype, batch, rows, cols);
    switch (dtype) {
        case LBFGS_TRAIN_F32: launch_orthogonalize<float>(q, update, out, f, s); break;
        case LBFGS_TRAIN_BF16: launch_orthogonalize<bf16>(q, update, out, f, s); break;
        default: launch_orthogonalize<f16>(q, update, out, f, s);
    }
    return lt_launched(who);
}
