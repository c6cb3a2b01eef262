// rust-lbfgs_amd/csrc/train/logprobs.hip -- token log-probabilities and the gradient of their logits.
//
//   l_t  = x_t[y_t]/tau - log sum_v exp(x_tv/tau)            dx_tv = g_t/tau * (1[v = y_t] - exp(x_tv/tau - lse_t))
//
// Both are bound by HBM: the forward pass reads every logit once (running maximum and sum in registers), the gradient
// reads it once more and writes as much.  Measured in bf16 (a copy of 2 GiB: 4.93 TB/s, read and written): 8192 x 131072 forward
// 347 us, 6.2 TB/s; 8192 x 32768 forward 79 to 110 us, 4.8 TB/s and more, gradient 173 us, 6.2 TB/s, part of what both read being in the
// caches yet; 1020 rows of 50001 in 32 bits, 16-byte loads at any alignment, 29 and 57 us; 4096 x 32768 in 64 bits
// 210 and 380, 5.1 and 5.6 TB/s.  Few rows are bound by the launch: 8 of 32768 5.
#include "common.h"

#include <algorithm>

namespace lt {

template <class A>
struct MaxSum {  // sum of exp((x - m)/tau) over what has been seen; m starts at the lowest finite value, never at -inf: (-inf) - (-inf)
    A m, s;      // would be NaN for a masked row part, while (-inf) - lowest is -inf and exp of it 0
};
template <class A>
__device__ __forceinline__ A lowest();
template <>
__device__ __forceinline__ float lowest<float>() {
    return -3.402823466e+38f;
}
template <>
__device__ __forceinline__ double lowest<double>() {
    return -1.7976931348623157e+308;
}

// (the larger of two, of three in one instruction; a NaN is passed over here and shows in the sum)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }

template <class A>
__device__ __forceinline__ void join(MaxSum<A>& a, A m, A s, A c) {
    const A M = larger(a.m, m);
    a.s = a.s * exp2_of((a.m - M) * c) + s * exp2_of((m - M) * c);
    a.m = M;
}

// U packs of N elements at once: one maximum, then one exponential an element.  Differences are taken before the scale
// (x - m is exact for 16-bit logits), so the scale's own rounding stays a relative error of the exponent's size.
template <class T, int N, int U, class A>
__device__ __forceinline__ void add(MaxSum<A>& a, const Pack<T, N> (&p)[U], A c) {
    A v = a.m;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int k = 0; k < N; k++) v = larger(v, (A)p[u].v[k]);
    if (v > a.m) {
        a.s *= exp2_of((a.m - v) * c);
        a.m = v;
    }
    A s = 0;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int k = 0; k < N; k++) s += exp2_of(((A)p[u].v[k] - a.m) * c);
    a.s += s;
}

// one workgroup's share of a row -> every thread of wave 0 holds the result
template <class T, int BLOCK>
__device__ __forceinline__ MaxSum<typename Num<T>::acc> row_part(const T* x, int64_t n, typename Num<T>::acc c) {
    typedef typename Num<T>::acc A;
    constexpr int N = vec_len<T>(), U = 4;
    MaxSum<A> a = {lowest<A>(), (A)0};
    const int tid = threadIdx.x;
    const int64_t lead = (int64_t)((16 - ((uintptr_t)x & 15)) & 15) / (int64_t)sizeof(T);  // elements before the first 16-byte boundary
    const int64_t head = lead < n ? lead : n;
    const int64_t packs = (n - head) / N;
    const Pack<T, N>* body = (const Pack<T, N>*)(x + head);
    int64_t i = tid;
    for (; i + (U - 1) * BLOCK < packs; i += U * BLOCK) {
        Pack<T, N> p[U];
#pragma unroll
        for (int u = 0; u < U; u++) p[u] = *(const Pack<T, N>*)__builtin_assume_aligned(body + i + u * BLOCK, 16);
        add<T, N, U, A>(a, p, c);
    }
    for (; i < packs; i += BLOCK) {
        Pack<T, N> p[1] = {*(const Pack<T, N>*)__builtin_assume_aligned(body + i, 16)};
        add<T, N, 1, A>(a, p, c);
    }
    const int64_t done = head + packs * N;
    for (int64_t k = tid; k < head + (n - done); k += BLOCK) {
        Pack<T, 1> p[1] = {{{x[k < head ? k : done + (k - head)]}}};
        add<T, 1, 1, A>(a, p, c);
    }
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) join(a, shfl_xor(a.m, o), shfl_xor(a.s, o), c);
    if (BLOCK > WAVE) {
        __shared__ A part[2][BLOCK / WAVE];
        if (tid % WAVE == 0) part[0][tid / WAVE] = a.m, part[1][tid / WAVE] = a.s;
        __syncthreads();
        const int k = tid % WAVE;
        a.m = k < BLOCK / WAVE ? part[0][k] : lowest<A>();
        a.s = k < BLOCK / WAVE ? part[1][k] : (A)0;
#pragma unroll
        for (int o = BLOCK / WAVE / 2; o; o >>= 1) join(a, shfl_xor(a.m, o), shfl_xor(a.s, o), c);
    }
    return a;
}

struct Rows {
    int64_t rows, inner, outer_stride, inner_stride, vocab;
    const int64_t* targets;
    int64_t ignore;
};
template <class T>
__device__ __forceinline__ const T* row_at(const T* x, const Rows& r, int64_t row) {
    return x + (row / r.inner) * r.outer_stride + (row % r.inner) * r.inner_stride;
}

// the target's logit, asked for before the row is read (NaN: there is none)
template <class T>
__device__ __forceinline__ typename Num<T>::acc target(const T* x, const Rows& r, int64_t y) {
    typedef typename Num<T>::acc A;
    return y >= 0 && y < r.vocab ? (A)x[y] : (A)NAN;
}
template <class A>
__device__ __forceinline__ void finish_row(A chosen, MaxSum<A> a, double tau, A* logp, double* lse) {
    // (x_y - m) - log s: nothing as large as the logits themselves is rounded, and a row masked by the type's lowest value
    // throughout keeps its log s
    *logp = (A)(((double)chosen - (double)a.m) / tau) - log(a.s);
    lse[0] = (double)a.m;
    lse[1] = log((double)a.s);
}

template <class T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void logprobs_kernel(const T* x, Rows r, double tau, typename Num<T>::acc c, typename Num<T>::acc* logps, double* lse) {
    for (int64_t row = blockIdx.x; row < r.rows; row += gridDim.x) {
        const int64_t y = r.targets[row];
        if (y == r.ignore) {  // not read
            if (threadIdx.x == 0) logps[row] = 0, lse[2 * row] = 0, lse[2 * row + 1] = 0;
            continue;
        }
        const T* at = row_at(x, r, row);
        const auto chosen = target(at, r, y);
        const auto a = row_part<T, BLOCK>(at, r.vocab, c);
        if (threadIdx.x == 0) finish_row(chosen, a, tau, logps + row, lse + 2 * row);
        __syncthreads();  // row_part's shared memory is written again
    }
}

// few rows: `splits` workgroups share a row (their parts start at multiples of `part` elements), a wave joins what they found
template <class T, int BLOCK>
__global__ __launch_bounds__(BLOCK) void logprobs_part_kernel(const T* x, Rows r, typename Num<T>::acc c, int64_t part, MaxSum<typename Num<T>::acc>* found) {
    const int64_t row = blockIdx.y, at = blockIdx.x * part;
    if (r.targets[row] == r.ignore) return;
    const auto a = row_part<T, BLOCK>(row_at(x, r, row) + at, r.vocab - at < part ? r.vocab - at : part, c);
    if (threadIdx.x == 0) found[row * gridDim.x + blockIdx.x] = a;
}
template <class T>
__global__ __launch_bounds__(WAVE) void logprobs_join_kernel(const T* x, Rows r, double tau, typename Num<T>::acc c, int splits,
                                                             const MaxSum<typename Num<T>::acc>* found, typename Num<T>::acc* logps, double* lse) {
    typedef typename Num<T>::acc A;
    const int64_t row = blockIdx.x, y = r.targets[row];
    if (y == r.ignore) {
        if (threadIdx.x == 0) logps[row] = 0, lse[2 * row] = 0, lse[2 * row + 1] = 0;
        return;
    }
    const A chosen = target(row_at(x, r, row), r, y);
    MaxSum<A> a = {lowest<A>(), (A)0};
    for (int k = threadIdx.x; k < splits; k += WAVE) join(a, found[row * splits + k].m, found[row * splits + k].s, c);
#pragma unroll
    for (int o = WAVE / 2; o; o >>= 1) join(a, shfl_xor(a.m, o), shfl_xor(a.s, o), c);
    if (threadIdx.x == 0) finish_row(chosen, a, tau, logps + row, lse + 2 * row);
}

// The gradient: element-wise once the row's maximum and sum are known, so a row is cut into as many parts as fill the chip.
// 16 bytes of it; PAST: by the caches, which a gradient of this size would empty of the logits that are to be read yet
typedef uint32_t uint4_ __attribute__((ext_vector_type(4)));
// (compiled apart: two stores to one place on either side of a branch become one, of the ordinary kind)
template <bool PAST, class T, int N>
__device__ __forceinline__ void put(T* dx, const Pack<T, N>& d) {
    uint4_* const to = (uint4_*)__builtin_assume_aligned(dx, 16);
    if (PAST)
        __builtin_nontemporal_store(*(const uint4_*)&d, to);
    else
        *to = *(const uint4_*)&d;
}
// exp((x - hi)/tau) with c + c_lo = log2(e)/tau.  Of 32-bit logits what the difference and its product round away is made up for:
// of 50 powers of e down, that was 40 roundings of the gradient.  (16-bit gradients round by more than it, and the pass waits for memory.)
template <class T, class A>
__device__ __forceinline__ A power(A x, A hi, A c, A c_lo) {
    const A e = x - hi, p = e * c, v = exp2_of(p);
    if constexpr (sizeof(T) == 4) {
        const A b = e - x, e_lo = (x - (e - b)) - (hi + b);
        const A p_lo = fmaf(e_lo, c, fmaf(e, c_lo, fmaf(e, c, -p)));
        return p > -200 ? fmaf(v, p_lo * 0.69314718f, v) : v;  // (0 beyond, and at -inf, where p_lo is NaN)
    }
    return v;
}
template <bool PAST, class T, int N, class A>
__device__ __forceinline__ void grad_pack(const Pack<T, N>& p, T* dx, int64_t v, int64_t y, A hi, A c, A c_lo, A scale, A at_target) {
    Pack<T, N> d;
#pragma unroll
    for (int k = 0; k < N; k++) d.v[k] = (T)(scale * power<T, A>((A)p.v[k], hi, c, c_lo));
    const uint64_t off = (uint64_t)(y - v);
    if (off < (uint64_t)N) {
#pragma unroll
        for (int k = 0; k < N; k++)
            if ((uint64_t)k == off) d.v[k] = (T)at_target;
    }
    if (N == 1)
        dx[v] = d.v[0];
    else
        put<PAST>(dx + v, d);
}

template <class T, int BLOCK, bool PAST>
__global__ __launch_bounds__(BLOCK) void logprobs_grad_kernel(const T* x, Rows r, double tau, typename Num<T>::acc c, typename Num<T>::acc c_lo, int splits, int64_t part,
                                                              const double* lse, const typename Num<T>::acc* grad, T* dx) {
    typedef typename Num<T>::acc A;
    constexpr int N = vec_len<T>(), U = 4;
    const int tid = threadIdx.x;
    for (int64_t unit = blockIdx.x; unit < r.rows * splits; unit += gridDim.x) {
        // the last rows first: what the forward pass read last is in the caches yet
        const int64_t row = r.rows - 1 - unit / splits, lo = (unit % splits) * part, hi_v = lo + part < r.vocab ? lo + part : r.vocab;
        const int64_t y = r.targets[row];
        const A g = y == r.ignore ? (A)0 : grad[row];
        T* out = dx + row * r.vocab;
        const int64_t lead = (int64_t)((16 - ((uintptr_t)(out + lo) & 15)) & 15) / (int64_t)sizeof(T);
        const int64_t head = lo + lead < hi_v ? lo + lead : hi_v;
        const int64_t packs = (hi_v - head) / N, done = head + packs * N;
        if (g == 0) {  // nothing comes in: the row is not read
            for (int64_t i = tid; i < packs; i += BLOCK) {
                Pack<T, N> z;
#pragma unroll
                for (int k = 0; k < N; k++) z.v[k] = (T)0;
                put<PAST>(out + head + i * N, z);
            }
            for (int64_t k = lo + tid; k < head; k += BLOCK) out[k] = (T)0;
            for (int64_t k = done + tid; k < hi_v; k += BLOCK) out[k] = (T)0;
            continue;
        }
        const T* in = row_at(x, r, row);
        const A hi = (A)lse[2 * row];
        const double l = lse[2 * row + 1];
        const A coef = y >= 0 && y < r.vocab ? (A)((double)g / tau) : (A)NAN;
        const A scale = -coef * (A)exp(-l);
        // 1 - p at the target by its own function: a difference of near numbers otherwise
        A at_target = 0;
        if (y >= lo && y < hi_v) at_target = -coef * (A)expm1(((double)(A)in[y] - (double)hi) / tau - l);
        int64_t i = tid;
        for (; i + (U - 1) * BLOCK < packs; i += U * BLOCK) {
            Pack<T, N> p[U];
#pragma unroll
            for (int u = 0; u < U; u++) p[u] = *(const Pack<T, N>*)(in + head + (i + u * BLOCK) * N);
#pragma unroll
            for (int u = 0; u < U; u++) grad_pack<PAST, T, N, A>(p[u], out, head + (i + u * BLOCK) * N, y, hi, c, c_lo, scale, at_target);
        }
        for (; i < packs; i += BLOCK) grad_pack<PAST, T, N, A>(*(const Pack<T, N>*)(in + head + i * N), out, head + i * N, y, hi, c, c_lo, scale, at_target);
        for (int64_t k = lo + tid; k < head; k += BLOCK) grad_pack<PAST, T, 1, A>({{in[k]}}, out, k, y, hi, c, c_lo, scale, at_target);
        for (int64_t k = done + tid; k < hi_v; k += BLOCK) grad_pack<PAST, T, 1, A>({{in[k]}}, out, k, y, hi, c, c_lo, scale, at_target);
    }
}

// ------------------------------------------------------------------------------------ launches
// A gradient of so many bytes is stored past the caches (half of the last one's 256 MB: a smaller one may be there for whoever reads it
// next).  Forward and gradient of other logits in every pass: 8192 x 32768 in bf16 254 us (294 through the caches), 1020 x 50001 in f32 102 (118).
constexpr double PAST_CACHES = 128e6;
constexpr int64_t MOST_BLOCKS = 1 << 22;  // a launch has less than 2^32 threads: kernels loop beyond

static int64_t elem_size(int dtype) { return dtype == LBFGS_TRAIN_F64 ? 8 : dtype == LBFGS_TRAIN_F32 ? 4 : 2; }

// Workgroups to a row of the forward pass: several, with a second launch to join them, only where few rows are long enough for one
// workgroup to need some 10 us more than that launch.  Measured for 1 and 64 rows, shared and not, in us: 131072 in f64 8.5 and 21
// (39, 47), 131072 in f32 8.1 and 9.4 (9.8, 11.1) and in bf16 8.3 and 8.9 (8.9, 10.5), 32768 in bf16 7.6 and 8.0 (4.1, 5.1).  A
// launch takes 3 us of the host beside.
static int forward_splits(int64_t rows, int64_t vocab, int dtype) {
    const int64_t cost = vocab * (dtype == LBFGS_TRAIN_F64 ? 6 : 1);  // (exponentials of 64 bits)
    if (rows > 128 || cost < 196608) return 1;
    const int64_t want = (512 + rows - 1) / rows, most = vocab * elem_size(dtype) / 16384;
    return (int)(want < most ? want : most);
}
static int64_t part_of(int64_t vocab, int splits) {
    const int64_t each = (vocab + splits - 1) / splits;
    return (each + 7) / 8 * 8;
}

template <class T>
static void launch_forward(const void* x, const Rows& r, double tau, void* logps, double* lse, void* ws, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const A c = (A)(1.4426950408889634 / tau);
    const int dtype = sizeof(T) == 8 ? LBFGS_TRAIN_F64 : sizeof(T) == 4 ? LBFGS_TRAIN_F32 : LBFGS_TRAIN_BF16;
    const int64_t bytes = r.vocab * (int64_t)sizeof(T), grid = r.rows < MOST_BLOCKS ? r.rows : MOST_BLOCKS;
    int splits = forward_splits(r.rows, r.vocab, dtype);
    if (splits > 1) {
        const int64_t part = part_of(r.vocab, splits);
        splits = (int)((r.vocab + part - 1) / part);
        MaxSum<A>* found = (MaxSum<A>*)ws;
        logprobs_part_kernel<T, 256><<<dim3(splits, (unsigned)r.rows), 256, 0, s>>>((const T*)x, r, c, part, found);
        logprobs_join_kernel<T><<<(unsigned)r.rows, WAVE, 0, s>>>((const T*)x, r, tau, c, splits, found, (A*)logps, lse);
        return;
    }
    // Many rows fill the chip with a wave each, few need the whole workgroup.  Measured in bf16 with 64, 256 and 512 threads, in us:
    // 4000 rows of 4000 10.4, 12.2, 19.0, of 8192 14.3, 15.9, 22.7, of 16384 23.6, 24.1, 28.8, of 32768 42.2, 41.3, 41.6, of 131072 184, 179,
    // 175; 64 rows of 1000 3.5, 3.6, 3.7, of 4000 4.5, 3.8, 3.7, of 16384 6.9, 4.4, 4.3, of 32768 10.5, 5.4, 5.1, of 131072 34, 11.2, 10.5.
    const bool many = r.rows >= 1024;
    if (bytes <= (many ? 16384 : 4096))
        logprobs_kernel<T, 64><<<(unsigned)grid, 64, 0, s>>>((const T*)x, r, tau, c, (A*)logps, lse);
    else if (bytes <= (many ? 131072 : 32768))
        logprobs_kernel<T, 256><<<(unsigned)grid, 256, 0, s>>>((const T*)x, r, tau, c, (A*)logps, lse);
    else
        logprobs_kernel<T, 512><<<(unsigned)grid, 512, 0, s>>>((const T*)x, r, tau, c, (A*)logps, lse);
}

template <class T>
static void launch_grad(const void* x, const Rows& r, double tau, const double* lse, const void* grad, void* dx, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const A c = (A)(1.4426950408889634 / tau), c_lo = (A)(1.4426950408889634 / tau - (double)c);
    const int64_t bytes = r.vocab * (int64_t)sizeof(T);
    // Workgroups to a row: so many that there are 512 of 16 KiB at least, or 2048 of 64 KiB.  Measured for one to a row, 512 and 2048 in all,
    // in us: in bf16 64 rows of 131072 16.6, 6.7, 9.8, 1 row 14.5, 3.2, 3.3, 255 rows of 32768 9.3, 6.9, 9.8, 1000 of 8192 6.9, 6.9, 9.8; in
    // f32, forward and gradient, 1020 of 50001 124, 124, 118 (all of them through the caches).
    auto shares = [&](int64_t all, int64_t least) { return std::min(all / r.rows, bytes / least); };
    int64_t splits = std::max<int64_t>({1, shares(512, 16384), shares(2048, 65536)});
    const int64_t part = part_of(r.vocab, (int)splits);
    splits = (r.vocab + part - 1) / part;
    const int64_t units = r.rows * splits;
    const unsigned grid = (unsigned)(units < MOST_BLOCKS ? units : MOST_BLOCKS);
    auto launch = [&](auto kernel, int block) { kernel<<<grid, block, 0, s>>>((const T*)x, r, tau, c, c_lo, (int)splits, part, lse, (const A*)grad, (T*)dx); };
    if (bytes <= 4096)  // (many short rows: no logits worth keeping)
        launch(logprobs_grad_kernel<T, 64, false>, 64);
    else if ((double)r.rows * bytes < PAST_CACHES)
        launch(logprobs_grad_kernel<T, 256, false>, 256);
    else
        launch(logprobs_grad_kernel<T, 256, true>, 256);
}

static int check_rows(const lbfgs_train_rows* q, double temperature, Rows* r, const char* who) {
    if (!q) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: no rows", who);
    if (q->dtype < LBFGS_TRAIN_F64 || q->dtype > LBFGS_TRAIN_F16) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: unknown element type %d", who, q->dtype);
    if (q->outer < 0 || q->inner < 0 || q->vocab < 1 || q->outer > (INT64_MAX >> 20) || q->inner > (INT64_MAX >> 20) || q->vocab > (INT64_MAX >> 20) ||
        (q->inner && q->outer > (INT64_MAX >> 20) / q->inner))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld x %lld rows of %lld logits", who, (long long)q->outer, (long long)q->inner, (long long)q->vocab);
    if (!(temperature > 0) || !std::isfinite(temperature)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: temperature %g is not a positive number", who, temperature);
    if (q->dtype != LBFGS_TRAIN_F64 && !(temperature >= 1e-37 && temperature <= 1e37))  // (its reciprocal is a number of 32 bits)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: temperature %g is out of range: 1e-37 to 1e37 for this element type", who, temperature);
    if (!(temperature >= 1e-300 && temperature <= 1e300)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: temperature %g is out of range: 1e-300 to 1e300", who, temperature);
    *r = {q->outer * q->inner, q->inner, q->outer_stride, q->inner_stride, q->vocab, q->targets, q->ignore_index};
    if (r->rows && (!q->logits || !q->targets)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: logits and targets are needed", who);
    return LBFGS_HIP_OK;
}

}  // namespace lt

using namespace lt;

extern "C" uint64_t lbfgs_train_token_logprobs_workspace(int32_t dtype, int64_t rows, int64_t vocab) {
    if (rows < 1 || vocab < 1 || dtype < LBFGS_TRAIN_F64 || dtype > LBFGS_TRAIN_F16) return 0;
    const int splits = forward_splits(rows, vocab, dtype);
    return splits > 1 ? (uint64_t)rows * splits * (dtype == LBFGS_TRAIN_F64 ? sizeof(MaxSum<double>) : sizeof(MaxSum<float>)) : 0;
}

extern "C" int lbfgs_train_token_logprobs(const lbfgs_train_rows* rows, double temperature, void* logps, double* lse, void* workspace, uint64_t workspace_bytes,
                                          void* stream) {
    const char* who = "lbfgs_train_token_logprobs";
    Rows r;
    if (int rc = check_rows(rows, temperature, &r, who)) return rc;
    if (!r.rows) return LBFGS_HIP_OK;
    if (!logps || !lse) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: logps and lse are needed", who);
    const uint64_t need = lbfgs_train_token_logprobs_workspace(rows->dtype, r.rows, r.vocab);
    if (need && (!workspace || workspace_bytes < need))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    if (need && (uintptr_t)workspace % 256) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: the workspace is not aligned to 256 bytes", who);
    hipStream_t s = (hipStream_t)stream;
    switch (rows->dtype) {
        case LBFGS_TRAIN_F64: launch_forward<double>(rows->logits, r, temperature, logps, lse, workspace, s); break;
        case LBFGS_TRAIN_F32: launch_forward<float>(rows->logits, r, temperature, logps, lse, workspace, s); break;
        case LBFGS_TRAIN_BF16: launch_forward<bf16>(rows->logits, r, temperature, logps, lse, workspace, s); break;
        default: launch_forward<f16>(rows->logits, r, temperature, logps, lse, workspace, s);
    }
    return lt_launched(who);
}

extern "C" int lbfgs_train_token_logprobs_grad(const lbfgs_train_rows* rows, double temperature, const double* lse, const void* grad, void* dlogits, void* stream) {
    const char* who = "lbfgs_train_token_logprobs_grad";
    Rows r;
    if (int rc = check_rows(rows, temperature, &r, who)) return rc;
    if (!r.rows) return LBFGS_HIP_OK;
    if (!lse || !grad || !dlogits) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: lse, grad and dlogits are needed", who);
    hipStream_t s = (hipStream_t)stream;
    switch (rows->dtype) {
        case LBFGS_TRAIN_F64: launch_grad<double>(rows->logits, r, temperature, lse, grad, dlogits, s); break;
        case LBFGS_TRAIN_F32: launch_grad<float>(rows->logits, r, temperature, lse, grad, dlogits, s); break;
        case LBFGS_TRAIN_BF16: launch_grad<bf16>(rows->logits, r, temperature, lse, grad, dlogits, s); break;
        default: launch_grad<f16>(rows->logits, r, temperature, lse, grad, dlogits, s);
    }
    return lt_launched(who);
}
