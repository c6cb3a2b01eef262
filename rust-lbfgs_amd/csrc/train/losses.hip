// rust-lbfgs_amd/csrc/train/losses.hip -- preference and policy losses over the token log-probabilities of many sequences,
// with their gradients.
//
// The sequences are ragged, so tokens -- not sequences -- are dealt to the workgroups: a CHUNK of adjacent tokens each,
// whatever sequences they belong to.  One answer of 100 000 tokens then occupies the chip as well as 10 000 of ten.
// What a chunk finds about its sequences (sums, counts) it leaves as
//     total[s]  for a sequence that lies inside the chunk,
//     tail[w]   for the one that starts in chunk w and goes on,       head[w]  for the one that started before chunk w,
// and whoever needs a sequence's sum adds tail + heads + head in chunk order: no atomics, one order, the same bits always.
// Every sum over tokens is held in 64 bits: the values wanted are differences of sums of thousands of terms.
#include "common.h"

namespace lt {

constexpr int E = 8;             // adjacent tokens of a thread: one 16-byte load of 16-bit values, two of 32
constexpr int BLOCK = 256, CHUNK = BLOCK * E;
constexpr int LOSS_BLOCKS = 1024;   // workgroups of the pass over pairs, each leaving one partial loss
constexpr int COUNT_BLOCKS = 64;    // ... of the pass over sequences of the policy loss
constexpr int POLICY_BLOCKS = 2048; // ... of its pass over tokens

struct Rec {
    double sum;
    int64_t count;
};

// the sequences: offsets [seqs + 1] in 32 or 64 bits, or `longest` tokens each.  Offsets are data of the device that the
// host does not see: they are clamped to the tokens there are, so that a bad one leads to no access out of range, and the
// loss of a call with a bad one is NaN.
struct Seqs {
    const void* offsets;
    int bits;
    int64_t longest, tokens, count;
    const uint8_t* mask;  // NULL: every token of a sequence counts
    __device__ __forceinline__ int64_t raw(int64_t s) const {
        return bits == 0 ? s * longest : bits == 32 ? (int64_t)((const int32_t*)offsets)[s] : ((const int64_t*)offsets)[s];
    }
    __device__ __forceinline__ int64_t at(int64_t s) const {
        const int64_t o = raw(s);
        return o < 0 ? 0 : o > tokens ? tokens : o;
    }
    __device__ __forceinline__ bool good(int64_t s) const { return raw(s) >= 0 && raw(s) <= raw(s + 1) && raw(s + 1) <= tokens; }
    // the sequence of token t: the last that starts at or before it; `count` where there is none
    __device__ __forceinline__ int64_t of(int64_t t) const {
        if (t >= tokens) return count;
        if (bits == 0) return t / longest;
        int64_t lo = -1, hi = count;  // at(lo) <= t < at(hi), taking at(-1) = -inf
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (at(mid) <= t)
                lo = mid;
            else
                hi = mid;
        }
        return lo < 0 ? 0 : lo;
    }
};

struct Space {  // the workspace
    Rec *total, *head, *tail;
    double* slope;       // [seqs] preference: d loss / d token; policy: 1 / tokens of the sequence
    double* loss;        // [LOSS_BLOCKS]
    double* counts;      // [COUNT_BLOCKS][2]: kept tokens, sequences with any (whole numbers below 2^53, or NaN)
    double* sums;        // [POLICY_BLOCKS][3]: loss, KL, clipped
};

// A thread's place in the sequences as it walks its tokens
struct Walk {
    int64_t s, begin, end;
    __device__ __forceinline__ void start(const Seqs& q, int64_t t) {
        s = q.of(t);
        begin = s < q.count ? q.at(s) : INT64_MAX;
        end = s < q.count ? q.at(s + 1) : INT64_MAX;
        if (end <= t && s < q.count) s = q.count, begin = end = INT64_MAX;  // behind the last sequence
    }
    __device__ __forceinline__ bool inside(int64_t t) const { return t >= begin; }
    // past the end of sequence s: the next one that has tokens
    __device__ __forceinline__ void next(const Seqs& q) {
        const int64_t t = end;
        do {
            s++;
        } while (s < q.count && q.at(s + 1) <= t);
        begin = s < q.count ? q.at(s) : INT64_MAX;
        end = s < q.count ? q.at(s + 1) : INT64_MAX;
    }
};

template <class T>
__device__ __forceinline__ void load(const T* p, int64_t t, int64_t n, Pack<T, E>& out) {
    if (t + E <= n)
        out = *(const Pack<T, E>*)(p + t);
    else
#pragma unroll
        for (int k = 0; k < E; k++) out.v[k] = t + k < n ? p[t + k] : (T)0;
}
template <class T>
__device__ __forceinline__ void store(T* p, int64_t t, int64_t n, const Pack<T, E>& in) {
    if (t + E <= n)
        *(Pack<T, E>*)(p + t) = in;
    else
#pragma unroll
        for (int k = 0; k < E; k++)
            if (t + k < n) p[t + k] = in.v[k];
}
__device__ __forceinline__ void load_mask(const Seqs& q, int64_t t, Pack<uint8_t, E>& keep) {
    if (q.mask) {
        load(q.mask, t, q.tokens, keep);
    } else {
#pragma unroll
        for (int k = 0; k < E; k++) keep.v[k] = 1;
    }
}

// Sums of (a - b) and counts over the sequences of chunk w (a NULL: counts alone; b NULL: 0).  A thread adds up its own
// tokens; a scan over the threads that restarts wherever a sequence ends carries the rest.
template <class T>
__device__ __forceinline__ void chunk_sums(const Seqs& q, const T* a, const T* b, int64_t w, const Space& sp) {
    __shared__ double wave_sum_[BLOCK / WAVE];
    __shared__ int wave_count_[BLOCK / WAVE], wave_closed_[BLOCK / WAVE];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int64_t chunk = w * CHUNK, t0 = chunk + tid * E;
    Walk at;
    at.start(q, t0);
    Pack<T, E> x, y;
    Pack<uint8_t, E> keep;
    load_mask(q, t0, keep);
    if (a) load(a, t0, q.tokens, x);
    if (b) load(b, t0, q.tokens, y);
    double sum = 0, first_sum = 0;
    int count = 0, first_count = 0;
    int64_t first = -1, first_begin = 0;  // the first sequence that ends among this thread's tokens
#pragma unroll
    for (int k = 0; k < E; k++) {
        const int64_t t = t0 + k;
        if (t < q.tokens) {
            if (at.inside(t) && keep.v[k]) {  // (what is masked is not looked at: it may be anything)
                if (a) sum += b ? (double)x.v[k] - (double)y.v[k] : (double)x.v[k];
                count++;
            }
            if (t + 1 == at.end) {
                if (first < 0)
                    first = at.s, first_begin = at.begin, first_sum = sum, first_count = count;
                else
                    sp.total[at.s] = {sum, count};
                sum = 0, count = 0;
                at.next(q);
            }
        }
    }
    // inclusive scan of (closed, sum, count): (c1, v1) + (c2, v2) = (c1 | c2, c2 ? v2 : v1 + v2)
    double run = sum;
    int run_count = count, closed = first >= 0;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const double v = __shfl_up(run, o, WAVE);
        const int n = __shfl_up(run_count, o, WAVE), c = __shfl_up(closed, o, WAVE);
        if (lane >= o) {
            if (!closed) run += v, run_count += n;
            closed |= c;
        }
    }
    if (lane == WAVE - 1) wave_sum_[wave] = run, wave_count_[wave] = run_count, wave_closed_[wave] = closed;
    // what comes in from the lane before
    double in = __shfl_up(run, 1, WAVE);
    int in_count = __shfl_up(run_count, 1, WAVE), in_closed = __shfl_up(closed, 1, WAVE);
    if (lane == 0) in = 0, in_count = 0, in_closed = 0;
    __syncthreads();
    double before = 0;  // ... and from the waves before
    int before_count = 0;
    for (int k = 0; k < wave; k++) {
        before = wave_closed_[k] ? wave_sum_[k] : before + wave_sum_[k];
        before_count = wave_closed_[k] ? wave_count_[k] : before_count + wave_count_[k];
    }
    if (!in_closed) in += before, in_count += before_count;
    if (first >= 0) {
        const Rec r = {in + first_sum, in_count + first_count};
        if (first_begin >= chunk)
            sp.total[first] = r;
        else
            sp.head[w] = r;
    }
    if (tid == BLOCK - 1 && at.s < q.count && at.begin < chunk + CHUNK) {  // goes on behind the chunk
        Rec r = {sum, count};
        if (first < 0) r.sum += in, r.count += in_count;
        if (at.begin >= chunk)
            sp.tail[w] = r;
        else
            sp.head[w] = r;
    }
    __syncthreads();  // the shared words are written again by the next chunk
}

// the whole of sequence s, by GROUP adjacent lanes; every one of them gets it
template <int GROUP>
__device__ __forceinline__ Rec sequence(const Seqs& q, const Space& sp, int64_t s, int l) {
    const int64_t begin = q.at(s), end = q.at(s + 1);
    Rec r = {0, 0};
    if (end > begin) {
        const int64_t w0 = begin / CHUNK, w1 = (end - 1) / CHUNK;
        if (w0 == w1) {
            if (l == 0) r = sp.total[s];
        } else {
            if (l == 0) r = sp.tail[w0];
            for (int64_t w = w0 + 1 + l; w <= w1; w += GROUP) r.sum += sp.head[w].sum, r.count += sp.head[w].count;
        }
    }
#pragma unroll
    for (int o = GROUP / 2; o; o >>= 1) r.sum += shfl_xor(r.sum, o), r.count += shfl_xor(r.count, o);
    return r;
}

__device__ __forceinline__ double block_sum(double v) {  // valid in thread 0
    __shared__ double part[BLOCK / WAVE];
    v = wave_sum(v);
    if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = v;
    __syncthreads();
    double s = 0;
    for (int k = 0; k < BLOCK / WAVE; k++) s += part[k];
    __syncthreads();
    return s;
}

// ------------------------------------------------------------------------------------ preference
struct Preference {
    double beta, smoothing;
    int kind, normalize;
};

// Pair i compares sequence i with sequence i + pairs.  In terms of the difference D of the two sums, h = beta D:
//   logistic  -(1-e) log sig(h) - e log sig(-h)      d/dD = beta (e - sig(-h))
//   hinge     max(0, 1 - h)                          d/dD = -beta where h < 1
//   squared   (D - 1/(2 beta))^2                     d/dD = 2 (D - 1/(2 beta))
template <class A>
__device__ __forceinline__ void pair_losses(const Seqs& q, const Preference& o, const Space& sp, A* rewards, int block, int blocks) {
    constexpr int GROUP = 8;
    const int64_t pairs = q.count / 2;
    const int l = threadIdx.x % GROUP;
    const int64_t rounds = (pairs + (int64_t)blocks * (BLOCK / GROUP) - 1) / ((int64_t)blocks * (BLOCK / GROUP));
    double total = 0;
    for (int64_t k = 0; k < rounds; k++) {  // (every lane goes through the shuffles of sequence())
        const int64_t i = (k * blocks + block) * (BLOCK / GROUP) + threadIdx.x / GROUP;
        const bool real = i < pairs;
        const Rec c = sequence<GROUP>(q, sp, real ? i : 0, l), r = sequence<GROUP>(q, sp, real ? i + pairs : 0, l);
        if (real && l == 0) {
            const double nc = o.normalize && c.count ? 1.0 / (double)c.count : 1.0, nr = o.normalize && r.count ? 1.0 / (double)r.count : 1.0;
            const double dc = c.sum * nc, dr = r.sum * nr, D = q.good(i) && q.good(i + pairs) ? dc - dr : NAN, h = o.beta * D;
            double loss, slope;
            if (o.kind == LBFGS_TRAIN_LOGISTIC) {
                const double soft = log1p(exp(-fabs(h)));
                loss = (1 - o.smoothing) * (soft + (h < 0 ? -h : 0)) + (o.smoothing != 0 ? o.smoothing * (soft + (h > 0 ? h : 0)) : 0);
                if (h != h) loss = h;
                slope = o.beta * (o.smoothing - 1.0 / (1.0 + exp(h)));
            } else if (o.kind == LBFGS_TRAIN_HINGE) {
                loss = h > 1 ? 0 : 1 - h;
                slope = h < 1 ? -o.beta : h != h ? h : 0;
            } else {
                const double e = D - 0.5 / o.beta;
                loss = e * e;
                slope = 2 * e;
            }
            total += loss;
            slope /= (double)pairs;
            sp.slope[i] = slope * nc;
            sp.slope[i + pairs] = -slope * nr;
            rewards[i] = (A)(o.beta * dc);
            rewards[i + pairs] = (A)(o.beta * dr);
        }
    }
    total = block_sum(total);
    if (threadIdx.x == 0) sp.loss[block] = total;
}

// gradient of chunk w: its sequence's slope at each token that counts, 0 at all others
template <class T>
__device__ __forceinline__ void chunk_slopes(const Seqs& q, const Space& sp, T* grad, int64_t w) {
    const int64_t t0 = w * CHUNK + threadIdx.x * E;
    if (t0 >= q.tokens) return;
    Walk at;
    at.start(q, t0);
    Pack<uint8_t, E> keep;
    load_mask(q, t0, keep);
    Pack<T, E> g;
    typename Num<T>::acc slope = at.s < q.count ? (typename Num<T>::acc)sp.slope[at.s] : 0;
#pragma unroll
    for (int k = 0; k < E; k++) {
        const int64_t t = t0 + k;
        g.v[k] = at.inside(t) && keep.v[k] ? (T)slope : (T)0;
        if (t + 1 == at.end) {
            at.next(q);
            if (k + 1 < E) slope = at.s < q.count ? (typename Num<T>::acc)sp.slope[at.s] : 0;
        }
    }
    store(grad, t0, q.tokens, g);
}

template <class A>
__device__ __forceinline__ void mean_loss(const Space& sp, int blocks, int64_t pairs, A* f) {
    double v = 0;
    for (int k = threadIdx.x; k < blocks; k += BLOCK) v += sp.loss[k];
    v = block_sum(v);
    if (threadIdx.x == 0) *f = (A)(v / (double)pairs);
}

template <class T>
__global__ __launch_bounds__(BLOCK) void sums_kernel(Seqs q, const T* a, const T* b, int64_t chunks, Space sp) {
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) chunk_sums(q, a, b, w, sp);
}
template <class A>
__global__ __launch_bounds__(BLOCK) void pairs_kernel(Seqs q, Preference o, Space sp, A* rewards) {
    pair_losses(q, o, sp, rewards, blockIdx.x, gridDim.x);
}
template <class T>
__global__ __launch_bounds__(BLOCK) void slopes_kernel(Seqs q, int64_t chunks, int blocks, Space sp, typename Num<T>::acc* f, T* grad) {
    if (blockIdx.x == 0) mean_loss(sp, blocks, q.count / 2, f);
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) chunk_slopes(q, sp, grad, w);
}
// a small batch: the three passes as one workgroup, so that one launch is all that is waited for
template <class T>
__global__ __launch_bounds__(BLOCK) void preference_small_kernel(Seqs q, Preference o, const T* a, const T* b, int64_t chunks, Space sp,
                                                                 typename Num<T>::acc* f, typename Num<T>::acc* rewards, T* grad) {
    for (int64_t w = 0; w < chunks; w++) chunk_sums(q, a, b, w, sp);
    __syncthreads();
    pair_losses(q, o, sp, rewards, 0, 1);
    __syncthreads();
    mean_loss(sp, 1, q.count / 2, f);
    for (int64_t w = 0; w < chunks; w++) chunk_slopes(q, sp, grad, w);
}

// ------------------------------------------------------------------------------------ policy
struct Policy {
    double low, high, log_low, log_high, kl;  // 1 - clip_low, 1 + clip_high and their logarithms, the KL term's weight
    int per_token, by_sequence;
};

// e^q - 1 and e^q - 1 - q without their cancellation
__device__ __forceinline__ void kl_terms(float q, float& em1, float& k) {
    if (fabsf(q) < 0.5f) {  // q^2 (1/2 + q/6 + ...): the first term left out is below 2^-24 of the sum
        k = q * q * (0.5f + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720 + q * (1.f / 5040 + q * (1.f / 40320)))))));
        em1 = q + k;
    } else {
        em1 = expf(q) - 1.f;
        k = em1 - q;
    }
}
__device__ __forceinline__ void kl_terms(double q, double& em1, double& k) {
    em1 = expm1(q);
    k = em1 - q;
}

// tokens of each sequence that count -> 1 / their number; kept tokens and sequences with any of this workgroup
__device__ __forceinline__ void sequence_weights(const Seqs& q, const Space& sp, int block, int blocks) {
    constexpr int GROUP = 8;
    const int l = threadIdx.x % GROUP;
    const int64_t each = (int64_t)blocks * (BLOCK / GROUP), rounds = (q.count + each - 1) / each;
    double kept = 0, some = 0;
    for (int64_t k = 0; k < rounds; k++) {
        const int64_t s = (k * blocks + block) * (BLOCK / GROUP) + threadIdx.x / GROUP;
        int64_t n;
        if (q.mask) {
            n = sequence<GROUP>(q, sp, s < q.count ? s : 0, l).count;
        } else {
            n = q.at(s < q.count ? s + 1 : 1) - q.at(s < q.count ? s : 0);
            if (n < 0) n = 0;
        }
        if (s < q.count && l == 0) {
            sp.slope[s] = n ? 1.0 / (double)n : 0;
            kept += q.good(s) ? (double)n : NAN;
            some += q.good(s) ? (n > 0 ? 1.0 : 0.0) : NAN;
        }
    }
    kept = block_sum(kept);
    some = block_sum(some);
    if (threadIdx.x == 0) sp.counts[2 * block] = kept, sp.counts[2 * block + 1] = some;
}

// the sum of both counts over the workgroups of sequence_weights (at most a wave of them), in every thread
__device__ __forceinline__ void all_counts(const Space& sp, int blocks, double& kept, double& some) {
    const int lane = threadIdx.x % WAVE;
    kept = wave_sum(lane < blocks ? sp.counts[2 * lane] : 0.0);
    some = wave_sum(lane < blocks ? sp.counts[2 * lane + 1] : 0.0);
    if (kept < 1) kept = 1;  // nothing counts: sums of nothing, divided by something
    if (some < 1) some = 1;
}

template <class T>
struct PolicyData {
    const T *logps, *old, *ref, *adv;
    T* grad;
};

// L = -min(r A, clip(r) A) + kl (e^q - 1 - q) with r = e^d, d = logp - old, q = ref - logp.  d is the exact difference, and
// whether r is clipped is decided by comparing d with the borders' logarithms in 64 bits: the gradient jumps there.  r is
// taken in 64 bits too: advantages have mean 0, and the mean of r A is what is left of terms a thousand times larger.
template <class T>
__device__ __forceinline__ void chunk_policy(const Seqs& q, const Policy& o, const PolicyData<T>& x, const Space& sp, double inv, int64_t w,
                                             double& f, double& kl, double& clipped) {
    typedef typename Num<T>::acc A;
    const int64_t t0 = w * CHUNK + threadIdx.x * E, n = q.tokens;
    if (t0 >= n) return;
    Pack<T, E> lp, old, ref, adv, g;
    Pack<uint8_t, E> keep;
    load(x.logps, t0, n, lp);
    load(x.old, t0, n, old);
    if (x.ref) load(x.ref, t0, n, ref);
    if (o.per_token) load(x.adv, t0, n, adv);
    load_mask(q, t0, keep);
    Walk at;
    at.start(q, t0);
    double a_seq = 0;
    double weight = inv;
    auto enter = [&]() {
        if (at.s < q.count) {
            if (!o.per_token) a_seq = (double)x.adv[at.s];
            if (o.by_sequence) weight = inv * sp.slope[at.s];
        }
    };
    enter();
#pragma unroll
    for (int k = 0; k < E; k++) {
        const int64_t t = t0 + k;
        A slope = 0;
        if (at.inside(t) && keep.v[k]) {
            const double d = (double)lp.v[k] - (double)old.v[k];
            const double a = o.per_token ? (double)adv.v[k] : a_seq;
            const bool over = (a > 0 && d > o.log_high) || (a < 0 && d < o.log_low);
            // (an advantage of 0 gives 0 for any ratio, one that overflowed too)
            const double ra = a == 0 && d == d ? 0 : exp(d) * a;
            double loss = over ? -(a > 0 ? o.high : o.low) * a : -ra;
            slope = over ? (A)0 : (A)-ra;
            if (o.kl != 0) {
                A em1, term;
                kl_terms((A)((double)ref.v[k] - (double)lp.v[k]), em1, term);
                loss += o.kl * (double)term;
                slope -= (A)o.kl * em1;
                kl += (double)term;
            }
            f += loss * weight;
            clipped += over;
            slope *= (A)weight;
        }
        g.v[k] = (T)slope;
        if (t + 1 == at.end) {
            at.next(q);
            if (k + 1 < E) enter();
        }
    }
    store(x.grad, t0, n, g);
}

template <class A>
__device__ __forceinline__ void policy_results(double f, double kl, double clipped, double kept, A* out_f, A* out_kl, A* out_clipped) {
    f = block_sum(f);
    kl = block_sum(kl);
    clipped = block_sum(clipped);
    if (threadIdx.x == 0) *out_f = (A)(kept == kept ? f : kept), *out_kl = (A)(kl / kept), *out_clipped = (A)(clipped / kept);
}

__global__ __launch_bounds__(BLOCK) void weights_kernel(Seqs q, Space sp) { sequence_weights(q, sp, blockIdx.x, gridDim.x); }
template <class T>
__global__ __launch_bounds__(BLOCK) void policy_kernel(Seqs q, Policy o, PolicyData<T> x, int64_t chunks, int count_blocks, Space sp) {
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, count_blocks, kept, some);
    const double inv = 1.0 / (o.by_sequence ? some : kept);
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) chunk_policy(q, o, x, sp, inv, w, f, kl, clipped);
    f = block_sum(f);
    kl = block_sum(kl);
    clipped = block_sum(clipped);
    if (threadIdx.x == 0) sp.sums[3 * blockIdx.x] = f, sp.sums[3 * blockIdx.x + 1] = kl, sp.sums[3 * blockIdx.x + 2] = clipped;
}
template <class A>
__global__ __launch_bounds__(BLOCK) void policy_results_kernel(Space sp, int count_blocks, int blocks, A* out_f, A* out_kl, A* out_clipped) {
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, count_blocks, kept, some);
    for (int k = threadIdx.x; k < blocks; k += BLOCK) f += sp.sums[3 * k], kl += sp.sums[3 * k + 1], clipped += sp.sums[3 * k + 2];
    policy_results(f, kl, clipped, kept, out_f, out_kl, out_clipped);
}
template <class T>
__global__ __launch_bounds__(BLOCK) void policy_small_kernel(Seqs q, Policy o, PolicyData<T> x, int64_t chunks, Space sp, typename Num<T>::acc* out_f,
                                                             typename Num<T>::acc* out_kl, typename Num<T>::acc* out_clipped) {
    if (q.mask)
        for (int64_t w = 0; w < chunks; w++) chunk_sums<T>(q, nullptr, nullptr, w, sp);
    __syncthreads();
    sequence_weights(q, sp, 0, 1);
    __syncthreads();
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, 1, kept, some);
    const double inv = 1.0 / (o.by_sequence ? some : kept);
    for (int64_t w = 0; w < chunks; w++) chunk_policy(q, o, x, sp, inv, w, f, kl, clipped);
    policy_results(f, kl, clipped, kept, out_f, out_kl, out_clipped);
}

// ------------------------------------------------------------------------------------ launches
// up to so many tokens and sequences one workgroup does the whole of a loss
constexpr int64_t SMALL_TOKENS = 2 * CHUNK, SMALL_SEQS = 256;

static int64_t chunks_of(int64_t tokens) { return (tokens + CHUNK - 1) / CHUNK; }

static uint64_t lay_out(Space* sp, void* base, int64_t tokens, int64_t seqs) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        void* p = (char*)base + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    const uint64_t chunks = (uint64_t)chunks_of(tokens);
    Space s;
    s.total = (Rec*)take((uint64_t)seqs * sizeof(Rec));
    s.head = (Rec*)take(chunks * sizeof(Rec));
    s.tail = (Rec*)take(chunks * sizeof(Rec));
    s.slope = (double*)take((uint64_t)seqs * sizeof(double));
    s.loss = (double*)take(LOSS_BLOCKS * sizeof(double));
    s.counts = (double*)take(COUNT_BLOCKS * 2 * sizeof(double));
    s.sums = (double*)take(POLICY_BLOCKS * 3 * sizeof(double));
    if (sp) *sp = s;
    return at;
}

template <class T>
static void launch_preference(const Seqs& q, const Preference& o, const void* a, const void* b, void* f, void* rewards, void* grad, const Space& sp, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const int64_t chunks = chunks_of(q.tokens), pairs = q.count / 2;
    if (q.tokens <= SMALL_TOKENS && q.count <= SMALL_SEQS) {
        preference_small_kernel<T><<<1, BLOCK, 0, s>>>(q, o, (const T*)a, (const T*)b, chunks, sp, (A*)f, (A*)rewards, (T*)grad);
        return;
    }
    const int64_t groups = (pairs * 8 + BLOCK - 1) / BLOCK;
    const int blocks = (int)(groups < LOSS_BLOCKS ? groups : LOSS_BLOCKS);
    const unsigned grid = (unsigned)(chunks < (1 << 20) ? (chunks ? chunks : 1) : (1 << 20));
    if (chunks) sums_kernel<T><<<grid, BLOCK, 0, s>>>(q, (const T*)a, (const T*)b, chunks, sp);
    pairs_kernel<A><<<blocks, BLOCK, 0, s>>>(q, o, sp, (A*)rewards);
    slopes_kernel<T><<<grid, BLOCK, 0, s>>>(q, chunks, blocks, sp, (A*)f, (T*)grad);
}

template <class T>
static void launch_policy(const Seqs& q, const Policy& o, const void* logps, const void* old, const void* ref, const void* adv, void* f, void* kl,
                          void* clipped, void* grad, const Space& sp, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const int64_t chunks = chunks_of(q.tokens);
    const PolicyData<T> x = {(const T*)logps, (const T*)old, (const T*)ref, (const T*)adv, (T*)grad};
    if (q.tokens <= SMALL_TOKENS && q.count <= SMALL_SEQS) {
        policy_small_kernel<T><<<1, BLOCK, 0, s>>>(q, o, x, chunks, sp, (A*)f, (A*)kl, (A*)clipped);
        return;
    }
    const int64_t groups = (q.count * 8 + BLOCK - 1) / BLOCK;
    const int count_blocks = (int)(groups < COUNT_BLOCKS ? groups : COUNT_BLOCKS);
    const int blocks = (int)(chunks < POLICY_BLOCKS ? (chunks ? chunks : 1) : POLICY_BLOCKS);
    if (q.mask && chunks) sums_kernel<T><<<(unsigned)(chunks < (1 << 20) ? chunks : (1 << 20)), BLOCK, 0, s>>>(q, (const T*)nullptr, (const T*)nullptr, chunks, sp);
    weights_kernel<<<count_blocks, BLOCK, 0, s>>>(q, sp);
    policy_kernel<T><<<blocks, BLOCK, 0, s>>>(q, o, x, chunks, count_blocks, sp);
    policy_results_kernel<A><<<1, BLOCK, 0, s>>>(sp, count_blocks, blocks, (A*)f, (A*)kl, (A*)clipped);
}

static int check_seqs(const lbfgs_train_sequences* in, Seqs* q, const char* who) {
    if (!in) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: no sequences", who);
    if (in->dtype < LBFGS_TRAIN_F64 || in->dtype > LBFGS_TRAIN_F16) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: unknown element type %d", who, in->dtype);
    if (in->tokens < 0 || in->count < 1 || in->tokens > (INT64_MAX >> 20) || in->count > (INT64_MAX >> 20))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld tokens in %lld sequences", who, (long long)in->tokens, (long long)in->count);
    if (in->offsets) {
        if (in->offset_bits != 32 && in->offset_bits != 64) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: offsets of %d bits", who, in->offset_bits);
    } else if (in->tokens % in->count) {
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld tokens are no padded batch of %lld sequences, and there are no offsets", who, (long long)in->tokens, (long long)in->count);
    }
    *q = {in->offsets, in->offsets ? in->offset_bits : 0, in->offsets ? 0 : in->tokens / in->count, in->tokens, in->count, in->mask};
    if (!in->offsets && !in->tokens) q->longest = 0;
    return LBFGS_HIP_OK;
}
static int check_workspace(const void* workspace, uint64_t bytes, const Seqs& q, Space* sp, const char* who) {
    const uint64_t need = lay_out(nullptr, nullptr, q.tokens, q.count);
    if (!workspace || bytes < need)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? bytes : 0), (unsigned long long)need);
    lay_out(sp, (void*)workspace, q.tokens, q.count);
    return LBFGS_HIP_OK;
}

static thread_local char g_error[512];

}  // namespace lt

using namespace lt;

int lt_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return code;
}
int lt_launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? LBFGS_HIP_OK : lt_fail(LBFGS_HIP_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

#ifndef LBFGS_TRAIN_BUILD_ID
#define LBFGS_TRAIN_BUILD_ID "unstamped"
#endif
extern "C" int lbfgs_train_abi_version(void) { return LBFGS_TRAIN_ABI_VERSION; }
extern "C" const char* lbfgs_train_build_id(void) {
    static const char id[] = "LBFGS_TRAIN_BUILD_ID=" LBFGS_TRAIN_BUILD_ID;
    return id + sizeof("LBFGS_TRAIN_BUILD_ID=") - 1;
}
extern "C" const char* lbfgs_train_last_error(void) { return g_error; }

extern "C" uint64_t lbfgs_train_sequences_workspace(int64_t tokens, int64_t count) {
    if (tokens < 0 || count < 1 || tokens > (INT64_MAX >> 20) || count > (INT64_MAX >> 20)) return 0;
    return lay_out(nullptr, nullptr, tokens, count);
}

extern "C" int lbfgs_train_preference(const lbfgs_train_sequences* seqs, const void* logps, const void* ref_logps, double beta, double label_smoothing,
                                      int32_t kind, int32_t normalize_lengths, void* f, void* rewards, void* grad, void* workspace, uint64_t workspace_bytes,
                                      void* stream) {
    const char* who = "lbfgs_train_preference";
    Seqs q;
    Space sp;
    if (int rc = check_seqs(seqs, &q, who)) return rc;
    if (q.count % 2) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %lld sequences are no pairs", who, (long long)q.count);
    if (!(beta > 0) || !std::isfinite(beta)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: beta %g is not a positive number", who, beta);
    if (!(label_smoothing >= 0 && label_smoothing < 0.5)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: label_smoothing %g is not in [0, 0.5)", who, label_smoothing);
    if (kind < LBFGS_TRAIN_LOGISTIC || kind > LBFGS_TRAIN_SQUARED) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: unknown kind %d", who, kind);
    if (label_smoothing != 0 && kind != LBFGS_TRAIN_LOGISTIC) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: label_smoothing goes with the logistic kind", who);
    if (!f || !rewards || (q.tokens && (!logps || !grad))) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: logps, f, rewards and grad are needed", who);
    if (int rc = check_workspace(workspace, workspace_bytes, q, &sp, who)) return rc;
    const Preference o = {beta, label_smoothing, kind, normalize_lengths != 0};
    hipStream_t s = (hipStream_t)stream;
    switch (seqs->dtype) {
        case LBFGS_TRAIN_F64: launch_preference<double>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_F32: launch_preference<float>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_BF16: launch_preference<bf16>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        default: launch_preference<f16>(q, o, logps, ref_logps, f, rewards, grad, sp, s);
    }
    return lt_launched(who);
}

extern "C" int lbfgs_train_policy(const lbfgs_train_sequences* seqs, const void* logps, const void* old_logps, const void* ref_logps, const void* advantages,
                                  int32_t per_token, double clip_low, double clip_high, double kl_coef, int32_t by_sequence, void* f, void* kl,
                                  void* clip_fraction, void* grad, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* who = "lbfgs_train_policy";
    Seqs q;
    Space sp;
    if (int rc = check_seqs(seqs, &q, who)) return rc;
    if (!(clip_low >= 0 && clip_low <= 1)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: clip_low %g is not in [0, 1]", who, clip_low);
    if (!(clip_high >= 0)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: clip_high %g is negative", who, clip_high);
    if (!std::isfinite(kl_coef)) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: kl_coef %g is not a number", who, kl_coef);
    if (kl_coef != 0 && !ref_logps && q.tokens) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: a KL term needs ref_logps", who);
    if (!f || !kl || !clip_fraction || ((q.tokens || !per_token) && !advantages) || (q.tokens && (!logps || !old_logps || !grad)))
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: logps, old_logps, advantages, f, kl, clip_fraction and grad are needed", who);
    if (int rc = check_workspace(workspace, workspace_bytes, q, &sp, who)) return rc;
    const Policy o = {1 - clip_low, 1 + clip_high, std::log1p(-clip_low), std::log1p(clip_high), kl_coef, per_token != 0, by_sequence != 0};
    if (kl_coef == 0) ref_logps = nullptr;
    hipStream_t s = (hipStream_t)stream;
    switch (seqs->dtype) {
        case LBFGS_TRAIN_F64: launch_policy<double>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_F32: launch_policy<float>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_BF16: launch_policy<bf16>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        default: launch_policy<f16>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s);
    }
    return lt_launched(who);
}
