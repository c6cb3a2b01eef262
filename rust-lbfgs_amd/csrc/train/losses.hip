// rust-lbfgs_amd/csrc/train/losses.hip -- preference and policy losses over the token log-probabilities of many sequences,
// with their gradients.
//
// The sequences are ragged, so tokens -- not sequences -- are dealt to the workgroups: a CHUNK of adjacent tokens each,
// whatever sequences they belong to.  One answer of 100 000 tokens then occupies the chip as well as 10 000 of ten.  (Its chunks' records are
// added up by one lane or by eight, by the mean length: one of 2 million among 1000 of 20 takes 85 us where 1000 of 2000 take 20.)
// What a chunk finds about its sequences (sums, counts) it leaves as
//     total[s]  for a sequence that lies inside the chunk,
//     tail[w]   for the one that starts in chunk w and goes on,       head[w]  for the one that started before chunk w,
// and whoever needs a sequence's sum adds tail + heads + head in chunk order: no atomics, one order, the same bits always.
// Every sum over tokens is held in 64 bits: the values wanted are differences of sums of thousands of terms.
//
// Large batches are bound by HBM, all others by launches and by how few loads wait for each other.  Measured in 32 bits: policy,
// 8.4 million tokens, a reference and a mask: 7 us to count, 36 for losses and gradients (4.9 TB/s), 5 for the results -- by sequences 17, 52
// (two exponentials of 64 bits a token, and the search) and 10 --; preference,
// 48 sequences of up to 131072 tokens: sums 8 us (3.7 TB/s), slopes, loss and gradient 15; 512 of up to 2047: 5 and 6 us.
#include "common.h"

namespace lt {

constexpr int E = 8;             // adjacent tokens of a thread: one 16-byte load of 16-bit values, two of 32
constexpr int BLOCK = 256, CHUNK = BLOCK * E;
constexpr int LOSS_BLOCKS = 1024;   // workgroups of the pass over pairs, each leaving one partial loss
constexpr int COUNT_BLOCKS = 256;   // ... of the pass of the policy loss that counts
constexpr int POLICY_BLOCKS = 2048; // ... of its pass over tokens
constexpr int FAR = 1 << 30;        // a distance in tokens beyond every chunk

struct Rec {
    double sum;
    int64_t count;
};

// Where a thread is in the sequences: number s, and the distances of its first and behind its last token from the thread's own
// first one (FAR where there is none; a sequence that started long ago: some negative number)
struct Spot {
    int64_t s;
    int begin, end;
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
    __device__ __forceinline__ static int distance(int64_t d) { return d > FAR ? FAR : d < -FAR ? -FAR : (int)d; }

    // The sequence of the thread's first token t (of its wave's: t - lane * E): the last that starts at or before it.  A whole
    // wave looks for its first token's, 64 offsets a round, and then has the next 64 offsets in its lanes: one to three rounds
    // of loads that wait for each other where a search of each thread's own had twelve.
    __device__ __forceinline__ Spot locate(int64_t t) const {
        if (bits == 0) {
            if (t >= tokens) return {count, FAR, FAR};
            const int64_t s = tokens < (int64_t)1 << 32 ? (int64_t)((uint32_t)t / (uint32_t)longest) : t / longest;
            return {s, distance(s * longest - t), distance((s + 1) * longest - t)};
        }
        const int lane = threadIdx.x % WAVE;
        const int64_t first = t - lane * E;
        int64_t lo = -1, hi = count;  // at(lo) <= first < at(hi), at(-1) being -inf
        while (hi - lo > WAVE) {
            const int64_t step = (hi - lo + WAVE - 1) / WAVE, probe = lo + step * (lane + 1);
            const int n = __popcll(__ballot(probe < hi && at(probe) <= first));
            lo += step * n;
            if (lo + step < hi) hi = lo + step;
        }
        const int64_t here = lo + 1 + lane;
        const int64_t value = here <= count ? at(here) : INT64_MAX;
        const int past = __popcll(__ballot(here < hi && value <= first));
        // the offsets that follow the first token, from these as far as they reach
        const int known = value == INT64_MAX ? FAR : distance(value - first);
        int next = __shfl(known, (lane + past) % WAVE, WAVE);
        int start = __shfl(known, past ? past - 1 : 0, WAVE);
        if (past == 0) start = lo >= 0 ? distance(at(lo) - first) : 0;
        lo += past;
        if (lane + past >= WAVE) next = lo + 1 + lane <= count ? distance(at(lo + 1 + lane) - first) : FAR;
        const int own = lane * E;
        int n = 0;  // how many of them are at or before t
#pragma unroll
        for (int o = WAVE / 2; o; o >>= 1)
            if (__shfl(next, n + o - 1, WAVE) <= own) n += o;
        const bool beyond = n == WAVE - 1 && __shfl(next, WAVE - 1, WAVE) <= own;
        const int before = __shfl(next, n ? n - 1 : 0, WAVE), after = __shfl(next, n, WAVE), second = __shfl(next, 1, WAVE);
        int64_t s = lo + n;
        int begin = n ? before : start, end = after;
        if (beyond) {  // more than 64 sequences begin among the tokens of a wave: a search of the thread's own
            int64_t h = count;
            s = lo + WAVE;
            while (h - s > 1) {
                const int64_t mid = (s + h) >> 1;
                if (at(mid) <= t)
                    s = mid;
                else
                    h = mid;
            }
            begin = distance(at(s) - first), end = s < count ? distance(at(s + 1) - first) : FAR;
        }
        if (s < 0) s = 0, begin = after, end = second;  // before the first sequence
        if (s >= count || (end != FAR && end <= own)) return {count, FAR, FAR};
        return {s, begin - own, end == FAR ? FAR : end - own};
    }
    // behind sequence at.s, which ends at `t + at.end`: the next one that has tokens
    __device__ __forceinline__ void next(Spot& at_, int64_t t) const {
        const int64_t from = t + at_.end;
        int64_t s = at_.s;
        do {
            s++;
        } while (s < count && at(s + 1) <= from);
        at_ = s < count ? Spot{s, distance(at(s) - t), distance(at(s + 1) - t)} : Spot{count, FAR, FAR};
    }
};

// The same of a small batch, its offsets in LDS
constexpr int SMALL_CHUNKS = 2, SMALL_TOKENS = SMALL_CHUNKS * CHUNK, SMALL_SEQS = 256;
struct SmallSeqs {
    const int* offsets;          // clamped
    const uint8_t* fine;         // good()
    int64_t tokens, count;
    const uint8_t* mask;
    __device__ __forceinline__ int64_t at(int64_t s) const { return offsets[s]; }
    __device__ __forceinline__ bool good(int64_t s) const { return fine[s]; }
    __device__ __forceinline__ Spot locate(int64_t t) const {
        int lo = -1, hi = (int)count;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (offsets[mid] <= t)
                lo = mid;
            else
                hi = mid;
        }
        if (lo < 0) lo = 0;
        if (offsets[lo + 1] <= t) return {count, FAR, FAR};
        return {lo, offsets[lo] - (int)t, offsets[lo + 1] - (int)t};
    }
    __device__ __forceinline__ void next(Spot& at_, int64_t t) const {
        const int from = (int)t + at_.end;
        int s = (int)at_.s;
        do {
            s++;
        } while (s < count && offsets[s + 1] <= from);
        at_ = s < count ? Spot{s, offsets[s] - (int)t, offsets[s + 1] - (int)t} : Spot{count, FAR, FAR};
    }
};
struct SmallSpace {
    int offsets[SMALL_SEQS + 1];
    uint8_t fine[SMALL_SEQS];
    Rec total[SMALL_SEQS], head[SMALL_CHUNKS], tail[SMALL_CHUNKS];
    double slope[SMALL_SEQS], loss[1], counts[2];
};

struct Space {  // the workspace
    Rec *total, *head, *tail;
    double* slope;       // [seqs] preference: d loss / d token; policy: 1 / tokens of the sequence
    double* loss;        // [LOSS_BLOCKS]
    double* counts;      // [COUNT_BLOCKS][2]: kept tokens, sequences with any (whole numbers below 2^53, or NaN)
    double* sums;        // [POLICY_BLOCKS][3]: loss, KL, clipped
};

__device__ __forceinline__ SmallSeqs small_seqs(const Seqs& q, SmallSpace& m, Space& sp) {
    for (int s = threadIdx.x; s <= q.count; s += BLOCK) {
        m.offsets[s] = (int)q.at(s);
        if (s < q.count) m.fine[s] = q.good(s);
    }
    sp.total = m.total, sp.head = m.head, sp.tail = m.tail, sp.slope = m.slope, sp.loss = m.loss, sp.counts = m.counts;
    return {m.offsets, m.fine, q.tokens, q.count, q.mask};
}

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
__device__ __forceinline__ void load_mask(const uint8_t* mask, int64_t t, int64_t n, Pack<uint8_t, E>& keep) {
    if (mask) {
        load(mask, t, n, keep);
    } else {
#pragma unroll
        for (int k = 0; k < E; k++) keep.v[k] = 1;
    }
}

// a thread's tokens of two tensors (a NULL: none are wanted; b NULL: zeros)
template <class T>
struct Tokens {
    Pack<T, E> a, b;
    Pack<uint8_t, E> keep;
    __device__ __forceinline__ void get(const uint8_t* mask, const T* pa, const T* pb, int64_t t, int64_t n) {
        load_mask(mask, t, n, keep);
        if (pa) load(pa, t, n, a);
        if (pb) load(pb, t, n, b);
    }
};

// Sums of (a - b) and counts over the sequences of chunk w.  A thread adds up its own tokens; a scan over the threads that restarts
// wherever a sequence ends carries the rest.
template <class T, class Q>
__device__ __forceinline__ void chunk_sums(const Q& q, const Tokens<T>& x, bool has_a, bool has_b, int64_t w, const Space& sp) {
    __shared__ double wave_sum_[BLOCK / WAVE];
    __shared__ int wave_count_[BLOCK / WAVE], wave_closed_[BLOCK / WAVE];
    const int tid = threadIdx.x, lane = tid % WAVE, wave = tid / WAVE;
    const int64_t t0 = w * CHUNK + tid * E;
    Spot at = q.locate(t0);
    double sum = 0, first_sum = 0;
    int count = 0, first_count = 0, first_begin = 0;
    int64_t first = -1;  // the first sequence that ends among this thread's tokens
#pragma unroll
    for (int k = 0; k < E; k++) {
        if (k >= at.begin && k < at.end && x.keep.v[k]) {  // (what is masked is not looked at: it may be anything)
            if (has_a) sum += has_b ? (double)x.a.v[k] - (double)x.b.v[k] : (double)x.a.v[k];
            count++;
        }
        if (k + 1 == at.end) {
            if (first < 0)
                first = at.s, first_begin = at.begin, first_sum = sum, first_count = count;
            else
                sp.total[at.s] = {sum, count};
            sum = 0, count = 0;
            q.next(at, t0);
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
        if (first_begin + tid * E >= 0)  // it began in this chunk
            sp.total[first] = r;
        else
            sp.head[w] = r;
    }
    if (tid == BLOCK - 1 && at.s < q.count && at.begin < E) {  // goes on behind the chunk
        Rec r = {sum, count};
        if (first < 0) r.sum += in, r.count += in_count;
        if (at.begin + tid * E >= 0)
            sp.tail[w] = r;
        else
            sp.head[w] = r;
    }
    __syncthreads();  // the shared words are written again by the next chunk
}

// the whole of sequence s, by GROUP adjacent lanes; every one of them gets it
template <int GROUP, class Q>
__device__ __forceinline__ Rec sequence(const Q& q, const Space& sp, int64_t s, int l) {
    const int64_t begin = q.at(s), end = q.at(s + 1);
    Rec r = {0, 0};
    if (end > begin) {
        const int64_t w0 = begin / CHUNK, w1 = (end - 1) / CHUNK;
        if (w0 == w1) {
            if (l == 0) r = sp.total[s];
        } else {
            if (l == 0) r = sp.tail[w0];
            int64_t w = w0 + 1 + l;
            for (; w + 3 * GROUP <= w1; w += 4 * GROUP) {  // (four loads under way at once)
                Rec v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = sp.head[w + k * GROUP];
#pragma unroll
                for (int k = 0; k < 4; k++) r.sum += v[k].sum, r.count += v[k].count;
            }
            for (; w <= w1; w += GROUP) r.sum += sp.head[w].sum, r.count += sp.head[w].count;
        }
    }
#pragma unroll
    for (int o = GROUP / 2; o; o >>= 1) r.sum += shfl_xor(r.sum, o), r.count += shfl_xor(r.count, o);
    return r;
}

__device__ __forceinline__ double block_sum(double v) {
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
struct Pair {
    double loss, preferred, rejected;  // d loss / d token of its sequences, of the mean over the pairs
    double d_preferred, d_rejected;    // their R
};

// Pair i compares sequence i with sequence i + pairs.  In terms of the difference D of the two sums, h = beta D:
//   logistic  -(1-e) log sig(h) - e log sig(-h)      d/dD = beta (e - sig(-h))
//   hinge     max(0, 1 - h)                          d/dD = -beta where h < 1
//   squared   (D - 1/(2 beta))^2                     d/dD = 2 (D - 1/(2 beta))
__device__ __forceinline__ Pair pair_of(const Preference& o, const Rec& c, const Rec& r, bool good, int64_t pairs) {
    const double nc = o.normalize && c.count ? 1.0 / (double)c.count : 1.0, nr = o.normalize && r.count ? 1.0 / (double)r.count : 1.0;
    const double dc = c.sum * nc, dr = r.sum * nr, D = good ? dc - dr : NAN, h = o.beta * D;
    double loss, slope;
    if (o.kind == LBFGS_TRAIN_LOGISTIC) {
        const double e = exp(-fabs(h)), soft = log1p(e);
        loss = (1 - o.smoothing) * (soft + (h < 0 ? -h : 0)) + (o.smoothing != 0 ? o.smoothing * (soft + (h > 0 ? h : 0)) : 0);
        if (h != h) loss = h;
        slope = o.beta * (o.smoothing - (h < 0 ? 1.0 : e) / (1.0 + e));  // sig(-h)
    } else if (o.kind == LBFGS_TRAIN_HINGE) {
        loss = h > 1 ? 0 : 1 - h;
        slope = h < 1 ? -o.beta : h != h ? h : 0;
    } else {
        const double e = D - 0.5 / o.beta;
        loss = e * e;
        slope = 2 * e;
    }
    slope /= (double)pairs;
    return {loss, slope * nc, -slope * nr, dc, dr};
}

// pairs [block], [block + blocks], ... in groups: losses into sp.loss[block], rewards, and -- if they are asked for -- slopes
template <int GROUP, class A, class Q>
__device__ __forceinline__ void pair_losses(const Q& q, const Preference& o, const Space& sp, A* rewards, bool slopes, int block, int blocks) {
    const int64_t pairs = q.count / 2, each = (int64_t)blocks * (BLOCK / GROUP), rounds = (pairs + each - 1) / each;
    const int l = threadIdx.x % GROUP;
    double total = 0;
    for (int64_t k = 0; k < rounds; k++) {  // (every lane goes through the shuffles of sequence())
        const int64_t i = k * each + (int64_t)block * (BLOCK / GROUP) + threadIdx.x / GROUP;
        const bool real = i < pairs;
        const Rec c = sequence<GROUP>(q, sp, real ? i : 0, l), r = sequence<GROUP>(q, sp, real ? i + pairs : 0, l);
        if (real && l == 0) {
            const Pair p = pair_of(o, c, r, q.good(i) && q.good(i + pairs), pairs);
            total += p.loss;
            if (slopes) sp.slope[i] = p.preferred, sp.slope[i + pairs] = p.rejected;
            rewards[i] = (A)(o.beta * p.d_preferred);
            rewards[i + pairs] = (A)(o.beta * p.d_rejected);
        }
    }
    total = block_sum(total);
    if (threadIdx.x == 0) sp.loss[block] = total;
}

// gradient of chunk w: its sequence's slope at each token that counts, 0 at all others.  slope[(s - base) & within]: with a table of
// the chunk's own sequences, bad offsets still lead nowhere else.
template <class G, class Q>
__device__ __forceinline__ void chunk_slopes(const Q& q, const double* slope, int64_t base, int64_t within, G* grad, int64_t w, Spot at, const Pack<uint8_t, E>& keep) {
    typedef typename Num<G>::acc A;
    const int64_t t0 = w * CHUNK + threadIdx.x * E;
    if (t0 >= q.tokens) return;
    Pack<G, E> g;
    A v = at.s < q.count ? (A)slope[(at.s - base) & within] : 0;
#pragma unroll
    for (int k = 0; k < E; k++) {
        g.v[k] = k >= at.begin && k < at.end && keep.v[k] ? (G)v : (G)0;
        if (k + 1 == at.end) {
            q.next(at, t0);
            if (k + 1 < E) v = at.s < q.count ? (A)slope[(at.s - base) & within] : 0;
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
__global__ __launch_bounds__(BLOCK, sizeof(T) == 8 ? 4 : 6) void sums_kernel(Seqs q, const T* a, const T* b, int64_t chunks, Space sp) {
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) {
        Tokens<T> x;
        x.get(q.mask, a, b, w * CHUNK + threadIdx.x * E, q.tokens);
        chunk_sums(q, x, a != nullptr, b != nullptr, w, sp);
    }
}
template <int GROUP, class A>
__global__ __launch_bounds__(BLOCK) void pairs_kernel(Seqs q, Preference o, Space sp, A* rewards) {
    pair_losses<GROUP>(q, o, sp, rewards, true, blockIdx.x, gridDim.x);
}
template <class G>
__global__ __launch_bounds__(BLOCK) void slopes_kernel(Seqs q, int64_t chunks, int blocks, Space sp, typename Num<G>::acc* f, G* grad) {
    if (blockIdx.x == 0) mean_loss(sp, blocks, q.count / 2, f);
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) {
        const int64_t t0 = w * CHUNK + threadIdx.x * E;
        Pack<uint8_t, E> keep;
        load_mask(q.mask, t0, q.tokens, keep);
        chunk_slopes(q, sp.slope, 0, -1, grad, w, q.locate(t0), keep);
    }
}
// Not too many pairs: no pass of their own (in us, without and with: 512 sequences of 200 10.2, 13.4; 2048 of 512 16.0, 13.4).  A chunk's workgroup finds the slopes of its sequences itself, from their sums and
// their partners'; the last workgroup, which has no chunk, the loss and the rewards.
constexpr int64_t FEW_SEQS = 1024;  // (a power of two)
constexpr int64_t FEW_LONG_SEQS = 128;  // ... of many chunks (in us: 128 of 20000 16.9, 17.9; 256 of 20000 27.6, 24.9; 1000 of 8200 63, 32)
template <class G, int GROUP>
__global__ __launch_bounds__(BLOCK) void few_slopes_kernel(Seqs q, Preference o, int64_t chunks, Space sp, typename Num<G>::acc* f, typename Num<G>::acc* rewards, G* grad) {
    __shared__ double slope[FEW_SEQS];
    __shared__ int64_t ends[2];
    if (blockIdx.x == gridDim.x - 1) {
        pair_losses<GROUP>(q, o, sp, rewards, false, 0, 1);
        if (threadIdx.x == 0) *f = (typename Num<G>::acc)(sp.loss[0] / (double)(q.count / 2));
        return;
    }
    const int64_t pairs = q.count / 2, groups = gridDim.x - 1;
    const int l = threadIdx.x % GROUP;
    int64_t had = -1, had_n = 0;  // adjacent chunks for a workgroup: long sequences stay the same, and what is known of them
    const int64_t last_w = (blockIdx.x + 1) * chunks / groups;
    for (int64_t w = blockIdx.x * chunks / groups; w < last_w; w++) {
        const int64_t t0 = w * CHUNK + threadIdx.x * E;
        Pack<uint8_t, E> keep;
        load_mask(q.mask, t0, q.tokens, keep);
        const Spot at = q.locate(t0);
        if (threadIdx.x == 0) ends[0] = at.s;
        if (threadIdx.x == BLOCK - 1) {  // the last sequence that begins in the chunk
            Spot last = at;
            while (last.end <= E) q.next(last, t0);
            ends[1] = last.s < q.count ? last.s : q.count - 1;
        }
        __syncthreads();
        const int64_t first = ends[0], n = ends[1] - first + 1;
        const bool known = first == had && n == had_n;
        had = first, had_n = n;
        for (int64_t k = 0; k < n && !known; k += BLOCK / GROUP) {
            const int64_t j = k + threadIdx.x / GROUP, s = first + j;
            const bool real = j < n;
            const int64_t other = !real ? 0 : s < pairs ? s + pairs : s - pairs;
            const Rec mine = sequence<GROUP>(q, sp, real && s < 2 * pairs ? s : 0, l), its = sequence<GROUP>(q, sp, real && s < 2 * pairs ? other : 0, l);
            if (real && s < 2 * pairs && l == 0) {
                const bool preferred = s < pairs;
                const Pair p = pair_of(o, preferred ? mine : its, preferred ? its : mine, q.good(s) && q.good(other), pairs);
                slope[j] = preferred ? p.preferred : p.rejected;
            }
        }
        __syncthreads();
        chunk_slopes(q, slope, first, FEW_SEQS - 1, grad, w, at, keep);
        __syncthreads();
    }
}
// a small batch: all of it as one workgroup, with nothing between the passes but LDS
template <class T, class G>
__global__ __launch_bounds__(BLOCK) void preference_small_kernel(Seqs whole, Preference o, const T* a, const T* b, int chunks,
                                                                 typename Num<T>::acc* f, typename Num<T>::acc* rewards, G* grad) {
    __shared__ SmallSpace m;
    Space sp;
    Tokens<T> x[SMALL_CHUNKS];
#pragma unroll
    for (int w = 0; w < SMALL_CHUNKS; w++)
        if (w < chunks) x[w].get(whole.mask, a, b, w * CHUNK + threadIdx.x * E, whole.tokens);
    const SmallSeqs q = small_seqs(whole, m, sp);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SMALL_CHUNKS; w++)
        if (w < chunks) chunk_sums(q, x[w], a != nullptr, b != nullptr, w, sp);
    __syncthreads();
    pair_losses<1>(q, o, sp, rewards, true, 0, 1);
    __syncthreads();
    if (threadIdx.x == 0) *f = (typename Num<T>::acc)(sp.loss[0] / (double)(q.count / 2));
#pragma unroll
    for (int w = 0; w < SMALL_CHUNKS; w++)
        if (w < chunks) chunk_slopes(q, sp.slope, 0, -1, grad, w, q.locate(w * CHUNK + threadIdx.x * E), x[w].keep);
}

// ------------------------------------------------------------------------------------ policy
struct Policy {
    double low, high, log_low, log_high, kl;  // 1 - clip_low, 1 + clip_high and their logarithms, the KL term's weight
    int per_token, by_sequence;
};

// tokens of each sequence that count -> 1 / their number; kept tokens and sequences with any of this workgroup
template <class Q>
__device__ __forceinline__ void sequence_weights(const Q& q, const Space& sp, int block, int blocks) {
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

// the mean over all tokens needs their number alone: kept places between the first offset and the last, and whether all are good
__global__ __launch_bounds__(BLOCK) void count_kernel(Seqs q, Space sp) {
    constexpr int N = 16;
    const int64_t begin = q.at(0), end = q.at(q.count), stride = (int64_t)gridDim.x * BLOCK;
    const int64_t me = (int64_t)blockIdx.x * BLOCK + threadIdx.x;
    int kept = 0;
    constexpr int U = 4;
    for (int64_t t = begin + me * N; t < end; t += stride * N * U) {
        Pack<uint8_t, N> m[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t at = t + u * stride * N;
            if (at + N <= end)
                m[u] = *(const Pack<uint8_t, N>*)(q.mask + at);
            else
#pragma unroll
                for (int k = 0; k < N; k++) m[u].v[k] = at + k < end ? q.mask[at + k] : 0;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int k = 0; k < N; k++) kept += m[u].v[k] != 0;
    }
    bool bad = false;
    for (int64_t s = me; s < q.count; s += stride) bad |= !q.good(s);
    const double n = block_sum((double)kept), b = block_sum(bad ? 1.0 : 0.0);
    if (threadIdx.x == 0) sp.counts[2 * blockIdx.x] = b > 0 ? NAN : n, sp.counts[2 * blockIdx.x + 1] = 0;
}

// the sum of both counts over the workgroups that counted, in every thread
__device__ __forceinline__ void all_counts(const Space& sp, int blocks, double& kept, double& some) {
    kept = some = 0;
    for (int k = threadIdx.x % WAVE; k < blocks; k += WAVE) kept += sp.counts[2 * k], some += sp.counts[2 * k + 1];
    kept = wave_sum(kept);
    some = wave_sum(some);
    if (kept < 1) kept = 1;  // nothing counts: sums of nothing, divided by something
    if (some < 1) some = 1;
}

// e^x, e^x - 1 and e^x - 1 - x, each of itself: to 2^-50 for 64-bit data, and to 2^-32 for others, whose results have 24 bits.
//   x = n log 2 + r, with n = 0 and r = x below 1/2;   t = e^r - 1 - r = r^2 (1/2 + r/6 + ...);   e^x = 2^n (1 + r + t);
// of n = 0 the others are r + t and t, where they would cancel.  No branch: in most waves one of 64 differences is beyond 1/2.  Of 32-bit
// data the series is 32-bit from r^5/120 on, to r^11: 2^-24 of that is 2^-32 of t.  (With the terms in 32 bits throughout the pass over 8.4
// million tokens took 2 us less, 49.5, and the KL term and its slope were off by six roundings of the result.)
template <class T>
struct Exponential {
    double x, e, rt, t;
    bool near;
    __device__ __forceinline__ explicit Exponential(double x_) : x(x_) {
        const double xc = __builtin_fmin(__builtin_fmax(x, -1000.0), 1000.0);  // (e^x is 0 or infinite there; and of a NaN some number)
        near = fabs(xc) < 0.5;
        const double n = near ? 0 : rint(xc * 1.4426950408889634);
        const double r = fma(n, -2.3190468138462996e-17, fma(n, -0.6931471805599453, xc));  // log 2 and what a double leaves of it
        double p;
        if constexpr (sizeof(T) == 8) {
            p = 1. / 1307674368000.;  // 15!
            p = fma(p, r, 1. / 87178291200.);
            p = fma(p, r, 1. / 6227020800.);
            p = fma(p, r, 1. / 479001600.);
            p = fma(p, r, 1. / 39916800.);
            p = fma(p, r, 1. / 3628800.);
            p = fma(p, r, 1. / 362880.);
            p = fma(p, r, 1. / 40320.);
            p = fma(p, r, 1. / 5040.);
            p = fma(p, r, 1. / 720.);
            p = fma(p, r, 1. / 120.);
            p = fma(p, r, 1. / 24.);
        } else {
            const float h = (float)r;
            float c = 1.f / 39916800.f;  // 11!
            c = fmaf(c, h, 1.f / 3628800.f);
            c = fmaf(c, h, 1.f / 362880.f);
            c = fmaf(c, h, 1.f / 40320.f);
            c = fmaf(c, h, 1.f / 5040.f);
            c = fmaf(c, h, 1.f / 720.f);
            c = fmaf(c, h, 1.f / 120.f);
            p = fma((double)c, r, 1. / 24.);
        }
        p = fma(p, r, 1. / 6.);
        t = r * r * fma(p, r, 0.5);
        rt = r + t;
        e = ldexp(1 + rt, (int)n);
        if (x != x) e = t = x;
    }
    __device__ __forceinline__ double value() const { return e; }
    __device__ __forceinline__ void less(double& em1, double& k) const { em1 = near ? rt : e - 1, k = near ? t : em1 - x; }
};

template <class T, class G>
struct PolicyData {
    const T *logps, *old, *ref, *adv;
    G* grad;
};
// a thread's tokens
template <class T>
struct PolicyTokens {
    Pack<T, E> lp, old, ref, adv;
    Pack<uint8_t, E> keep;
    template <class G>
    __device__ __forceinline__ void get(const PolicyData<T, G>& x, const uint8_t* mask, bool per_token, int64_t t, int64_t n) {
        load(x.logps, t, n, lp);
        load(x.old, t, n, old);
        if (x.ref) load(x.ref, t, n, ref);
        if (per_token) load(x.adv, t, n, adv);
        load_mask(mask, t, n, keep);
    }
};

// L = -min(r A, clip(r) A) + kl (e^q - 1 - q) with r = e^d, d = logp - old, q = ref - logp.  All of it in 64 bits, the slope rounded once, to
// the gradient's type: advantages have mean 0, and the mean of r A is what is left of terms a thousand times larger; where they are 0, as a
// group of equal rewards has them, the KL term is all there is; and at the border that an advantage goes with the gradient jumps.
template <class T>
__device__ __forceinline__ void token(const Policy& o, T lp, T old, T ref, double a, double weight, double& slope, double& f, double& kl, double& clipped) {
    const double d = (double)lp - (double)old;
    const bool over = a > 0 ? d > o.log_high : a < 0 && d < o.log_low;
    const double ra = a == 0 && d == d ? 0 : Exponential<T>(d).value() * a;  // (an advantage of 0 gives 0 for any ratio, one that overflowed too)
    double loss = over ? -(a > 0 ? o.high : o.low) * a : -ra;
    slope = over ? 0 : -ra;
    if (o.kl != 0) {
        double em1, term;
        Exponential<T>((double)ref - (double)lp).less(em1, term);
        loss += o.kl * term;
        slope -= o.kl * em1;
        kl += term;
    }
    f += loss * weight;
    clipped += over;
    slope *= weight;
}

template <class T, class G, class Q>
__device__ __forceinline__ void chunk_policy(const Q& q, const Policy& o, const PolicyTokens<T>& x, const T* advantages, G* grad, const double* inverse, double inv,
                                             int64_t w, double& f, double& kl, double& clipped) {
    const int64_t t0 = w * CHUNK + threadIdx.x * E, n = q.tokens;
    Spot at = q.locate(t0);
    if (t0 >= n) return;
    Pack<G, E> g;
    double a_seq = 0, weight = inv;
    auto enter = [&]() {
        if (at.s < q.count) {
            if (!o.per_token) a_seq = (double)advantages[at.s];
            if (o.by_sequence) weight = inv * inverse[at.s];
        }
    };
    enter();
#pragma unroll
    for (int k = 0; k < E; k++) {
        double slope = 0;
        if (k >= at.begin && k < at.end && x.keep.v[k])
            token<T>(o, x.lp.v[k], x.old.v[k], x.ref.v[k], o.per_token ? (double)x.adv.v[k] : a_seq, weight, slope, f, kl, clipped);
        g.v[k] = (G)slope;
        if (k + 1 == at.end) {
            q.next(at, t0);
            if (k + 1 < E) enter();
        }
    }
    store(grad, t0, n, g);
}

template <class A>
__device__ __forceinline__ void policy_results(double f, double kl, double clipped, double kept, A* out_f, A* out_kl, A* out_clipped) {
    f = block_sum(f);
    kl = block_sum(kl);
    clipped = block_sum(clipped);
    if (threadIdx.x == 0) *out_f = (A)(kept == kept ? f : kept), *out_kl = (A)(kl / kept), *out_clipped = (A)(clipped / kept);
}

__global__ __launch_bounds__(BLOCK) void weights_kernel(Seqs q, Space sp) { sequence_weights(q, sp, blockIdx.x, gridDim.x); }
template <class T, class G>
__global__ __launch_bounds__(BLOCK) void policy_kernel(Seqs q, Policy o, PolicyData<T, G> x, int64_t chunks, int count_blocks, Space sp) {
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, count_blocks, kept, some);
    const double inv = 1.0 / (o.by_sequence ? some : kept);
    for (int64_t w = blockIdx.x; w < chunks; w += gridDim.x) {
        PolicyTokens<T> t;
        t.get(x, q.mask, o.per_token, w * CHUNK + threadIdx.x * E, q.tokens);
        chunk_policy(q, o, t, x.adv, x.grad, sp.slope, inv, w, f, kl, clipped);
    }
    f = block_sum(f);
    kl = block_sum(kl);
    clipped = block_sum(clipped);
    if (threadIdx.x == 0) sp.sums[3 * blockIdx.x] = f, sp.sums[3 * blockIdx.x + 1] = kl, sp.sums[3 * blockIdx.x + 2] = clipped;
}
// The mean over all tokens with an advantage for each: nothing is a sequence's own, all tokens from the first offset to the last are
// alike, and nobody looks for their sequences.  One pack of 16 bytes of each tensor a thread.  2048 x 4096 tokens in 32 bits with a
// reference: 45 us in all (53 by the pass that knows sequences), with a mask 51 (59).
constexpr int ALIKE_BLOCKS = 1280;  // five to a compute unit
template <class T, class G>
__global__ __launch_bounds__(BLOCK) void policy_alike_kernel(Seqs q, Policy o, PolicyData<T, G> x, int count_blocks, Space sp) {
    constexpr int N = vec_len<T>();
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, count_blocks, kept, some);
    const double inv = 1.0 / kept;
    const int64_t begin = q.at(0), end = q.at(q.count), n = q.tokens, stride = (int64_t)gridDim.x * BLOCK * N;
    for (int64_t t = ((int64_t)blockIdx.x * BLOCK + threadIdx.x) * N; t < n; t += stride) {
        Pack<T, N> lp, old, ref, adv;
        Pack<G, N> g;
        Pack<uint8_t, N> keep;
        if (t + N <= n) {
            lp = *(const Pack<T, N>*)(x.logps + t), old = *(const Pack<T, N>*)(x.old + t), adv = *(const Pack<T, N>*)(x.adv + t);
            if (x.ref) ref = *(const Pack<T, N>*)(x.ref + t);
            if (q.mask) keep = *(const Pack<uint8_t, N>*)(q.mask + t);
#pragma unroll
            for (int k = 0; k < N; k++) {
                double slope = 0;
                if (t + k >= begin && t + k < end && (!q.mask || keep.v[k])) token<T>(o, lp.v[k], old.v[k], ref.v[k], (double)adv.v[k], 1.0, slope, f, kl, clipped);
                g.v[k] = (G)(slope * inv);
            }
            *(Pack<G, N>*)(x.grad + t) = g;
        } else {
            for (int64_t k = t; k < n; k++) {
                double slope = 0;
                if (k >= begin && k < end && (!q.mask || q.mask[k]))
                    token<T>(o, x.logps[k], x.old[k], x.ref ? x.ref[k] : (T)0, (double)x.adv[k], 1.0, slope, f, kl, clipped);
                x.grad[k] = (G)(slope * inv);
            }
        }
    }
    f = block_sum(f);
    kl = block_sum(kl);
    clipped = block_sum(clipped);
    if (threadIdx.x == 0) sp.sums[3 * blockIdx.x] = f * inv, sp.sums[3 * blockIdx.x + 1] = kl, sp.sums[3 * blockIdx.x + 2] = clipped;
}
template <class A>
__global__ __launch_bounds__(BLOCK) void policy_results_kernel(Space sp, int count_blocks, int blocks, A* out_f, A* out_kl, A* out_clipped) {
    double kept, some, f = 0, kl = 0, clipped = 0;
    all_counts(sp, count_blocks, kept, some);
    for (int k = threadIdx.x; k < blocks; k += BLOCK) f += sp.sums[3 * k], kl += sp.sums[3 * k + 1], clipped += sp.sums[3 * k + 2];
    policy_results(f, kl, clipped, kept, out_f, out_kl, out_clipped);
}
template <class T, class G>
__global__ __launch_bounds__(BLOCK) void policy_small_kernel(Seqs whole, Policy o, PolicyData<T, G> x, int chunks, typename Num<T>::acc* out_f,
                                                             typename Num<T>::acc* out_kl, typename Num<T>::acc* out_clipped) {
    __shared__ SmallSpace m;
    Space sp;
    PolicyTokens<T> t[SMALL_CHUNKS];
#pragma unroll
    for (int w = 0; w < SMALL_CHUNKS; w++)
        if (w < chunks) t[w].get(x, whole.mask, o.per_token, w * CHUNK + threadIdx.x * E, whole.tokens);
    const SmallSeqs q = small_seqs(whole, m, sp);
    __syncthreads();
    double kept, some = 1, f = 0, kl = 0, clipped = 0;
    if (!o.by_sequence) {  // the number of all tokens is wanted, not each sequence's
        int n = 0;
        bool bad = false;
#pragma unroll
        for (int w = 0; w < SMALL_CHUNKS; w++)
#pragma unroll
            for (int k = 0; k < E; k++) {
                const int at = w * CHUNK + (int)threadIdx.x * E + k;
                if (w < chunks && at >= q.at(0) && at < q.at(q.count)) n += t[w].keep.v[k] != 0;
            }
        for (int64_t s = threadIdx.x; s < q.count; s += BLOCK) bad |= !q.good(s);
        kept = block_sum(bad ? NAN : (double)n);
        if (kept < 1) kept = 1;
    } else {
        if (q.mask) {
#pragma unroll
            for (int w = 0; w < SMALL_CHUNKS; w++)
                if (w < chunks) {
                    Tokens<T> k;
                    k.keep = t[w].keep;
                    chunk_sums(q, k, false, false, w, sp);
                }
            __syncthreads();
        }
        sequence_weights(q, sp, 0, 1);
        __syncthreads();
        all_counts(sp, 1, kept, some);
    }
    const double inv = 1.0 / (o.by_sequence ? some : kept);
#pragma unroll
    for (int w = 0; w < SMALL_CHUNKS; w++)
        if (w < chunks) chunk_policy(q, o, t[w], x.adv, x.grad, sp.slope, inv, w, f, kl, clipped);
    policy_results(f, kl, clipped, kept, out_f, out_kl, out_clipped);
}

// ------------------------------------------------------------------------------------ launches
// Up to so many tokens and sequences one workgroup does the whole of a loss, without a workspace.  Measured, whole calls one after the
// other, in us (as several launches in brackets): 8 sequences of 60 tokens, preference 7.6 (10.9), policy 8.1 (13.9); 2 of 2048, 9.4 (10.3)
// and 10.4 (13.8), with a mask and a mean of means 13.1 (18.0); 256 of 16, 11.3 (11.2), 11.6 (14.3) and 18.1 (19.7).
static bool small(int64_t tokens, int64_t seqs) { return tokens <= SMALL_TOKENS && seqs <= SMALL_SEQS; }

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

template <class T, class G>
static void launch_preference(const Seqs& q, const Preference& o, const void* a, const void* b, void* f, void* rewards, void* grad, const Space& sp, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const int64_t chunks = chunks_of(q.tokens), pairs = q.count / 2;
    if (small(q.tokens, q.count)) {
        preference_small_kernel<T, G><<<1, BLOCK, 0, s>>>(q, o, (const T*)a, (const T*)b, (int)chunks, (A*)f, (A*)rewards, (G*)grad);
        return;
    }
    // The records of a sequence (one for each chunk it reaches) are added up by one lane, or by eight where there are many.  Measured, in
    // us, one and eight: 48 sequences of 131072 44.4, 27.9, of 65536 25.9, 19.4; 512 of 2048 10.5, 27.9.
    const bool many = q.tokens / q.count > 4 * CHUNK;
    const int64_t groups = (pairs * (many ? 8 : 1) + BLOCK - 1) / BLOCK;
    const int blocks = (int)(groups < LOSS_BLOCKS ? groups : LOSS_BLOCKS);
    const unsigned grid = (unsigned)(chunks < (1 << 20) ? (chunks ? chunks : 1) : (1 << 20));
    if (chunks) sums_kernel<T><<<grid, BLOCK, 0, s>>>(q, (const T*)a, (const T*)b, chunks, sp);
    if (q.count <= (many ? FEW_LONG_SEQS : FEW_SEQS)) {
        const unsigned grid = (unsigned)(chunks < 768 ? chunks : 768);  // (three to a compute unit: all of them at once)
        if (many)
            few_slopes_kernel<G, 8><<<grid + 1, BLOCK, 0, s>>>(q, o, chunks, sp, (A*)f, (A*)rewards, (G*)grad);
        else
            few_slopes_kernel<G, 1><<<grid + 1, BLOCK, 0, s>>>(q, o, chunks, sp, (A*)f, (A*)rewards, (G*)grad);
        return;
    }
    if (many)
        pairs_kernel<8, A><<<blocks, BLOCK, 0, s>>>(q, o, sp, (A*)rewards);
    else
        pairs_kernel<1, A><<<blocks, BLOCK, 0, s>>>(q, o, sp, (A*)rewards);
    slopes_kernel<G><<<grid, BLOCK, 0, s>>>(q, chunks, blocks, sp, (A*)f, (G*)grad);
}

template <class T, class G>
static void launch_policy(const Seqs& q, const Policy& o, const void* logps, const void* old, const void* ref, const void* adv, void* f, void* kl,
                          void* clipped, void* grad, const Space& sp, hipStream_t s) {
    typedef typename Num<T>::acc A;
    const int64_t chunks = chunks_of(q.tokens);
    const PolicyData<T, G> x = {(const T*)logps, (const T*)old, (const T*)ref, (const T*)adv, (G*)grad};
    if (small(q.tokens, q.count)) {
        policy_small_kernel<T, G><<<1, BLOCK, 0, s>>>(q, o, x, (int)chunks, (A*)f, (A*)kl, (A*)clipped);
        return;
    }
    const bool total = q.mask && !o.by_sequence;  // the number of all tokens is wanted, not each sequence's
    const int64_t groups = total ? (q.tokens + 16 * BLOCK - 1) / (16 * BLOCK) + 1 : (q.count * 8 + BLOCK - 1) / BLOCK;
    const int count_blocks = (int)(groups < COUNT_BLOCKS ? groups : COUNT_BLOCKS);
    int blocks = (int)(chunks < POLICY_BLOCKS ? (chunks ? chunks : 1) : POLICY_BLOCKS);
    if (total) {
        count_kernel<<<count_blocks, BLOCK, 0, s>>>(q, sp);
    } else {
        if (q.mask && chunks) sums_kernel<T><<<(unsigned)(chunks < (1 << 20) ? chunks : (1 << 20)), BLOCK, 0, s>>>(q, (const T*)nullptr, (const T*)nullptr, chunks, sp);
        weights_kernel<<<count_blocks, BLOCK, 0, s>>>(q, sp);
    }
    if (o.per_token && !o.by_sequence) {
        const int64_t packs = (q.tokens + vec_len<T>() - 1) / vec_len<T>(), need = (packs + BLOCK - 1) / BLOCK;
        blocks = (int)(need < ALIKE_BLOCKS ? (need ? need : 1) : ALIKE_BLOCKS);
        policy_alike_kernel<T, G><<<blocks, BLOCK, 0, s>>>(q, o, x, count_blocks, sp);
    } else {
        policy_kernel<T, G><<<blocks, BLOCK, 0, s>>>(q, o, x, chunks, count_blocks, sp);
    }
    policy_results_kernel<A><<<1, BLOCK, 0, s>>>(sp, count_blocks, blocks, (A*)f, (A*)kl, (A*)clipped);
}

static int check_seqs(const lbfgs_train_sequences* in, Seqs* q, const char* who) {
    if (!in) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: no sequences", who);
    if ((in->dtype & ~LBFGS_TRAIN_WIDE_GRAD) < LBFGS_TRAIN_F64 || (in->dtype & ~LBFGS_TRAIN_WIDE_GRAD) > LBFGS_TRAIN_F16)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: unknown element type %d", who, in->dtype);
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
    const uint64_t need = lbfgs_train_sequences_workspace(q.tokens, q.count);
    *sp = Space();
    if (!need) return LBFGS_HIP_OK;
    if (!workspace || bytes < need)
        return lt_fail(LBFGS_HIP_ERR_ARG, "%s: %llu bytes of workspace, %llu are needed", who, (unsigned long long)(workspace ? bytes : 0), (unsigned long long)need);
    if ((uintptr_t)workspace % 256) return lt_fail(LBFGS_HIP_ERR_ARG, "%s: the workspace is not aligned to 256 bytes", who);
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
    return small(tokens, count) ? 0 : lay_out(nullptr, nullptr, tokens, count);
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
        case LBFGS_TRAIN_F64:
        case LBFGS_TRAIN_F64 | LBFGS_TRAIN_WIDE_GRAD: launch_preference<double, double>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_F32:
        case LBFGS_TRAIN_F32 | LBFGS_TRAIN_WIDE_GRAD: launch_preference<float, float>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_BF16: launch_preference<bf16, bf16>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_F16: launch_preference<f16, f16>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        case LBFGS_TRAIN_BF16 | LBFGS_TRAIN_WIDE_GRAD: launch_preference<bf16, float>(q, o, logps, ref_logps, f, rewards, grad, sp, s); break;
        default: launch_preference<f16, float>(q, o, logps, ref_logps, f, rewards, grad, sp, s);
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
        case LBFGS_TRAIN_F64:
        case LBFGS_TRAIN_F64 | LBFGS_TRAIN_WIDE_GRAD: launch_policy<double, double>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_F32:
        case LBFGS_TRAIN_F32 | LBFGS_TRAIN_WIDE_GRAD: launch_policy<float, float>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_BF16: launch_policy<bf16, bf16>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_F16: launch_policy<f16, f16>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        case LBFGS_TRAIN_BF16 | LBFGS_TRAIN_WIDE_GRAD: launch_policy<bf16, float>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s); break;
        default: launch_policy<f16, float>(q, o, logps, old_logps, ref_logps, advantages, f, kl, clip_fraction, grad, sp, s);
    }
    return lt_launched(who);
}
