/*
 * include/lbfgs_train.h -- C-ABI of the operators that stand beside the optimiser when what it minimises is the loss of a
 * language model: token log-probabilities, preference and policy losses with their gradients, and the matrix form of an
 * update.  Extension: the reference crate has no such operators.
 *
 * Conventions (those of lbfgs_hip.h, whose status codes these functions return)
 *  - plain C, no torch / HIP types in signatures (a stream is passed as void*, NULL = the device's default stream);
 *  - every function returns an int status (0 = ok, <0 = error) and never unwinds; lbfgs_train_last_error() gives the
 *    calling thread's message.  Arguments are checked before anything is enqueued;
 *  - all pointers are device memory of ONE device, which is the calling thread's current one; nothing is allocated,
 *    copied to the host or waited for: a call only enqueues kernels, also into a stream that is being captured;
 *  - outputs overlap neither inputs nor each other;
 *  - workspaces are the caller's, aligned to 256 bytes and at least as large as the matching *_workspace() says, one for each
 *    call in flight (calls on one stream may share one); their contents need no preparation and mean nothing afterwards;
 *  - element types: F64, F32, BF16, F16.  The wide type of a call is F64 for F64 data and F32 for the others: sums and
 *    losses come out in it (sums over tokens are taken in 64 bits for all of them);
 *  - results are the same, bit for bit, from call to call: no sum's order depends on timing.
 */
#ifndef LBFGS_TRAIN_H
#define LBFGS_TRAIN_H

#include <stddef.h>
#include <stdint.h>

#include "lbfgs_hip.h" /* status codes */

#ifdef __cplusplus
extern "C" {
#endif

#define LBFGS_TRAIN_ABI_VERSION 1

enum { LBFGS_TRAIN_F64 = 0, LBFGS_TRAIN_F32 = 1, LBFGS_TRAIN_BF16 = 2, LBFGS_TRAIN_F16 = 3 };

int lbfgs_train_abi_version(void);
/* 16 hex digits: hash of the sources and flags this library was built from (as lbfgs_hip_build_id) */
const char* lbfgs_train_build_id(void);
/* the message of the calling thread's latest refused or failed call; "" if there was none */
const char* lbfgs_train_last_error(void);

/* ------------------------------------------------------------------------- */
/* token log-probabilities                                                     */
/* ------------------------------------------------------------------------- */
/* outer x inner rows of `vocab` logits each; row (i, j) starts at logits + i*outer_stride + j*inner_stride (elements),
 * its logits are adjacent: a batch [outer, inner + 1, vocab] without its last position needs no copy */
typedef struct lbfgs_train_rows {
    const void* logits;
    const int64_t* targets;    /* [outer*inner]: the token of each row */
    int32_t dtype;
    int32_t _pad;
    int64_t outer, inner, vocab;
    int64_t outer_stride, inner_stride;
    int64_t ignore_index;      /* a target of this value: the row is not read, its log-probability and gradient are 0 */
} lbfgs_train_rows;
/*   logps[t] = (x_t[y_t] - m_t)/temperature - l_t,   m_t = max_v x_t[v],   l_t = log sum_v exp((x_t[v] - m_t)/temperature)
 * logps in the wide type; lse[2 t] = m_t and lse[2 t + 1] = l_t in 64 bits, the log-sum-exp in two parts: their sum would lose
 * the second where the first is large, as in a row masked by its type's lowest value.
 * A target outside [0, vocab) that is not ignore_index gives NaN.  Temperatures: 1e-37 to 1e37, for F64 1e-300 to 1e300. */
uint64_t lbfgs_train_token_logprobs_workspace(int32_t dtype, int64_t rows, int64_t vocab);
int lbfgs_train_token_logprobs(const lbfgs_train_rows* rows, double temperature, void* logps, double* lse, void* workspace,
                               uint64_t workspace_bytes, void* stream);
/*   dlogits[t][v] = grad[t]/temperature * (1[v == y_t] - exp((x_t[v] - m_t)/temperature - l_t))     [outer*inner, vocab], dense
 * grad in the wide type; a row whose grad is 0 is not read and gets zeros. */
int lbfgs_train_token_logprobs_grad(const lbfgs_train_rows* rows, double temperature, const double* lse, const void* grad,
                                    void* dlogits, void* stream);

/* ------------------------------------------------------------------------- */
/* losses over the token log-probabilities of many sequences                   */
/* ------------------------------------------------------------------------- */
/* `tokens` adjacent values in `count` sequences: sequence s is tokens [offsets[s], offsets[s+1]) (offsets[count+1], not
 * decreasing, 32 or 64 bits), or, with offsets NULL, the s-th of `count` equal parts: a padded batch.  Tokens that no
 * sequence has, and those whose mask is 0, are not looked at: their values may be anything, their gradient is 0.  Offsets that
 * decrease or leave [0, tokens] make the loss NaN (nothing out of range is read or written). */
/* (A loss that is a mean has slopes of 1 / tokens or 1 / (pairs * length), and what is multiplied into them comes later.  By then F16, whose
 * smallest normal number is 6e-5 and whose smallest step 6e-8, has lost bits from some 10^4 tokens on, and from 3e7 on everything.) */
enum { LBFGS_TRAIN_WIDE_GRAD = 256 };
typedef struct lbfgs_train_sequences {
    const void* offsets;
    const uint8_t* mask;       /* [tokens] or NULL */
    int32_t offset_bits;
    int32_t dtype;             /* of every tensor over tokens; | LBFGS_TRAIN_WIDE_GRAD: but of grad, which is in the wide type */
    int64_t tokens, count;
} lbfgs_train_sequences;
uint64_t lbfgs_train_sequences_workspace(int64_t tokens, int64_t count);

/* Paired log ratios.  R_s = sum over the sequence's tokens of logps - ref_logps (ref NULL: 0), divided by their number if
 * normalize_lengths; pair i is sequence i (preferred) and sequence i + count/2 (rejected); D = R_i - R_{i+count/2}, h = beta D:
 *   LOGISTIC  -(1-e) log sigmoid(h) - e log sigmoid(-h), e = label_smoothing
 *   HINGE     max(0, 1 - h)
 *   SQUARED   (D - 1/(2 beta))^2
 * *f = the mean over pairs, rewards[s] = beta R_s (both in the wide type), grad = df/dlogps.  A sequence without tokens has R = 0. */
enum { LBFGS_TRAIN_LOGISTIC = 0, LBFGS_TRAIN_HINGE = 1, LBFGS_TRAIN_SQUARED = 2 };
int lbfgs_train_preference(const lbfgs_train_sequences* seqs, const void* logps, const void* ref_logps, double beta, double label_smoothing,
                           int32_t kind, int32_t normalize_lengths, void* f, void* rewards, void* grad, void* workspace,
                           uint64_t workspace_bytes, void* stream);

/* Clipped importance ratios.  For each token, with r = exp(logps - old_logps), q = ref_logps - logps, A its advantage
 * (advantages[tokens] if per_token, else advantages[count]):
 *   L = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - 1 - q)
 * *f = sum of L / N over the N tokens that count, or, by_sequence, the mean over the sequences that have tokens of their own
 * mean; *kl = mean of exp(q) - 1 - q (0 if kl_coef is 0); *clip_fraction = share of tokens whose ratio is clipped; all three in
 * the wide type; grad = df/dlogps.  No tokens at all: zeros. */
int lbfgs_train_policy(const lbfgs_train_sequences* seqs, const void* logps, const void* old_logps, const void* ref_logps,
                       const void* advantages, int32_t per_token, double clip_low, double clip_high, double kl_coef,
                       int32_t by_sequence, void* f, void* kl, void* clip_fraction, void* grad, void* workspace,
                       uint64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------- */
/* the matrix form of an update                                                */
/* ------------------------------------------------------------------------- */
/* `batch` dense matrices rows x cols (F32, BF16, F16; batch <= 32767, sides <= 2^20): each is divided by its Frobenius norm (a
 * matrix of zeros stays one), and then `steps` times (1 to 64) every singular value s becomes a s + b s^3 + c s^5, the singular
 * vectors staying as they are:  X <- (a I + b S + c S S) X, S = X X^T.  Products and sums have 32-bit precision or more; for
 * BF16 and F16 the last steps are taken together, which adds at most 2^-10 (BF16) or 2^-13 (F16) of the result's norm to the
 * rounding of the result, half of what that alone may be.  Coefficients that lead a singular value of [0, 1] beyond 64, or
 * multiply one by 128 or more in a step, are refused. */
uint64_t lbfgs_train_orthogonalize_workspace(int32_t dtype, int64_t batch, int64_t rows, int64_t cols);
int lbfgs_train_orthogonalize(int32_t dtype, int64_t batch, int64_t rows, int64_t cols, const void* update, void* out, int32_t steps,
                              double a, double b, double c, void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LBFGS_TRAIN_H */
