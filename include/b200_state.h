/* b200_state.h -- models that keep a state of fixed size per sequence, and beam search over them.
 *
 * The mixers of b200_ggml_ops.h (mLSTM, linear attention, gated delta rule, minGRU, time mixing) keep a state per slot.  Here are the selective state space scan with the
 * short convolution in front of it, the selection of a beam search, and what that makes necessary: slots that become what other slots held.
 *
 * A step's rows name their sequences through seq_info, int32 [4][n_seq]: a sequence's first row, its count of rows, its slot, and whether it begins (!= 0: its state and its last
 * inputs are zeros, whatever the slot holds).  Sequences whose slot is outside [0, n_slots) or whose first row is none of the n_tokens are left out, and so are rows behind these; rows that belong
 * to no sequence stay as they are, and so do the slots of sequences without rows, also of those that begin.  A slot appears once in a step, and no two sequences have a row in common.  seq_info
 * NULL: n_seq sequences of n_tokens / n_seq rows each, one behind the other, in the slots 0, 1, .., none of which begins.
 * max_new: no sequence has more rows than that; those behind are left out (0: n_tokens).
 *
 * Types of rows: B200_TYPE_F32, B200_TYPE_F16, B200_TYPE_BF16, at any alignment of their own type; strides in values.  States, weights and sums are f32.  All functions
 * return a b200_status, check their arguments on the host, launch on `stream` and the current device, allocate nothing, do not wait for the device, and can be captured into
 * CUDA graphs.  Results do not depend on timing.  A workspace belongs to one stream: calls that may run at the same time have one each.  It needs no particular contents.
 */
#ifndef B200_STATE_H
#define B200_STATE_H

#include "b200_ggml.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_STATE_MAX_INDEX (1 << 30) /* rows of a step, channels: no more (B200_ERR_UNSUPPORTED) */

/* Short causal convolution, every channel by itself: y[t][c] = act(bias[c] + sum_j w[c][j] * x[t - taps + 1 + j][c]), zeros in front of a sequence; act is silu or nothing.
 * The last taps - 1 inputs of a sequence wait in its slot of `tail` for its next rows.  dst is other memory than x.  (b200_op_short_conv has its bias in front and rows of f32.) */
typedef struct {
    const void *x; int64_t x_stride;       /* [n_tokens][channels] */
    const float *w, *bias;                 /* [channels][taps]; [channels] or NULL */
    const int32_t *seq_info;
    float *tail; int64_t slot_stride;      /* [taps - 1][channels] per slot; NULL with taps == 1 */
    void *dst; int64_t dst_stride;         /* [n_tokens][channels] */
    int32_t n_seq, n_slots, n_tokens, max_new;
    int32_t channels, taps;                /* taps <= 16 */
    int32_t silu, type;                    /* type: of x and dst */
} b200_ssm_conv_args;
B200_API int b200_op_ssm_conv(const b200_ssm_conv_args *a, b200_stream_t stream);

/* Selective state space scan: per channel a state of d_state numbers,
 *   d = dt[t][c] + dt_bias[c], softplus != 0: d = ln(1 + e^d);   h[c][n] <- exp(d * a[c][n]) * h[c][n] + d * x[t][c] * b[t][g][n];
 *   y = sum_n c[t][g][n] * h[c][n] + skip[c] * x[t][c];   dst[t][c] = y, or y * silu(z[t][c]) with z,
 * where channel c belongs to group g = c / (channels / groups).  Everything between the rows is f32.  Rates
 * a of -inf and +inf count as the largest numbers of f32: a row with d = 0 leaves the state as it is.  `from` (optional): states are read there, in slots of from_stride, instead of
 * from `state` (other memory than that).  Few channels and a long sequence: the rows are shared out in stretches, whose states meet in the workspace (b200_ssm_scan_workspace_bytes bytes, 16-byte
 * aligned, 0: none).  How many goes by how a step is cut, and a smaller step may need more than a larger one; B200_SSM_SCAN_WORKSPACE_MAX are enough for every step. */
#define B200_SSM_SCAN_WORKSPACE_MAX (1 << 24)
typedef struct {
    const void *x, *dt; int64_t x_stride, dt_stride;         /* [n_tokens][channels] */
    const void *b, *c; int64_t b_stride, c_stride;           /* [n_tokens][groups * d_state] */
    const void *z; int64_t z_stride;                         /* [n_tokens][channels] or NULL */
    const float *a;                                          /* [channels][d_state] */
    const float *dt_bias, *d;                                /* [channels] or NULL each; d: the skip */
    const int32_t *seq_info;
    float *state; int64_t slot_stride;                       /* [channels][d_state] per slot */
    const float *from; int64_t from_stride;
    void *dst; int64_t dst_stride;                           /* [n_tokens][channels]; may be x, dt or z at its stride */
    int32_t n_seq, n_slots, n_tokens, max_new;
    int32_t channels, d_state, groups;                       /* d_state <= 128; groups divides channels */
    int32_t softplus, type;                                  /* type: of x, dt, b, c, z and dst */
} b200_ssm_scan_args;
B200_API size_t b200_ssm_scan_workspace_bytes(const b200_ssm_scan_args *a);
B200_API int b200_op_ssm_scan(const b200_ssm_scan_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream);

/* ---- beam search -------------------------------------------------------------------------------------------------------------------------------------
 * Every request has n_beams beams, a row of logits each, one behind the other.  The successors of a beam that has not ended are all tokens: score[beam] + logit - ln(sum of exp(logits));
 * those of an ended one (ended != NULL and not 0 there) are end_token alone: score[beam].  The n_keep best of a request go to to_*, best first, equal ones in the order of
 * (beam, token); to_beam counts within the request, to_slot (optional) is that beam's entry of `slot`.  Scores are compared in 64 bits before they are rounded to f32; the ln(sum) in
 * them is a sum of f32 exponentials, good to 2^-21, so the order of successors of different beams is no better than that.  A successor of
 * score -inf is none: neither is a token whose logit is -inf or NaN, or any of a beam whose score is -inf or NaN.  (Beams of a request that has just begun: all scores but one are -inf.)
 * Where there are fewer than n_keep successors, the rest are score -inf, beam -1, token -1, slot -1.  The workspace (b200_beam_select_workspace_bytes bytes) is 8-byte aligned.  With logits of +inf those tokens share their row evenly. */
#define B200_BEAM_MAX 64     /* beams of a request */
#define B200_BEAM_KEEP 128   /* successors that are kept */
#define B200_BEAM_VOCAB (1 << 30)
typedef struct {
    const void *logits; int64_t logits_stride;               /* [n_requests * n_beams][n_vocab] */
    const float *score;                                      /* [n_requests * n_beams] */
    const int32_t *ended, *slot;                             /* [n_requests * n_beams] or NULL each */
    float *to_score; int32_t *to_beam, *to_token, *to_slot;  /* [n_requests * n_keep]; to_slot may be NULL; none of them is an input */
    int32_t n_requests, n_beams, n_vocab, n_keep, end_token;
    int32_t type;                                            /* of logits */
} b200_beam_select_args;
B200_API size_t b200_beam_select_workspace_bytes(const b200_beam_select_args *a);
B200_API int b200_op_beam_select(const b200_beam_select_args *a, void *workspace, size_t workspace_bytes, b200_stream_t stream);

/* What slots hold moves, all at once: slot dst[i] becomes what slot src[i] held before the call, i < n, in all the states (one for each layer and kind of state).  Entries
 * with a slot outside [0, n_slots), and those whose dst an entry before them has, count as refused and change nothing; *refused (optional) is raised by their number.  States
 * lie apart; pointers, strides and sizes are multiples of 4 bytes. */
#define B200_STATE_MAX_SLOTS 4096
#define B200_STATE_MAX_MOVES 1024
typedef struct {
    void *base;          /* slot s is at base + s * stride */
    int64_t stride;      /* bytes from slot to slot */
    int64_t bytes;       /* of a slot that move */
} b200_slot_state;
B200_API int b200_op_state_reorder(const b200_slot_state *states, int32_t n_states, const int32_t *src, const int32_t *dst, int32_t n, int32_t n_slots, int32_t *refused,
                                   b200_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* B200_STATE_H */
