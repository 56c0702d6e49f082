/* cail_ops.h — language-model operators of libcail_ops.so (sm_100a kernels).
 *
 * Every entry point queues its work on `stream` of the current device and
 * returns without waiting, so calls may run from several host threads and may
 * be captured into CUDA graphs.  Pointers are device pointers; strides are in
 * elements.  Scratch memory is the caller's and belongs to one call until that
 * call's work has finished.  Nothing is allocated or kept from one call to the
 * next but one word of mapped host memory per device: the first call of a
 * kernel that waits for its data (16-bit attention and decoding, the loss of
 * many rows) allocates it, which may synchronise, and where such a kernel gave
 * up, the next such call on the device fails (cail_ops_device_error_word).
 *
 * Return value: CAIL_OPS_OK, CAIL_OPS_EINVAL (refused before any launch) or
 * CAIL_OPS_ECUDA (a CUDA call failed); cail_ops_last_error() gives the text
 * of this thread's last failure.  No entry point throws.
 */
#ifndef CAIL_OPS_H
#define CAIL_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CAIL_OPS_OK 0
#define CAIL_OPS_EINVAL 1
#define CAIL_OPS_ECUDA 2

/* element types */
#define CAIL_OPS_F32 0
#define CAIL_OPS_BF16 1
#define CAIL_OPS_F16 2

typedef void *cail_ops_stream; /* a cudaStream_t */

/* A [B, T, H, D] array whose last dimension is contiguous. */
typedef struct {
    void *ptr;
    int64_t sb, st, sh; /* strides of B, T and H in elements */
} cail_ops_bthd;

/* Rotary positions on q and k (k.ptr may be NULL).  Pair i of the rotated
 * part (r = `part` elements) turns by pos * turns[i] full turns, scaled by
 * `amplitude`; `inverse` turns back.  Elements from `part` on are copied
 * (nothing when the output is the input).  In place when out.ptr == in.ptr
 * with equal strides; otherwise outputs must not overlap inputs. */
typedef struct {
    int type, B, T, H, Hk, D, part;
    int interleaved, inverse;
    cail_ops_bthd q, k, q_out, k_out;
    const void *positions;  /* int32 or int64, NULL: 0 .. T-1 */
    int positions64;
    int64_t pos_sb, pos_st; /* strides of the positions over B and T */
    const double *turns;    /* [part / 2] */
    float amplitude;
} cail_ops_rotary_args;
int cail_ops_rotary(const cail_ops_rotary_args *a, cail_ops_stream stream);

/* values of lse and of delta: rows of T rounded up to 4, and 64 behind the last (tiles are read whole) */
#define CAIL_OPS_LSE_FLOATS(B, H, T) ((size_t)(B) * (size_t)(H) * (((size_t)(T) + 3) / 4 * 4) + 64)

/* Causal attention with a sliding window and sinks.  Row i sees key j iff
 * i < n, j <= i and (i - j < window or j < sinks), n = lengths[b] (T when
 * lengths is NULL; clamped to [0, T]).  Rows that see nothing give zeros. */
typedef struct {
    int type, B, T, H, Hkv, D;
    int window, sinks;
    float scale;
    const int32_t *lengths;
    cail_ops_bthd q, k, v, o;
    float *lse;             /* CAIL_OPS_LSE_FLOATS(B, H, T) values, 16-byte aligned, kept by forward for
                               backward (B * H rows, T rounded up to 4 apart); NULL: not kept */
    cail_ops_bthd o_rest;   /* 16-bit types: what rounding took from o, in the same type, kept by forward and read by
                               backward (for do.o, which the rounded o alone gives too coarsely); ptr NULL: not kept */
    int rest_rows;          /* o_rest is [B, rest_rows, H, D], of the first rest_rows tokens: cail_ops_rest_rows() */
    /* backward only */
    cail_ops_bthd dout, dq, dk, dv;
    float *delta;           /* scratch of the same size and alignment */
    void *workspace;        /* cail_ops_window_attention_workspace() bytes, 16-byte aligned */
    size_t workspace_bytes;
} cail_ops_attention_args;
/* How many of a sequence's first rows keep what rounding to 16 bits takes from
 * o, and have p rounded to twice the bits.  delta = do.o, on which the
 * gradients of q and k rest, is off where p and o are rounded: for a row of k
 * keys and heads of D that adds about 2 (1/k + 1/D) to the two squared
 * roundings that its gradient has anyway (ds and the result). */
static inline int cail_ops_rest_rows(int T, int D, int window, int sinks) {
    const long long keys = (long long)window + sinks;
    return T <= 128 || keys <= 128 || D < 64 ? T : 128;
}
int cail_ops_window_attention(const cail_ops_attention_args *a, cail_ops_stream stream);
size_t cail_ops_window_attention_workspace(const cail_ops_attention_args *a);
int cail_ops_window_attention_backward(const cail_ops_attention_args *a, cail_ops_stream stream);

/* One token per sequence against a cache: q [B, H, D] (st unused), caches
 * [B, T, Hkv, D]; the query is token lengths[b] - 1 (lengths clamped to
 * [0, T]; 0 gives zeros). */
int cail_ops_window_attention_decode(const cail_ops_attention_args *a, cail_ops_stream stream);

/* Distillation from a teacher's top logits (see cail_b200.ops.distill_loss). */
#define CAIL_OPS_DISTILL_MAX_K 1024
typedef struct {
    int type;               /* of the logits and their gradient */
    int64_t N, V;
    int K;
    const void *logits;     /* [N, V], rows ld_logits apart */
    int64_t ld_logits;
    const void *ids;        /* [N, K] contiguous, int32 or int64; entries outside [0, V) are left out */
    int ids64;
    const void *teacher;    /* [N, K] contiguous, of type teacher_type */
    int teacher_type;
    const int64_t *targets; /* [N] or NULL; a row whose target is outside [0, V) is left out */
    float temperature, hard_weight;
    int mean;               /* 1: mean over the rows that count, 0: sum, -1: none */
    float *rows;            /* [N] losses of the rows */
    float *stats;           /* [N, 8] kept for backward */
    float *loss;            /* one value (mean and sum) */
    float *factor;          /* one value kept for backward: what mean and sum multiply every row by */
    /* backward only */
    const float *grad_loss; /* one value, or N values when mean == -1 */
    void *grad;             /* [N, V], rows ld_grad apart */
    int64_t ld_grad;
} cail_ops_distill_args;
int cail_ops_distill(const cail_ops_distill_args *a, cail_ops_stream stream);
int cail_ops_distill_backward(const cail_ops_distill_args *a, cail_ops_stream stream);

/* The text of this thread's last failure ("" if none). */
const char *cail_ops_last_error(void);

/* The host word that a kernel on the device sets when a bounded wait of its
 * runs out (its results are then wrong); NULL before the first call that
 * launches such a kernel there.  The next call of such a kernel on the device
 * fails with CAIL_OPS_ECUDA, once, and clears the word. */
int *cail_ops_device_error_word(int device);

/* Kernels launched by this process so far (all entry points). */
unsigned long long cail_ops_launches(void);

#ifdef __cplusplus
}
#endif
#endif
