/* C ABI of the operators that the models are trained with: group normalisation
 * with its activation, the distillation loss, the gated projection.  Device
 * pointers; strides and counts in elements; dtype values are those of
 * stdml/bits/collective/dtype.hpp (8: bf16, 9: f16, 10: f32).  Every function
 * enqueues on `stream` of GPU `device` and returns the codes of capi_cuda.h;
 * stdmlc_last_error() has the message.  Nothing here allocates or synchronises. */
#ifndef STDML_COLLECTIVE_CAPI_TRAIN_H
#define STDML_COLLECTIVE_CAPI_TRAIN_H
#ifdef __cplusplus
extern "C" {
#endif

enum {
    STDMLC_ACT_NONE = 0,
    STDMLC_ACT_RELU = 1,
    STDMLC_ACT_SILU = 2,
    STDMLC_ACT_GELU = 3,
    STDMLC_ACT_GELU_TANH = 4,
};

/* A matrix of images: element (n, s, c) at n * image + s * row + c. */
typedef struct {
    void *ptr;
    long long image, row;
} stdmlc_rows;

/* y = act(xh * weight + bias [+ residual]), xh the values of a group of channels of an
 * image less their mean, over their standard deviation. */
typedef struct {
    stdmlc_rows x, residual, y; /* residual.ptr null: none */
    const void *weight, *bias;  /* null: one, zero */
    double *stats;              /* [images][groups][2]: mean, 1 / sqrt(var + eps) */
    long long images, positions;
    int channels, groups, dt, weight_dt, act;
    double eps;
    /* backward only; null: not wanted */
    stdmlc_rows dy, dx, dresidual;
    void *dweight, *dbias; /* weight_dt */
    void *workspace;       /* stdmlc_norm_workspace() bytes */
} stdmlc_norm;

/* How many bytes of workspace a call with these sizes (and operands and results, as far as they are set) takes on the
 * current GPU; -1: undefined sizes, or no GPU. */
long long stdmlc_norm_workspace(const stdmlc_norm *a, int backward);
int stdmlc_norm_forward(const stdmlc_norm *a, int device, void *stream);
int stdmlc_norm_backward(const stdmlc_norm *a, int device, void *stream);

/* Per row: alpha * CE(z, label) + (1 - alpha) * t^2 * KL(teacher || softmax(z / t)); without
 * labels t^2 * KL.  The teacher's distribution is that of `top` logits at `index`; an index
 * outside [0, classes) is no entry.  A row counts where its label lies in [0, classes) or, without
 * labels, where the teacher has an entry; other rows give zero. */
typedef struct {
    const void *logits; /* row r at r * logits_row */
    long long logits_row;
    const void *top;
    const void *index;  /* 32 or 64 bits, as index_bytes says */
    const void *labels; /* null: none; 64 bits */
    long long ignore;
    long long rows, classes, top_row, index_row;
    int top_count, dt, top_dt, index_bytes;
    float temperature, alpha;
    int reduction;     /* 0: each row, 1: sum, 2: mean over the rows that count */
    float *loss;       /* one value, or one of each row */
    float *row_stats;  /* [rows][5]: maximum, the two sums, the teacher's maximum, weight of the row */
    void *workspace;   /* stdmlc_distill_workspace() bytes */
    /* backward */
    const float *dloss; /* one value, or one of each row (dloss_row apart) */
    long long dloss_row;
    /* rows x classes, packed.  In a forward call (bf16 and f32, reductions to one value): null, or where to write the
     * gradient of the loss.  In a backward call where to write it; with `written` it has the forward call's already, which
     * is what a loss of gradient one wants, and is written again for another. */
    void *dlogits;
    int written;
} stdmlc_distill;

long long stdmlc_distill_workspace(const stdmlc_distill *a);
int stdmlc_distill_forward(const stdmlc_distill *a, int device, void *stream);
int stdmlc_distill_backward(const stdmlc_distill *a, int device, void *stream);
long long stdmlc_stream_capturing(void *stream); /* the number of the capture that it is in; 0: none */

/* h = act(g) * u, g = x w_gate^T + b_gate, u = x w_up^T + b_up. */
typedef struct {
    const void *x; /* tokens x hidden */
    long long x_row;
    const void *w_gate, *w_up; /* ffn x hidden */
    long long w_gate_row, w_up_row;
    const void *b_gate, *b_up; /* both or none */
    void *h;                   /* tokens x ffn, packed */
    long long tokens, hidden, ffn;
    int dt, act;
    void *saved;     /* stdmlc_gated_saved() bytes for the backward pass; null: none follows */
    void *workspace; /* stdmlc_gated_workspace() bytes */
    /* backward; a null result is not computed */
    const void *dh;
    long long dh_row;
    void *dx, *dw_gate, *dw_up, *db_gate, *db_up; /* packed */
    /* How long a wait inside a kernel may last before it gives up, which stdmlc_train_status() reports.  0: ten
     * seconds; negative: none may, and nothing is computed (a call of more than four tokens, or backward, gives up at once). */
    long long wait_limit_ns;
} stdmlc_gated;

long long stdmlc_gated_saved(const stdmlc_gated *a);
long long stdmlc_gated_workspace(const stdmlc_gated *a, int backward);
int stdmlc_gated_forward(const stdmlc_gated *a, int device, void *stream);
int stdmlc_gated_backward(const stdmlc_gated *a, int device, void *stream);

/* Waits for all of the GPU's work, on whatever stream (so not while one is captured).  *out: 0, or 1 where a bounded wait of an operator has run out since the last
 * question (its results are not complete). */
int stdmlc_train_status(int device, int *out);

#ifdef __cplusplus
}
#endif
#endif
