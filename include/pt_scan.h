/*
 * pt_scan.h — C ABI of the gated linear recurrences (gfx950, libptscan.so).
 *
 * The state update of the framework's cells with gates that come from the
 * input alone, so that time can be scanned instead of walked:
 *   leaky  h_t = (1 - s(z_t)) h_{t-1} + s(z_t) n_t,              y_t = h_t
 *          (the update of models/InT.py:166,175 and models/kys.py:46-48)
 *   lstm   c_t = s(f_t) c_{t-1} + s(i_t) tanh(n_t),  y_t = s(o_t) tanh(c_t)
 *          (models/convlstm.py:84-90 without its hidden-to-gate convolutions)
 * with s the logistic function and z, n / i, f, n, o pre-activations, in that
 * order (the gate order i, f, c, o of pt_lstm.h).
 *
 * A sequence tensor is [batch][channels][steps][inner] with any strides over
 * the first three and stride 1 over the last: [B,T,D] has channels = 1 and
 * inner = D, a clip batch [B,C,T,H,W] has inner = H W.  States (h0, h_last,
 * c_last and their gradients) are dense f32 [batch][channels][inner]; inside
 * the kernels the state is always f32.
 *
 * Conventions as pt_cell.h: caller-allocated device buffers, explicit stream,
 * 0 or PT_SCAN_ERR_* with a thread-local message, no state between calls.  No
 * call synchronises; every call can be captured into a graph.  Results do not
 * depend on timing: two runs agree bit for bit.  What a call writes shares no
 * memory with anything else that it is given.
 */
#ifndef PT_SCAN_H
#define PT_SCAN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* pt_scan_stream_t;   /* == hipStream_t */

enum { PT_SCAN_OK = 0, PT_SCAN_ERR_ARG = 1, PT_SCAN_ERR_UNSUPPORTED = 2, PT_SCAN_ERR_HIP = 3 };
enum { PT_SCAN_LEAKY = 0, PT_SCAN_LSTM = 1 };
enum { PT_SCAN_F32 = 0, PT_SCAN_BF16 = 1, PT_SCAN_F16 = 2 };

typedef struct pt_scan_desc {
    int32_t form;       /* PT_SCAN_LEAKY (2 gates) / PT_SCAN_LSTM (4 gates)      */
    int32_t dtype;      /* of x, y and their gradients                           */
    int64_t batch;      /* B >= 1                                                */
    int64_t channels;   /* C >= 1                                                */
    int64_t steps;      /* T, 1 to 2^30                                          */
    int64_t inner;      /* N, 1 to 2^29 - 1                                      */
} pt_scan_desc;
/* A call is one launch of fewer than 2^32 threads; what needs more is refused.  64
 * columns of a row, or what is left of them, take 64 to 1024 threads, or, where there
 * are few, 4 (leaky) or 8 (lstm) a step; an unaligned step takes one a column. */

/* One sequence tensor: element strides over batch, channel and step.  The gates
 * of a call share theirs (as slices of one tensor do), and so do their
 * gradients; x, y and dx may differ from each other. */
typedef struct pt_scan_view {
    void* data;
    int64_t sb, sc, st;
} pt_scan_view;

/* Bytes of `saved`, the states that the backward starts its pieces from. */
size_t pt_scan_saved_bytes(const pt_scan_desc* d);
/* Bytes of the scratch of one call (forward and backward alike); may be 0.  Its
 * contents do not matter, and calls that may run at once need one each. */
size_t pt_scan_workspace_bytes(const pt_scan_desc* d);

/* x: one view per gate.  h0: the state before the first step, or NULL (zeros).
 * lengths: int64 [batch] row ends (taken into [0, T]), or NULL (all T); what
 * stands at or behind a row's end is not read, y is written as 0 there and the
 * state stays.  y: NULL if the sequence is not wanted.  h_last: y of the row's
 * last step (leaky: the last state, h0 for an empty row; lstm: 0 for an empty
 * row); c_last: the last state; either may be NULL.  saved: NULL without a
 * backward. */
int pt_scan_forward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0,
                    const int64_t* lengths, const pt_scan_view* y, float* h_last, float* c_last,
                    void* saved, void* workspace, pt_scan_stream_t stream);

/* Gradients of the forward.  dy, d_h_last, d_c_last: NULL for zero.  dx: one
 * view per gate, written everywhere (0 behind a row's end).  d_h0: may be NULL. */
int pt_scan_backward(const pt_scan_desc* d, const pt_scan_view* x, const float* h0,
                     const int64_t* lengths, const pt_scan_view* dy, const float* d_h_last,
                     const float* d_c_last, const void* saved, const pt_scan_view* dx, float* d_h0,
                     void* workspace, pt_scan_stream_t stream);

/* One step for every row (d->steps = 1): state is read and written in place
 * (f32, strides sb and sc), y is written.  st of the views is not used. */
int pt_scan_step(const pt_scan_desc* d, const pt_scan_view* x, const pt_scan_view* state,
                 const pt_scan_view* y, pt_scan_stream_t stream);

const char* pt_scan_last_error(void);
const char* pt_scan_version(void);

#ifdef __cplusplus
}
#endif
#endif
