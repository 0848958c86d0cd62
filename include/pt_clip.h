/*
 * pt_clip.h — C ABI of the gradient norm and clipping (gfx950, libptclip.so).
 *
 * The reference's clip_grad_norm_ (utils/misc_functions.py:48-69) over a list
 * of tensors of any sizes and types, in two launches for every 192 to 320 of them:
 *   N = (sum over all elements |g|^p)^(1/p)  (p = 1, 2; inf: the largest |g|)
 *   k = min(1, max_norm / (N + 1e-6)),  out = k g
 * Sums are held in 64 bits, so that squares of f32 neither overflow nor
 * vanish, and are added in an order that depends on the sizes alone: two calls
 * on the same numbers agree bit for bit.  A NaN or an infinite norm goes into
 * k as the formula has it (NaN: every output NaN; infinite: k = 0).
 *
 * Conventions as pt_cell.h: caller-allocated device buffers, explicit stream,
 * 0 or PT_CLIP_ERR_* with a thread-local message, no state between calls.  No
 * call synchronises; every call can be captured into a graph.
 */
#ifndef PT_CLIP_H
#define PT_CLIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* pt_clip_stream_t;   /* == hipStream_t */

enum { PT_CLIP_OK = 0, PT_CLIP_ERR_ARG = 1, PT_CLIP_ERR_UNSUPPORTED = 2, PT_CLIP_ERR_HIP = 3 };
enum { PT_CLIP_F32 = 0, PT_CLIP_BF16 = 1, PT_CLIP_F16 = 2 };
enum { PT_CLIP_INF = 0, PT_CLIP_L1 = 1, PT_CLIP_L2 = 2 };

/* n elements each, dense in any order, aligned to their elements. */
typedef struct pt_clip_tensor {
    const void* grad;
    void* out;            /* grad itself (in place), or memory that no tensor shares */
    int64_t n;            /* >= 0; pointers of empty tensors are not looked at       */
    int32_t grad_type;
    int32_t out_type;     /* grad_type or PT_CLIP_F32                                */
} pt_clip_tensor;

/* Bytes of the scratch of one call over these tensors. */
size_t pt_clip_workspace_bytes(const pt_clip_tensor* t, int64_t count);

/* norm (f32 [1], on the device) = N. */
int pt_clip_norm(const pt_clip_tensor* t, int64_t count, int norm_type, float* norm, void* workspace,
                 pt_clip_stream_t stream);

/* norm = N, out = k grad.  All in place and k = 1, no tensor is touched.
 * Refused: an out that overlaps another tensor, or its own grad other than
 * exactly; max_norm below 0 or NaN. */
int pt_clip_grads(const pt_clip_tensor* t, int64_t count, int norm_type, double max_norm, float* norm,
                  void* workspace, pt_clip_stream_t stream);

const char* pt_clip_last_error(void);
const char* pt_clip_version(void);

#ifdef __cplusplus
}
#endif
#endif
