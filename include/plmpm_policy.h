/* plmpm_policy.h -- C ABI of the policy-training operators of libplmpm.so.
 *
 * What a policy that is a sequence model needs next to the simulator (include/plmpm.h): a gated linear recurrence (its memory
 * over the horizon), the norms around a block with its gate and residual scale, and an AdamW step over many tensors.  The
 * reference's policy is a per-step MLP in Taichi (plb/engine/nn/mlp.py) trained with a numpy Adam (plb/optimizer/optim.py);
 * there is nothing of this kind to be compatible with.
 *
 * No engine handle: every call takes device pointers and the HIP stream to enqueue on, and the device that owns them has to be
 * the calling thread's current one.  Nothing here synchronises or allocates, so every call can be captured into a graph.
 * Status and errors as in plmpm.h: 0, or non-zero with the text in plmpm_last_error; nothing throws across the boundary.
 * Sizes of zero are accepted and do nothing.
 */
#ifndef PLMPM_POLICY_H
#define PLMPM_POLICY_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum plmpm_nn_dtype { PLMPM_NN_F32 = 0, PLMPM_NN_BF16 = 1, PLMPM_NN_F16 = 2 };

/* ---- gated linear recurrence ---------------------------------------------------------------------------------------------
 *   la_t = -c softplus(decay) sigmoid(r_t),  a_t = exp(la_t)  (0 where reset_t),  m_t = sqrt(1 - a_t^2)
 *   h_t  = a_t h_{t-1} + m_t sigmoid(i_t) x_t
 * x, r, i: [batch][steps][width], unit stride over the width, element strides over batch and steps as given (slices of one
 * projection are read in place).  h and every gradient: contiguous.  decay, h0, h_last, dh0, dlast, ddecay: float.
 * checkpoint: float [ceil(steps / 64)][batch][width], the state each run of 64 steps starts from: written by the forward call
 * if not null, read by the backward call (and a forward call that is given it is refused where that would be).  h0, reset, h_last, dh, dlast, dh0 may be null. */
typedef struct plmpm_scan {
    int32_t dtype, reserved;
    int64_t batch, steps, width;
    int64_t stride_b[3], stride_t[3];       /* of x, r, i */
    double c;
    const void *x, *r, *i;
    const float *decay, *h0;
    const uint8_t* reset;                   /* [batch][steps], contiguous */
    void* h;
    float *h_last, *checkpoint;
    const void* dh;                         /* backward: d loss / d h, contiguous */
    const float* dlast;                     /*           d loss / d h_last */
    void *dx, *dr, *di;
    float *ddecay, *dh0;
    void* workspace;
    size_t workspace_bytes;
} plmpm_scan;
/* bytes of workspace a call needs (any content); its dtype and sizes are looked at, its pointers for their alignment only */
int plmpm_scan_workspace(const plmpm_scan* s, int backward, size_t* bytes);
int plmpm_scan_forward(const plmpm_scan* s, void* hip_stream);
int plmpm_scan_backward(const plmpm_scan* s, void* hip_stream);

/* ---- norms before and after a block, with its gate and residual scale ------------------------------------------------------
 *   y = x + scale * f(gate) * post * u / sqrt(mean(u^2) + eps)          (u null: y = x, and y is not written)
 *   z = pre * y / sqrt(mean(y^2) + eps)                                 (z null: not computed)
 * rows x width; unit stride over the width, row strides as given for x, u, gate, dy, dz; y, z, dx, du, dgate contiguous.
 * x, y, dx, dy: x_dtype; u, gate, z and their gradients: u_dtype; u_dtype is x_dtype, or 16 bits where x_dtype is float.
 * scale, post, pre (and their gradients): [width] of w_dtype; null scale or post count as ones; gate null as ones. */
enum plmpm_gate { PLMPM_GATE_IDENTITY = 0, PLMPM_GATE_SIGMOID = 1, PLMPM_GATE_SILU = 2 };
typedef struct plmpm_norm {
    int32_t x_dtype, u_dtype, w_dtype, gate_fn;
    int64_t rows, width;
    int64_t stride_x, stride_u, stride_gate, stride_dy, stride_dz;
    double eps;
    const void *x, *u, *gate, *scale, *post, *pre;
    void *y, *z;
    const void *dy, *dz;                    /* backward; either may be null (zero) */
    void *dx, *du, *dgate, *dscale, *dpost, *dpre;
    void* workspace;
    size_t workspace_bytes;
} plmpm_norm;
int plmpm_norm_workspace(const plmpm_norm* n, size_t* bytes);      /* of the backward call; the forward needs none */
int plmpm_norm_forward(const plmpm_norm* n, void* hip_stream);
int plmpm_norm_backward(const plmpm_norm* n, void* hip_stream);

/* ---- AdamW over many tensors -----------------------------------------------------------------------------------------------
 *   k = min(1, max_norm / sqrt(sum of g^2 over all tensors)) if max_norm > 0, else 1;   g' = k g
 *   m = beta_1 m + (1 - beta_1) g';  v = beta_2 v + (1 - beta_2) g'^2;   t = updates + 1
 *   w = clip(w - lr weight_decay w - lr / (1 - beta_1^t) m / (sqrt(v / (1 - beta_2^t)) + epsilon), lo, hi)
 * w is the float master where one is given (the 16-bit parameter is then its rounding), else the parameter itself.
 * State of 32 bits: float m, v.  State of 8 bits: blocks of 256 elements with a float scale s, the block's largest magnitude:
 * m = s sign(c) (c / 127)^2 with int8 c, v = s (c / 255)^4 with uint8 c, where a v above zero keeps a code above zero.
 * What a call writes may not overlap anything else of the call, except that a gradient may be its parameter itself. */
typedef struct plmpm_adamw_tensor {
    void* p;
    const void* g;                          /* of the parameter's type */
    void *m, *v;                            /* float, or int8 / uint8 codes */
    float *m_scale, *v_scale;               /* 8 bits: [ceil(n / 256)] */
    float* master;                          /* float copy of a 16-bit parameter, or null */
    int64_t n;
    int32_t dtype, reserved;                /* of p and g; tensors of different types may share a call */
} plmpm_adamw_tensor;
typedef struct plmpm_adamw {
    int32_t state_bits, reserved;
    double lr, beta_1, beta_2, epsilon, weight_decay, max_norm, lo, hi;
    int64_t* step;                          /* device, two words: updates done, updates begun (equal between calls; set the first) */
    float* grad_norm;                       /* device, where max_norm > 0: the norm before clipping; may be null */
    void* workspace;
    size_t workspace_bytes;
} plmpm_adamw;
int plmpm_adamw_workspace(const plmpm_adamw* a, const plmpm_adamw_tensor* tensors, int count, size_t* bytes);
int plmpm_adamw_step(const plmpm_adamw* a, const plmpm_adamw_tensor* tensors, int count, void* hip_stream);
/* read 8-bit state back: out = the values the codes stand for; which: 0 first moment (int8), 1 second (uint8) */
int plmpm_adamw_values(const void* const* codes, const float* const* scales, float* const* out, const int64_t* n, const int32_t* which,
                       int count, void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif /* PLMPM_POLICY_H */
