// One element's AdamW step and the step's scalars: what the kernels over 32-bit moments (adamw.hip) and over 8-bit ones (adamw8.hip) share.
#pragma once
#include "common.h"

namespace {

// The divide form once both bias corrections have become 1.0f (160 steps at beta 0.9, 325 at 0.95): x / 1.0f is x.
constexpr int kFormDiv1 = 2;

template <int FORM>
__device__ __forceinline__ void adamw_elem(float g, float &m, float &v, float &p,
                                           const anc_adamw_hyper_t &h, float wd, float clip) {
  const float gs = g * clip;
  if (FORM == ANC_ADAMW_FORM_DIV) {
    m = h.beta1 * m + h.omb1 * gs;
    v = h.beta2 * v + (h.omb2 * gs) * gs;
    const float mh = m / h.bc1;
    const float vh = v / h.bc2;
    p = p - h.lr * (mh / (sqrtf(vh) + h.eps) + wd * p);
  } else if (FORM == kFormDiv1) {
    m = h.beta1 * m + h.omb1 * gs;
    v = h.beta2 * v + (h.omb2 * gs) * gs;
    p = p - h.lr * (m / (sqrtf(v) + h.eps) + wd * p);
  } else {
    const float o1 = 1.0f - h.beta1, o2 = 1.0f - h.beta2;
    m = h.beta1 * m + o1 * gs;
    v = h.beta2 * v + (o2 * gs) * gs;
    p = p - h.lr * ((m * h.bc1) / (sqrtf(v * h.bc2) + h.eps) + wd * p);
  }
}

__device__ __forceinline__ bool load_ctl(const anc_step_ctl_t *ctl, float &clip) {
  clip = 1.0f;
  if (ctl == nullptr) return true;
  if (ctl->skip != 0u) return false;
  clip = ctl->clip_scale;
  return true;
}

struct RowStep { float bc1, bc2, lr; uint32_t seed_base; };   // anc_adamw_step_t; entry s: counted step s (1-based)

// Steps counted on the device: the bias corrections of step ctl->t from the table the host filled
// ahead (the same fp32 values it would pass per step), the rounding seed from the count itself.
__device__ __forceinline__ void step_scalars(anc_adamw_hyper_t &h, const anc_step_ctl_t *ctl) {
  if (ctl == nullptr) return;
  const uint32_t t = ctl->t;
  if (h.step_table != 0) {
    const uint32_t i = t < 1u ? 1u : (t > (uint32_t)h.step_cap ? (uint32_t)h.step_cap : t);
    const RowStep rs = ((const RowStep *)h.step_table)[i];
    h.bc1 = rs.bc1;
    h.bc2 = rs.bc2;
  }
  if (h.sr & ANC_SR_STEP_SEED) h.seed_base += ANC_SR_SEED_STRIDE * t;
}

}  // namespace

// Turn the runtime (form, sr) pair into template arguments.
template <int V> struct IC { static constexpr int value = V; };
template <typename F> static void dispatch_form_sr(int form, int sr, F &&f) {
  if (form == ANC_ADAMW_FORM_DIV) {
    if (sr) f(IC<ANC_ADAMW_FORM_DIV>{}, IC<1>{}); else f(IC<ANC_ADAMW_FORM_DIV>{}, IC<0>{});
  } else {
    if (sr) f(IC<ANC_ADAMW_FORM_IBC>{}, IC<1>{}); else f(IC<ANC_ADAMW_FORM_IBC>{}, IC<0>{});
  }
}
