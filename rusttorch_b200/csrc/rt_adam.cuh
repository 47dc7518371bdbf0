// rt_adam.cuh — the element rule of Adam and AdamW, shared by the one-tensor
// and the many-tensor kernels.
#pragma once
#include "rt_internal.h"
#include "rt_libm.cuh"

namespace rt {

// One Adam/AdamW element, in the order of optimizer.rs:293-309 and :413-421.
__device__ __forceinline__ void adam1(const AdamCoeffs& c, float p, float g, float m, float v,
                                      float& po, float& mo, float& vo) {
  const float nm = fadd(fmul(m, c.b1), fmul(g, c.one_minus_b1));
  const float nv = fadd(fmul(v, c.b2), fmul(fmul(g, g), c.one_minus_b2));
  const float mh = fdiv(nm, c.bc1);
  const float vh = fdiv(nv, c.bc2);
  const float den = fadd(fsqrt(vh), c.eps);
  float np = fsub(p, fmul(fdiv(mh, den), c.lr));
  if (c.decay) np = fsub(np, fmul(p, c.lr_wd));
  po = np;
  mo = nm;
  vo = nv;
}

}  // namespace rt
