// adam_multi.cu — one AdamW step over many tensors in few launches, the
// moments in f32 or in 8 bits.
//
// The tensors' addresses and lengths travel as a kernel argument (at most
// kMaxTensors of them a launch), so a call copies nothing to the device, keeps
// nothing, and can be captured.  Every tensor is cut into chunks of kChunk
// elements, one block each (f32), or units of kUnit (8 bits).
//
// HBM bounds the f32 step (139 M elements in 194 tensors: 605 us, 6.4 TB/s).
// With 8-bit moments instructions do, before HBM (417 M elements, bf16 gradients
// and copies: 1.34 ms, 5.0 TB/s).
#include "rt_adam.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_pairs.cuh"
#include "rt_tma.cuh"
#include "rt_types.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace rt {
namespace {

constexpr int kChunk = 4096;       // elements to a block, moments in f32
constexpr int kMaxTensors = 400;   // a launch; a kernel's arguments end at 32,764 bytes
constexpr int kFewTensors = 32;    // shorter lists travel in a smaller argument
constexpr int kSomeTensors = 128;

template <int CAP>
struct Table {
  AdamTensor t[CAP];
  unsigned first[CAP];   // the tensor's first chunk in the grid
  int n;
  unsigned index0;       // t[0]'s place in the caller's list
};
static_assert(sizeof(Table<kMaxTensors>) + sizeof(Adam8Coeffs) + 64 <= 32764,
              "kernel argument limit");

// The tensor that chunk c of the grid belongs to.
template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP>& tab, unsigned c) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float load_as_f32(const void* p, StoreType t, size_t i) {
  switch (t) {
    case kF32: return static_cast<const float*>(p)[i];
    case kBF16: return to_f32(static_cast<const bf16*>(p)[i]);
    default: return to_f32(static_cast<const f16*>(p)[i]);
  }
}
__device__ __forceinline__ void store_copy(void* p, StoreType t, size_t i, float x) {
  if (t == kBF16) static_cast<bf16*>(p)[i] = from_f32<bf16>(x);
  else static_cast<f16*>(p)[i] = from_f32<f16>(x);
}

// Four elements from a boundary of four (16, or 8, bytes).
__device__ __forceinline__ float4 ld4(const float* p) {
  return __ldcs(reinterpret_cast<const float4*>(p));
}
__device__ __forceinline__ void st4(float* p, float4 v) {
  __stcs(reinterpret_cast<float4*>(p), v);
}
// Gradients as they are stored, and as f32.
template <class G>
struct Grad4 {
  uint2 w;
  __device__ __forceinline__ void load(const void* p, size_t i) {
    w = __ldcs(reinterpret_cast<const uint2*>(static_cast<const G*>(p) + i));
  }
  __device__ __forceinline__ void load_shared(const void* p, unsigned i) {
    w = *reinterpret_cast<const uint2*>(static_cast<const G*>(p) + i);
  }
  __device__ __forceinline__ float4 get() const {
    const G* x = reinterpret_cast<const G*>(&w);
    return make_float4(to_f32(x[0]), to_f32(x[1]), to_f32(x[2]), to_f32(x[3]));
  }
};
template <>
struct Grad4<float> {
  float4 v;
  __device__ __forceinline__ void load(const void* p, size_t i) {
    v = ld4(static_cast<const float*>(p) + i);
  }
  __device__ __forceinline__ void load_shared(const void* p, unsigned i) {
    v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
  }
  __device__ __forceinline__ float4 get() const { return v; }
};
__device__ __forceinline__ void store_copy4(void* p, StoreType t, size_t i, float4 v) {
  uint2 w;
  if (t == kBF16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  __stcs(reinterpret_cast<uint2*>(static_cast<bf16*>(p) + i), w);
}

// Whether four elements of every list are one access each.
__device__ __forceinline__ bool in_fours(const AdamTensor& t) {
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const uintptr_t half = bits(t.copy) | (t.gtype == kF32 ? 0 : bits(t.g));
  const uintptr_t full = bits(t.p) | (t.gtype == kF32 ? bits(t.g) : 0);
  return (((full | bits(t.m) | bits(t.v)) & 15) | (half & 7)) == 0;
}

// Whether a unit of every list of the 8-bit moments can be copied in bulk, and
// its copies written four at a time.
__device__ __forceinline__ bool in_sixteens(const AdamTensor& t) {
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  return (((bits(t.p) | bits(t.g) | bits(t.m) | bits(t.v)) & 15) | (bits(t.copy) & 7)) == 0;
}

// Elements [begin, end) of a chunk, four at a time, two fours of each list in
// flight; begin is a multiple of four.
template <class G>
__device__ __forceinline__ void adam_fours(const AdamTensor& t, const AdamCoeffs& c, size_t begin,
                                           size_t end) {
  constexpr int U = 2;
  float* m = static_cast<float*>(t.m);
  float* v = static_cast<float*>(t.v);
  for (size_t i0 = begin + 4 * threadIdx.x; i0 < end; i0 += 4 * U * kThreads) {
    float4 P[U], M[U], V[U];
    Grad4<G> g[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const size_t i = i0 + 4 * u * kThreads;
      if (i < end) {
        P[u] = ld4(t.p + i);
        g[u].load(t.g, i);
        M[u] = ld4(m + i);
        V[u] = ld4(v + i);
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const size_t i = i0 + 4 * u * kThreads;
      if (i < end) {
        const float4 G4 = g[u].get();
        float4 po, mo, vo;
        adam1(c, P[u].x, G4.x, M[u].x, V[u].x, po.x, mo.x, vo.x);
        adam1(c, P[u].y, G4.y, M[u].y, V[u].y, po.y, mo.y, vo.y);
        adam1(c, P[u].z, G4.z, M[u].z, V[u].z, po.z, mo.z, vo.z);
        adam1(c, P[u].w, G4.w, M[u].w, V[u].w, po.w, mo.w, vo.w);
        st4(t.p + i, po);
        st4(m + i, mo);
        st4(v + i, vo);
        if (t.copy) store_copy4(t.copy, t.ctype, i, po);
      }
    }
  }
}

template <int CAP>
__global__ void __launch_bounds__(kThreads)
adam_multi_kernel(const __grid_constant__ Table<CAP> tab, AdamCoeffs c) {
  const int k = tensor_of(tab, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  size_t begin = (size_t)(blockIdx.x - tab.first[k]) * kChunk;
  const size_t end = min((unsigned long long)begin + kChunk, t.n);
  if (in_fours(t)) {
    const size_t fours = end & ~size_t(3);
    if (t.gtype == kF32) adam_fours<float>(t, c, begin, fours);
    else if (t.gtype == kBF16) adam_fours<bf16>(t, c, begin, fours);
    else adam_fours<f16>(t, c, begin, fours);
    begin = fours;
  }
  float* m = static_cast<float*>(t.m);
  float* v = static_cast<float*>(t.v);
  for (size_t i = begin + threadIdx.x; i < end; i += kThreads) {
    float p, mo, vo;
    adam1(c, t.p[i], load_as_f32(t.g, t.gtype, i), m[i], v[i], p, mo, vo);
    t.p[i] = p;
    m[i] = mo;
    v[i] = vo;
    if (t.copy) store_copy(t.copy, t.ctype, i, p);
  }
}

// ------------------------------------------------------------ 8-bit moments

__device__ __forceinline__ float decode8(unsigned char c) {
  __nv_fp8_e4m3 x;
  x.__x = c;
  return static_cast<float>(x);
}
// |z| <= 448 or NaN; exact where z is one of the format's values.
__device__ __forceinline__ unsigned char encode8(float z) {
  return __nv_cvt_float_to_fp8(z, __NV_SATFINITE, __NV_E4M3);
}

// The least power of two 2^e with top <= 448 * 2^e, e >= -126, and 2^-e, from
// top's bits.  448 is 1.75 * 2^8, so e is top's exponent less 8, one more
// where its fraction is above 0.75: adding 0x1fffff carries exactly there.
__device__ __forceinline__ void block_scale(uint32_t top, float* scale, float* inv) {
  const uint32_t e = max((top + 0x1fffffu) >> 23, 9u) - 8u;   // biased
  *scale = u2f(e << 23);
  *inv = u2f((254u - e) << 23);
}

// The size an element contributes to its block's scale: 0 if not finite.
__device__ __forceinline__ float finite_size(float x) {
  const float a = u2f(f2u(x) & 0x7fffffffu);
  return a < INFINITY ? a : 0.0f;
}

// x under the block's 2^-e, rounded to e4m3: up with the probability of the
// part cut off (`bits16` of 2^16), or to nearest.  The 20 low bits of a
// normal f32 are what e4m3's 3-bit fraction cuts off; adding random bits there
// and truncating is the rounding, its carry the step to the next value.  The
// format's subnormals have one spacing, that of [2^-6, 2^-5): 2^-6 is added
// to put them there.
__device__ __forceinline__ float round_stochastic(float y, uint32_t bits16) {
  const bool low = y < 0x1p-6f;
  float z = low ? fadd(y, 0x1p-6f) : y;
  z = u2f((f2u(z) + (bits16 << 4) + 8u) & 0xfff00000u);
  return low ? fsub(z, 0x1p-6f) : z;
}
template <bool LEAST>
__device__ __forceinline__ unsigned char code_of(float x, float inv, bool stochastic,
                                                 uint32_t bits16) {
  const float a = u2f(f2u(x) & 0x7fffffffu);
  const float y = fmul(a, inv);
  float z = stochastic ? round_stochastic(y, bits16) : y;
  unsigned char c = encode8(z);
  if (LEAST && c == 0 && a > 0.0f) c = 1;
  if (!(a < INFINITY)) c = 0x7f;
  return c | (unsigned char)((f2u(x) >> 24) & 0x80u);
}

// 32 random bits of a counter: multiplications by odd constants (the
// fractions of sqrt 2 and sqrt 3) between shifts.
__device__ __forceinline__ uint32_t mix32_high(uint32_t x) {   // its high half
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  return (x ^ (x >> 15)) * 0xBB67AE85u;
}
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = mix32_high(x);
  return x ^ (x >> 16);
}
// Element i of Steele, Lea and Flood's splittable generator (2014), its low
// half: a tensor's key.
__device__ __forceinline__ uint32_t tensor_key(unsigned long long seed, unsigned long long i) {
  unsigned long long z = seed + (i + 1) * 0x9E3779B97F4A7C15ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (uint32_t)(z ^ (z >> 31));
}
__device__ __forceinline__ uint32_t element_bits(uint32_t key, size_t i) {
  return mix32(key + (uint32_t)i * 0x9E3779B1u + (uint32_t)(i >> 32) * 0xBB67AE85u);
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}

// 1/x within an ulp (x >= 2^-126; 0 from 2^126 on): the step's quotient is
// within 2 ulp, a 2^-22 part of what a step moves a parameter, whose moments
// have 4 bits.  IEEE division took 9 of 87 instructions an element.
__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// One element's update in f32: its new moment, root and parameter.
__device__ __forceinline__ void adam8_one(const Adam8Coeffs& c, float g, float m, float root,
                                          float& p, float& nm, float& r) {
  nm = fadd(fmul(m, c.b1), fmul(g, c.one_minus_b1));
  r = fsqrt(fadd(fmul(fmul(root, root), c.b2), fmul(fmul(g, g), c.one_minus_b2)));
  const float den = fadd(fmul(r, c.c2), c.eps);
  const float np = fsub(p, fmul(fmul(nm, reciprocal(den)), c.step));
  p = fsub(np, fmul(p, c.lr_wd));
}

// The largest of the warp's sizes (f32 bits without a sign order as integers).
__device__ __forceinline__ uint32_t warp_top(uint32_t bits) {
  return __reduce_max_sync(0xffffffffu, bits);
}

__device__ __forceinline__ uint32_t codes2(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}
// Codes 2i and 2i + 1 of four as f32.
__device__ __forceinline__ F2 decode2(uint32_t w, int i) {
  uint32_t h;
  const uint16_t c = (uint16_t)(w >> (16 * i));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return f2_of(x.x, x.y);
}
// The smallest of three sizes, NaN if one is.
__device__ __forceinline__ float small_of(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// ---- units of 2048 elements through shared memory
// A producer warp brings a unit's parameters, gradients and codes into one of
// kStages buffers by bulk copy; the consumer warps take two blocks of 128
// elements each from there and write back to memory themselves.
constexpr int kUnit = 2048;
constexpr int kStages = 3;
constexpr int kConsumers = 8;                       // warps
constexpr int kUnitThreads = 32 * (kConsumers + 1);
constexpr int kUnitBlocks = kUnit / kMomentBlock;

// What the consumers need to know of a unit.
struct Unit8 {
  float* p;
  uint32_t *mc, *vc;      // four codes each
  float *ms, *vs;
  void* copy;
  const AdamTensor* t;
  size_t begin, end;      // in the tensor
  uint32_t whole;         // elements of whole blocks, which are in the buffer
  uint32_t key, counter;  // of the tensor, and of the unit's first element
};
struct Stage8 {
  float4 p[kUnit / 4];
  uint4 g[kUnit / 4];     // f32 at most
  uint32_t mc[kUnit / 4], vc[kUnit / 4];
  float sm[kUnitBlocks], sv[kUnitBlocks];
  Unit8 unit;
  uint64_t full, empty;
};

// One whole block, four elements to a lane.  At 16 bytes an element the step
// is bound by instructions before HBM (417 M elements in 1.34 ms, 72 for each), so
// arithmetic that allows it goes in pairs, and where all of a lane's new values
// are finite and in the format's normal range its rounding asks no question.
template <class G, int COPY>
__device__ __forceinline__ void adam8_block(const Stage8& st, const Adam8Coeffs& c, F2 one,
                                            unsigned blk, unsigned lane) {
  const Unit8& u = st.unit;
  const unsigned o = blk * kMomentBlock + 4 * lane;
  const float4 p4 = st.p[o / 4];
  Grad4<G> gr;
  gr.load_shared(st.g, o);
  const uint32_t cm = st.mc[o / 4], cv = st.vc[o / 4];
  const float sm = st.sm[blk], sv = st.sv[blk];
  const float4 g4 = gr.get();
  const F2 gs[2] = {f2_of(g4.x, g4.y), f2_of(g4.z, g4.w)};
  const F2 ps[2] = {f2_of(p4.x, p4.y), f2_of(p4.z, p4.w)};
  float nm[4], r[4];
  float4 po;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const F2 g = gs[h];
    const F2 m = f2_mul(decode2(cm, h), f2_of(sm, sm));
    const F2 root = f2_mul(decode2(cv, h), f2_of(sv, sv));
    const F2 m2 = f2_add(f2_mul(m, f2_of(c.b1, c.b1)),
                         f2_mul(g, f2_of(c.one_minus_b1, c.one_minus_b1)), one);
    const F2 v2 = f2_add(f2_mul(f2_mul(root, root), f2_of(c.b2, c.b2)),
                         f2_mul(f2_mul(g, g), f2_of(c.one_minus_b2, c.one_minus_b2)), one);
    float va, vb, da, db;
    f2_to(m2, nm[2 * h], nm[2 * h + 1]);
    f2_to(v2, va, vb);
    r[2 * h] = fsqrt(va);
    r[2 * h + 1] = fsqrt(vb);
    f2_to(f2_add(f2_mul(f2_of(r[2 * h], r[2 * h + 1]), f2_of(c.c2, c.c2)), f2_of(c.eps, c.eps),
                 one),
          da, db);
    const F2 q = f2_mul(m2, f2_of(reciprocal(da), reciprocal(db)));
    // a - b*c as a + b*(-c): the same rounding
    F2 np = f2_add(f2_mul(q, f2_of(-c.step, -c.step)), ps[h], one);
    np = f2_add(f2_mul(ps[h], f2_of(-c.lr_wd, -c.lr_wd)), np, one);
    if (h == 0) f2_to(np, po.x, po.y);
    else f2_to(np, po.z, po.w);
  }
  st4(u.p + o, po);
  if constexpr (COPY == 1) store_copy4(u.copy, kBF16, o, po);
  if constexpr (COPY == 2) store_copy4(u.copy, kF16, o, po);
  // maxima of sizes (as bits; NaN passed over unless nothing else is there)
  uint32_t topm =
      warp_top(f2u(fmaxf(max3(fabsf(nm[0]), fabsf(nm[1]), fabsf(nm[2])), fabsf(nm[3]))));
  uint32_t topv = warp_top(f2u(fmaxf(max3(r[0], r[1], r[2]), r[3])));
  const bool odd = topm >= 0x7f800000u || topv >= 0x7f800000u;   // an infinity, or only NaN
  if (odd) {
    topm = topv = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      topm = max(topm, f2u(finite_size(nm[e])));
      topv = max(topv, f2u(finite_size(r[e])));
    }
    topm = warp_top(topm);
    topv = warp_top(topv);
  }
  float scale_m, inv_m, scale_v, inv_v;
  block_scale(topm, &scale_m, &inv_m);
  block_scale(topv, &scale_v, &inv_v);
  float ym[4], yv[4];
  f2_to(f2_mul(f2_of(nm[0], nm[1]), f2_of(inv_m, inv_m)), ym[0], ym[1]);
  f2_to(f2_mul(f2_of(nm[2], nm[3]), f2_of(inv_m, inv_m)), ym[2], ym[3]);
  f2_to(f2_mul(f2_of(r[0], r[1]), f2_of(inv_v, inv_v)), yv[0], yv[1]);
  f2_to(f2_mul(f2_of(r[2], r[3]), f2_of(inv_v, inv_v)), yv[2], yv[3]);
  const float least = small_of(small_of(small_of(ym[0], ym[1], ym[2]), ym[3], yv[0]),
                               yv[1], small_of(yv[2], yv[3], yv[3]));
  uint32_t wm = 0, wv = 0;
  const uint32_t counter = u.counter + o * 0x9E3779B1u;
  if (least >= 0x1p-6f && !odd) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t h = mix32_high(counter + e * 0x9E3779B1u);
      const uint32_t high = h >> 12;
      // the rounding is an addition and a mask; the sign stays
      ym[e] = u2f((f2u(ym[e]) + ((h << 4 ^ high) & 0xffff0u) + 8u) & 0xfff00000u);
      yv[e] = u2f((f2u(yv[e]) + (high & 0xffff0u) + 8u) & 0xfff00000u);
    }
    wm = codes2(ym[0], ym[1]) | codes2(ym[2], ym[3]) << 16;
    wv = codes2(yv[0], yv[1]) | codes2(yv[2], yv[3]) << 16;
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const uint32_t h = mix32(counter + e * 0x9E3779B1u);
      wm |= (uint32_t)code_of<false>(nm[e], inv_m, true, h & 0xffffu) << (8 * e);
      wv |= (uint32_t)code_of<true>(r[e], inv_v, true, h >> 16) << (8 * e);
    }
  }
  __stcs(u.mc + o / 4, wm);
  __stcs(u.vc + o / 4, wv);
  if (lane == 0) {
    u.ms[blk] = scale_m;
    u.vs[blk] = scale_v;
  }
}

template <class G>
__device__ __forceinline__ void adam8_unit(const Stage8& st, const Adam8Coeffs& c, unsigned warp,
                                           unsigned lane) {
  const F2 one = f2_of(c.one, c.one);
  const unsigned blocks = st.unit.whole / kMomentBlock;
  if (!st.unit.copy) {
    for (unsigned b = warp; b < blocks; b += kConsumers) adam8_block<G, 0>(st, c, one, b, lane);
  } else if (st.unit.t->ctype == kBF16) {
    for (unsigned b = warp; b < blocks; b += kConsumers) adam8_block<G, 1>(st, c, one, b, lane);
  } else {
    for (unsigned b = warp; b < blocks; b += kConsumers) adam8_block<G, 2>(st, c, one, b, lane);
  }
}

// Blocks of 128 elements from `begin` on, one at a time to a warp: a tensor's
// last one, and tensors that are not aligned.
__device__ void adam8_any(const AdamTensor& t, const Adam8Coeffs& c, uint32_t key, size_t begin,
                          size_t end, unsigned warp, unsigned lane) {
  unsigned char* mc = static_cast<unsigned char*>(t.m);
  unsigned char* vc = static_cast<unsigned char*>(t.v);
  for (size_t b = begin + (size_t)warp * kMomentBlock; b < end; b += kConsumers * kMomentBlock) {
    const size_t blk = b / kMomentBlock;
    const float sm = t.ms[blk], sv = t.vs[blk];
    float nm[4], r[4], topm = 0.0f, topv = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const size_t i = b + u * 32 + lane;
      nm[u] = r[u] = 0.0f;
      if (i < end) {
        float p = t.p[i];
        adam8_one(c, load_as_f32(t.g, t.gtype, i), fmul(decode8(mc[i]), sm),
                  fmul(decode8(vc[i]), sv), p, nm[u], r[u]);
        t.p[i] = p;
        if (t.copy) store_copy(t.copy, t.ctype, i, p);
        topm = fmaxf(topm, finite_size(nm[u]));
        topv = fmaxf(topv, finite_size(r[u]));
      }
    }
    float scale_m, inv_m, scale_v, inv_v;
    block_scale(f2u(warp_max(topm)), &scale_m, &inv_m);
    block_scale(f2u(warp_max(topv)), &scale_v, &inv_v);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const size_t i = b + u * 32 + lane;
      if (i < end) {
        const uint32_t bits = element_bits(key, i);
        mc[i] = code_of<false>(nm[u], inv_m, true, bits & 0xffffu);
        vc[i] = code_of<true>(r[u], inv_v, true, bits >> 16);
      }
    }
    if (lane == 0) {
      t.ms[blk] = scale_m;
      t.vs[blk] = scale_v;
    }
  }
}

template <int CAP>
__global__ void __launch_bounds__(kUnitThreads, 3)
adam8_multi_kernel(const __grid_constant__ Table<CAP> tab, Adam8Coeffs c, unsigned long long seed,
                   unsigned units, int* gave_up) {
  extern __shared__ __align__(128) unsigned char shared[];
  Stage8* stages = reinterpret_cast<Stage8*>(shared);
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; s++) {
      mbar_init(&stages[s].full, 1);
      mbar_init(&stages[s].empty, kConsumers);
    }
    mbar_fence_init();
  }
  __syncthreads();
  unsigned turn = 0;
  bool fine = true;
  if (warp == kConsumers) {
    for (unsigned u = blockIdx.x; u < units && fine; u += gridDim.x, turn++) {
      Stage8& st = stages[turn % kStages];
      if (turn >= kStages) fine = mbar_wait(&st.empty, (turn / kStages - 1) & 1);
      if (!fine) break;
      const int k = tensor_of(tab, u);
      const AdamTensor& t = tab.t[k];
      const size_t begin = (size_t)(u - tab.first[k]) * kUnit;
      const size_t end = min((unsigned long long)begin + kUnit, t.n);
      const unsigned n = (unsigned)(end - begin);
      const unsigned whole = in_sixteens(t) ? n - n % kMomentBlock : 0;
      // the scales by plain loads: a unit's last ones need not fill 16 bytes
      if (lane < whole / kMomentBlock) {
        st.sm[lane] = t.ms[begin / kMomentBlock + lane];
        st.sv[lane] = t.vs[begin / kMomentBlock + lane];
      }
      if (lane == 0) {
        const uint32_t key = tensor_key(seed, tab.index0 + (unsigned)k);
        st.unit.p = t.p + begin;
        st.unit.mc = static_cast<uint32_t*>(t.m) + begin / 4;
        st.unit.vc = static_cast<uint32_t*>(t.v) + begin / 4;
        st.unit.ms = t.ms + begin / kMomentBlock;
        st.unit.vs = t.vs + begin / kMomentBlock;
        st.unit.copy = t.copy ? static_cast<char*>(t.copy) + begin * 2 : nullptr;
        st.unit.t = &t;
        st.unit.begin = begin;
        st.unit.end = end;
        st.unit.whole = whole;
        st.unit.key = key;
        // a unit begins at a multiple of its size: the high half of the
        // element's number is the same for all of it
        st.unit.counter =
            key + (uint32_t)begin * 0x9E3779B1u + (uint32_t)(begin >> 32) * 0xBB67AE85u;
      }
      __syncwarp();
      if (lane == 0) {
        const size_t gsize = t.gtype == kF32 ? 4 : 2;
        mbar_arrive_expect_tx(&st.full, whole * (unsigned)(4 + gsize + 2));
        if (whole) {
          bulk_load(st.p, t.p + begin, whole * 4, &st.full);
          bulk_load(st.g, static_cast<const char*>(t.g) + begin * gsize, whole * (unsigned)gsize,
                    &st.full);
          bulk_load(st.mc, static_cast<const char*>(t.m) + begin, whole, &st.full);
          bulk_load(st.vc, static_cast<const char*>(t.v) + begin, whole, &st.full);
        }
      }
    }
    // no copy may be on its way when the block ends: the consumers wait for
    // each, or gave up
  } else {
    for (unsigned u = blockIdx.x; u < units && fine; u += gridDim.x, turn++) {
      Stage8& st = stages[turn % kStages];
      fine = mbar_wait(&st.full, (turn / kStages) & 1);
      if (!fine) break;
      const AdamTensor& t = *st.unit.t;
      if (t.gtype == kF32) adam8_unit<float>(st, c, warp, lane);
      else if (t.gtype == kBF16) adam8_unit<bf16>(st, c, warp, lane);
      else adam8_unit<f16>(st, c, warp, lane);
      if (st.unit.begin + st.unit.whole < st.unit.end)
        adam8_any(t, c, st.unit.key, st.unit.begin + st.unit.whole, st.unit.end, warp, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&st.empty);
    }
  }
  if (!fine) {
    if (lane == 0) atomicExch(gave_up, 1);
    for (int s = 0; s < kStages; s++, turn++)
      mbar_wait(&stages[turn % kStages].full, (turn / kStages) & 1);
  }
}

// A warp per block; v arrives as itself and is stored as its root.  (2^27
// elements: 520 us, and 377 us back, for 209 at the copy's rate: both once in a
// training run's start.)
__global__ void __launch_bounds__(kThreads)
adam8_pack_kernel(const float* m, const float* v, unsigned char* mc, float* ms, unsigned char* vc,
                  float* vs, size_t n) {
  const unsigned lane = threadIdx.x & 31;
  const size_t blocks = (n + kMomentBlock - 1) / kMomentBlock;
  for (size_t blk = ((size_t)blockIdx.x * kThreads + threadIdx.x) >> 5; blk < blocks;
       blk += (size_t)gridDim.x * (kThreads / 32)) {
    float x[4], r[4], topm = 0.0f, topv = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const size_t i = blk * kMomentBlock + u * 32 + lane;
      x[u] = i < n ? m[i] : 0.0f;
      r[u] = i < n ? fsqrt(v[i]) : 0.0f;
      topm = fmaxf(topm, finite_size(x[u]));
      topv = fmaxf(topv, finite_size(r[u]));
    }
    float scale_m, inv_m, scale_v, inv_v;
    block_scale(f2u(warp_max(topm)), &scale_m, &inv_m);
    block_scale(f2u(warp_max(topv)), &scale_v, &inv_v);
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const size_t i = blk * kMomentBlock + u * 32 + lane;
      if (i < n) {
        mc[i] = code_of<false>(x[u], inv_m, false, 0);
        vc[i] = code_of<true>(r[u], inv_v, false, 0);
      }
    }
    if (lane == 0) {
      ms[blk] = scale_m;
      vs[blk] = scale_v;
    }
  }
}

__global__ void __launch_bounds__(kThreads)
adam8_unpack_kernel(const unsigned char* mc, const float* ms, const unsigned char* vc,
                    const float* vs, float* m, float* v, size_t n) {
  for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < n;
       i += (size_t)gridDim.x * kThreads) {
    const float r = fmul(decode8(vc[i]), vs[i / kMomentBlock]);
    m[i] = fmul(decode8(mc[i]), ms[i / kMomentBlock]);
    v[i] = fmul(r, r);
  }
}

// Runs launch(table, chunks) over the tensors, CAP and at most 2^30 chunks at
// a time.
template <int CAP, class F>
cudaError_t for_tables(const AdamTensor* t, size_t n, size_t chunk, F launch) {
  Table<CAP> tab;
  size_t i = 0;
  while (i < n) {
    tab.n = 0;
    tab.index0 = (unsigned)i;
    unsigned chunks = 0;
    for (; i < n && tab.n < CAP; i++) {
      const unsigned long long need = (t[i].n + chunk - 1) / chunk;
      if (chunks && chunks + need > (1u << 30)) break;
      tab.t[tab.n] = t[i];
      tab.first[tab.n++] = chunks;
      chunks += (unsigned)need;
    }
    if (chunks) {
      const cudaError_t e = launch(tab, chunks);
      if (e != cudaSuccess) return e;
    }
  }
  return cudaSuccess;
}

unsigned grid_of(size_t units, size_t per_block) {
  return (unsigned)std::min<size_t>((units + per_block - 1) / per_block, 1u << 16);
}

}  // namespace

cudaError_t launch_adam_multi(const AdamTensor* t, size_t n, const AdamCoeffs& c, cudaStream_t s) {
  auto launch = [&](const auto& tab, unsigned chunks) {
    adam_multi_kernel<<<chunks, kThreads, 0, s>>>(tab, c);
    return cudaGetLastError();
  };
  return n <= kFewTensors    ? for_tables<kFewTensors>(t, n, kChunk, launch)
         : n <= kSomeTensors ? for_tables<kSomeTensors>(t, n, kChunk, launch)
                             : for_tables<kMaxTensors>(t, n, kChunk, launch);
}

namespace {
template <int CAP>
cudaError_t adam8_by_tables(const AdamTensor* t, size_t n, const Adam8Coeffs& c, uint64_t seed,
                            int* gave_up, cudaStream_t s) {
  const auto kernel = adam8_multi_kernel<CAP>;
  const int smem = kStages * (int)sizeof(Stage8);
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return for_tables<CAP>(t, n, kUnit, [&](const Table<CAP>& tab, unsigned units) {
    const unsigned grid = std::min(units, 3u * (unsigned)sm_count(device));
    kernel<<<grid, kUnitThreads, smem, s>>>(tab, c, seed, units, gave_up);
    return cudaGetLastError();
  });
}
}  // namespace

cudaError_t launch_adam8_multi(const AdamTensor* t, size_t n, const Adam8Coeffs& c, uint64_t seed,
                               int* gave_up, cudaStream_t s) {
  return n <= kFewTensors    ? adam8_by_tables<kFewTensors>(t, n, c, seed, gave_up, s)
         : n <= kSomeTensors ? adam8_by_tables<kSomeTensors>(t, n, c, seed, gave_up, s)
                             : adam8_by_tables<kMaxTensors>(t, n, c, seed, gave_up, s);
}

cudaError_t launch_adam8_pack(const float* m, const float* v, void* mc, float* ms, void* vc,
                              float* vs, size_t n, cudaStream_t s) {
  if (n == 0) return cudaSuccess;
  adam8_pack_kernel<<<grid_of(n, kThreads * 4), kThreads, 0, s>>>(
      m, v, static_cast<unsigned char*>(mc), ms, static_cast<unsigned char*>(vc), vs, n);
  return cudaGetLastError();
}

cudaError_t launch_adam8_unpack(const void* mc, const float* ms, const void* vc, const float* vs,
                                float* m, float* v, size_t n, cudaStream_t s) {
  if (n == 0) return cudaSuccess;
  adam8_unpack_kernel<<<grid_of(n, kThreads), kThreads, 0, s>>>(
      static_cast<const unsigned char*>(mc), ms, static_cast<const unsigned char*>(vc), vs, m, v,
      n);
  return cudaGetLastError();
}

}  // namespace rt
