// adam_multi.cu — one AdamW step over many tensors in few launches, the
// moments in f32 or in 8 bits.
//
// The tensors' addresses and lengths travel as a kernel argument (at most
// kMaxTensors of them a launch), so a call copies nothing to the device, keeps
// nothing, and can be captured.  Every tensor is cut into chunks of kChunk
// elements, one block each.
#include "rt_adam.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_types.cuh"

#include <cuda_fp8.h>

#include <algorithm>

namespace rt {
namespace {

constexpr int kChunk = 4096;
constexpr int kMaxTensors = 400;   // a launch; a kernel's arguments end at 32,764 bytes
constexpr int kFewTensors = 32;    // short lists travel in a smaller argument

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
__device__ __forceinline__ bool in_fours(const AdamTensor& t, int moment_bytes) {
  auto bits = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  const uintptr_t half = bits(t.copy) | (t.gtype == kF32 ? 0 : bits(t.g));
  const uintptr_t full = bits(t.p) | (t.gtype == kF32 ? bits(t.g) : 0);
  return ((full & 15) | (half & 7) | ((bits(t.m) | bits(t.v)) & (moment_bytes * 4 - 1))) == 0;
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
  if (in_fours(t, 4)) {
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

// The least power of two 2^e with top <= 448 * 2^e, e >= -126.  448 is
// 1.75 * 2^8, so e is top's exponent less 8, one more where its significand
// is above 1.75.  `inv` is 2^-e.
__device__ __forceinline__ void block_scale(float top, float* scale, float* inv) {
  const uint32_t b = f2u(top);
  int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u);
  e = max(e, -126);
  *scale = u2f((uint32_t)(e + 127) << 23);
  *inv = u2f((uint32_t)(127 - e) << 23);
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
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}
// The low half of splitmix64's element i: a tensor's key.
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

// One element's update in f32: its new moment, root and parameter.
__device__ __forceinline__ void adam8_one(const Adam8Coeffs& c, float g, float m, float root,
                                          float& p, float& nm, float& r) {
  nm = fadd(fmul(m, c.b1), fmul(g, c.one_minus_b1));
  r = fsqrt(fadd(fmul(fmul(root, root), c.b2), fmul(fmul(g, g), c.one_minus_b2)));
  const float den = fadd(fmul(r, c.c2), c.eps);
  float np = fsub(p, fmul(fdiv(nm, den), c.step));
  if (c.decay) np = fsub(np, fmul(p, c.lr_wd));
  p = np;
}

// The largest of the warp's sizes (f32 bits without a sign order as integers).
__device__ __forceinline__ uint32_t warp_top(uint32_t bits) {
  return __reduce_max_sync(0xffffffffu, bits);
}

// Two codes, x0's in the low byte, of finite values under a scale, each a sum of
// z's bits and a random number cut to e4m3's fraction.
__device__ __forceinline__ float cut(float y, uint32_t r20, float* bias) {
  const float b = y < 0x1p-6f ? 0x1p-6f : 0.0f;
  *bias = b;
  return u2f((f2u(fadd(y, b)) + r20) & 0xfff00000u);
}
__device__ __forceinline__ uint32_t codes2(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}
// Four codes as f32.
__device__ __forceinline__ float4 decode4(uint32_t w) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(x.x, x.y, y.x, y.y);
}

// A whole block of 128 elements to a warp, four to a lane, U blocks' loads in
// flight.  Where every new moment is finite (the warp's maximum tells) the
// codes need no further question.
template <class G>
__device__ __forceinline__ void adam8_fours(const AdamTensor& t, const Adam8Coeffs& c,
                                            uint32_t key, size_t begin, size_t end) {
  constexpr int U = 2;
  constexpr int kWarps = kThreads / 32;
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* mc = static_cast<uint32_t*>(t.m);
  uint32_t* vc = static_cast<uint32_t*>(t.v);
  for (size_t b0 = begin / kMomentBlock + warp * U; b0 * kMomentBlock < end; b0 += U * kWarps) {
    float4 P[U];
    Grad4<G> g[U];
    uint32_t cm[U], cv[U];
    float sm[U], sv[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      const size_t b = b0 + u, i = b * kMomentBlock + 4 * lane;
      if (b * kMomentBlock < end) {
        P[u] = ld4(t.p + i);
        g[u].load(t.g, i);
        cm[u] = __ldcs(mc + i / 4);
        cv[u] = __ldcs(vc + i / 4);
        sm[u] = t.ms[b];
        sv[u] = t.vs[b];
      }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      const size_t b = b0 + u, i = b * kMomentBlock + 4 * lane;
      if (b * kMomentBlock >= end) break;      // the warp's lanes agree
      const float4 g4 = g[u].get(), m4 = decode4(cm[u]), r4 = decode4(cv[u]);
      const float gs[4] = {g4.x, g4.y, g4.z, g4.w};
      const float ms[4] = {m4.x, m4.y, m4.z, m4.w};
      const float rs[4] = {r4.x, r4.y, r4.z, r4.w};
      float ps[4] = {P[u].x, P[u].y, P[u].z, P[u].w};
      float nm[4], r[4];
#pragma unroll
      for (int e = 0; e < 4; e++)
        adam8_one(c, gs[e], fmul(ms[e], sm[u]), fmul(rs[e], sv[u]), ps[e], nm[e], r[e]);
      const float4 po = make_float4(ps[0], ps[1], ps[2], ps[3]);
      st4(t.p + i, po);
      if (t.copy) store_copy4(t.copy, t.ctype, i, po);
      uint32_t topm = 0, topv = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        topm = max(topm, f2u(nm[e]) & 0x7fffffffu);
        topv = max(topv, f2u(r[e]) & 0x7fffffffu);
      }
      topm = warp_top(topm);
      topv = warp_top(topv);
      const bool fine = topm < 0x7f800000u && topv < 0x7f800000u;
      if (!fine) {
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
      block_scale(u2f(topm), &scale_m, &inv_m);
      block_scale(u2f(topv), &scale_v, &inv_v);
      uint32_t wm = 0, wv = 0;
      const uint32_t counter = key + (uint32_t)i * 0x9E3779B1u + (uint32_t)(i >> 32) * 0xBB67AE85u;
      if (fine) {
        float zm[4], zv[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t h = mix32(counter + e * 0x9E3779B1u);
          float bias;
          const float ym = fmul(fabsf(nm[e]), inv_m);
          zm[e] = cut(ym, (h << 4 & 0xffff0u) | 8u, &bias);
          zm[e] = u2f(f2u(fsub(zm[e], bias)) | (f2u(nm[e]) & 0x80000000u));
          const float yv = fmul(r[e], inv_v);
          zv[e] = cut(yv, (h >> 12 & 0xffff0u) | 8u, &bias);
          zv[e] = fmaxf(fsub(zv[e], bias), r[e] > 0.0f ? 0x1p-9f : 0.0f);
        }
        wm = codes2(zm[0], zm[1]) | codes2(zm[2], zm[3]) << 16;
        wv = codes2(zv[0], zv[1]) | codes2(zv[2], zv[3]) << 16;
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint32_t h = mix32(counter + e * 0x9E3779B1u);
          wm |= (uint32_t)code_of<false>(nm[e], inv_m, true, h & 0xffffu) << (8 * e);
          wv |= (uint32_t)code_of<true>(r[e], inv_v, true, h >> 16) << (8 * e);
        }
      }
      __stcs(mc + i / 4, wm);
      __stcs(vc + i / 4, wv);
      if (lane == 0) {
        t.ms[b] = scale_m;
        t.vs[b] = scale_v;
      }
    }
  }
}

// Blocks of 128 elements from `begin` on, one at a time to a warp: a tensor's
// last one, and tensors that are not aligned.
__device__ void adam8_any(const AdamTensor& t, const Adam8Coeffs& c, uint32_t key, size_t begin,
                          size_t end) {
  unsigned char* mc = static_cast<unsigned char*>(t.m);
  unsigned char* vc = static_cast<unsigned char*>(t.v);
  const unsigned lane = threadIdx.x & 31;
  for (size_t b = begin + (size_t)(threadIdx.x >> 5) * kMomentBlock; b < end;
       b += (kThreads / 32) * kMomentBlock) {
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
    block_scale(warp_max(topm), &scale_m, &inv_m);
    block_scale(warp_max(topv), &scale_v, &inv_v);
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
__global__ void __launch_bounds__(kThreads)
adam8_multi_kernel(const __grid_constant__ Table<CAP> tab, Adam8Coeffs c,
                   unsigned long long seed) {
  const int k = tensor_of(tab, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  const uint32_t key = tensor_key(seed, tab.index0 + (unsigned)k);
  size_t begin = (size_t)(blockIdx.x - tab.first[k]) * kChunk;
  const size_t end = min((unsigned long long)begin + kChunk, t.n);
  if (in_fours(t, 1)) {
    const size_t whole = end - end % kMomentBlock;
    if (t.gtype == kF32) adam8_fours<float>(t, c, key, begin, whole);
    else if (t.gtype == kBF16) adam8_fours<bf16>(t, c, key, begin, whole);
    else adam8_fours<f16>(t, c, key, begin, whole);
    begin = whole;
  }
  adam8_any(t, c, key, begin, end);
}

// A warp per block; v arrives as itself and is stored as its root.
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
    block_scale(warp_max(topm), &scale_m, &inv_m);
    block_scale(warp_max(topv), &scale_v, &inv_v);
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
cudaError_t for_tables(const AdamTensor* t, size_t n, F launch) {
  Table<CAP> tab;
  size_t i = 0;
  while (i < n) {
    tab.n = 0;
    tab.index0 = (unsigned)i;
    unsigned chunks = 0;
    for (; i < n && tab.n < CAP; i++) {
      const unsigned long long need = (t[i].n + kChunk - 1) / kChunk;
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
  return n <= kFewTensors ? for_tables<kFewTensors>(t, n, launch)
                          : for_tables<kMaxTensors>(t, n, launch);
}

cudaError_t launch_adam8_multi(const AdamTensor* t, size_t n, const Adam8Coeffs& c, uint64_t seed,
                               cudaStream_t s) {
  auto launch = [&](const auto& tab, unsigned chunks) {
    adam8_multi_kernel<<<chunks, kThreads, 0, s>>>(tab, c, seed);
    return cudaGetLastError();
  };
  return n <= kFewTensors ? for_tables<kFewTensors>(t, n, launch)
                          : for_tables<kMaxTensors>(t, n, launch);
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
