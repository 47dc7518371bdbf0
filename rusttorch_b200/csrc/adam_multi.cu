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
constexpr int kMaxTensors = 400;

struct Table {
  AdamTensor t[kMaxTensors];
  unsigned first[kMaxTensors + 1];   // the tensor's first chunk in the grid
  int n;
  unsigned index0;                   // t[0]'s place in the caller's list
};
static_assert(sizeof(Table) + sizeof(Adam8Coeffs) + 64 <= 32764, "kernel argument limit");

// The tensor that chunk c of the grid belongs to.
__device__ __forceinline__ int tensor_of(const Table& tab, unsigned c) {
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

__global__ void __launch_bounds__(kThreads)
adam_multi_kernel(const __grid_constant__ Table tab, AdamCoeffs c) {
  const int k = tensor_of(tab, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  const size_t begin = (size_t)(blockIdx.x - tab.first[k]) * kChunk;
  const size_t end = min((unsigned long long)begin + kChunk, t.n);
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

// A warp per block of 128 elements, four to a lane.
__global__ void __launch_bounds__(kThreads)
adam8_multi_kernel(const __grid_constant__ Table tab, Adam8Coeffs c, unsigned long long seed) {
  const int k = tensor_of(tab, blockIdx.x);
  const AdamTensor& t = tab.t[k];
  const uint32_t key = tensor_key(seed, tab.index0 + (unsigned)k);
  const size_t begin = (size_t)(blockIdx.x - tab.first[k]) * kChunk;
  const size_t end = min((unsigned long long)begin + kChunk, t.n);
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
        const float p = t.p[i], g = load_as_f32(t.g, t.gtype, i);
        const float root = fmul(decode8(vc[i]), sv);
        nm[u] = fadd(fmul(fmul(decode8(mc[i]), sm), c.b1), fmul(g, c.one_minus_b1));
        r[u] = fsqrt(fadd(fmul(fmul(root, root), c.b2), fmul(fmul(g, g), c.one_minus_b2)));
        const float den = fadd(fmul(r[u], c.c2), c.eps);
        float np = fsub(p, fmul(fdiv(nm[u], den), c.step));
        if (c.decay) np = fsub(np, fmul(p, c.lr_wd));
        t.p[i] = np;
        if (t.copy) store_copy(t.copy, t.ctype, i, np);
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

// Runs launch(table, chunks) over the tensors, kMaxTensors and at most 2^30
// chunks at a time.
template <class F>
cudaError_t for_tables(const AdamTensor* t, size_t n, F launch) {
  Table tab;
  size_t i = 0;
  while (i < n) {
    tab.n = 0;
    tab.index0 = (unsigned)i;
    unsigned chunks = 0;
    for (; i < n && tab.n < kMaxTensors; i++) {
      const unsigned long long need = (t[i].n + kChunk - 1) / kChunk;
      if (chunks && chunks + need > (1u << 30)) break;
      tab.t[tab.n] = t[i];
      tab.first[tab.n++] = chunks;
      chunks += (unsigned)need;
    }
    tab.first[tab.n] = chunks;
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
  return for_tables(t, n, [&](const Table& tab, unsigned chunks) {
    adam_multi_kernel<<<chunks, kThreads, 0, s>>>(tab, c);
    return cudaGetLastError();
  });
}

cudaError_t launch_adam8_multi(const AdamTensor* t, size_t n, const Adam8Coeffs& c, uint64_t seed,
                               cudaStream_t s) {
  return for_tables(t, n, [&](const Table& tab, unsigned chunks) {
    adam8_multi_kernel<<<chunks, kThreads, 0, s>>>(tab, c, seed);
    return cudaGetLastError();
  });
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
