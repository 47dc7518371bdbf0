// token_loss.cuh — softmax cross entropy of logits against token ids, and its
// gradient.
//
// With M = max_j x_j, o = sum_{j != t} e^(x_j - M) and s = o + e^(x_t - M):
//   loss = log s - (x_t - M), which is log1p(o) where x_t = M,
//   gradient = k e^(x_j - M)/s for j != t and -k o/s for j = t,
// k the upstream gradient (over the count of rows for a mean).  The target's
// term stays out of o, so a token that the model is sure of keeps the digits
// of its small loss and gradient, which 1 - p_t would lose.
//
// HBM bounds it: the gradient call has to read and write each logit once.  So
// there a row stays in shared memory between its statistics and its gradient, over a
// block or a cluster of up to eight, and while the blocks work on one row the
// next one's bytes arrive by bulk copy.  What comes next are the two
// exponentials an element (the SM's special function units give 16 a clock),
// and 12 other instructions (19 for f32, whose gradient's exponentials are
// closer), most of them on pairs.  Measured: 4096 x 32768 f32 170 us (6.3 TB/s; a
// call 176 us, on a GPU that a tenth of a second of them brings to its power
// limit 181 to 186); 8192 x 50257 bf16 316 us (5.2), where the exponentials take
// 183 us of every SM and without them it would be 264 us.
#pragma once
#include "../../include/rusttorch_cuda.h"
#include "rt_chain.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_pairs.cuh"
#include "rt_tma.cuh"
#include "rt_types.cuh"
#include "token_loss.h"

#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

namespace rt {
namespace {

namespace cg = cooperative_groups;

struct Target {
  long long t;     // the class, or -1: none of the row's elements is it
  bool counted;    // takes part in the loss
  bool bad;        // outside the vocabulary
};

__device__ __forceinline__ Target target_of(long long t, long long vocab, long long ignore) {
  if (t == ignore) return {-1, false, false};
  if (t < 0 || t >= vocab) return {-1, true, true};
  return {t, true, false};
}

__device__ __forceinline__ float nan_f() { return u2f(0x7fc00000u); }

// A row's loss from its statistics.
__device__ __forceinline__ float row_loss(float top, float sum, float others, float xt) {
  if (sum != sum) return sum;   // a NaN or +inf in the row, or nothing but -inf
  return xt == top ? log1pf(others) : fsub(logf(sum), fsub(xt, top));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The larger, NaN if one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kLog2e = 1.44269504f;
// log 2 as f32, and what that leaves.
constexpr float kLn2 = 0.693147182f, kLn2Low = -1.90465421e-9f;
// Below this a term is 0, and it bounds what the split below has to hold.
constexpr float kLeast = -128.0f;

// e^d for d = x - m <= 0, rounded once as the difference: with y = fl(d log2 e),
// 2^y times 1 + r, r = d - y log 2 (at most 7e-6, so its square is below 2^-34).
// The hardware's 2^y is within 2^-22 and the last sum rounds once: within
// 2.5 * 2^-23 of e^d; results below 2^-126 are 0.
__device__ __forceinline__ float exp_below(float x, float m) {
  const float d = max_nan(fsub(x, m), kLeast);
  const float y = fmul(d, kLog2e);
  const float r = __fmaf_rn(-y, kLn2Low, __fmaf_rn(-y, kLn2, d));
  const float e = exp2_approx(y);
  return __fmaf_rn(e, r, e);
}
// The two parts of that for a pair: 2^y, not yet multiplied by 1 + r, and r.
__device__ __forceinline__ void exp_parts2(F2 d, float& ea, float& eb, F2& r) {
  const F2 y = f2_mul(d, f2_of(kLog2e, kLog2e));
  r = f2_fma(y, f2_of(-kLn2Low, -kLn2Low), f2_fma(y, f2_of(-kLn2, -kLn2), d));
  f2_to(y, ea, eb);
  ea = exp2_approx(ea);
  eb = exp2_approx(eb);
}
__device__ __forceinline__ F2 exp_below2(F2 x, float m) {
  float a, b;
  f2_to(f2_sum(x, f2_of(-m, -m)), a, b);
  F2 r;
  exp_parts2(f2_of(max_nan(a, kLeast), max_nan(b, kLeast)), a, b, r);
  return f2_fma(f2_of(a, b), r, f2_of(a, b));
}
// The same where a row that holds NaN or +inf is known to be one: the last sum,
// in [0, 1], saturates, which makes 0 of the NaN that r is far below m and so
// needs no kLeast; x that is NaN or +inf gives 0 as well.
__device__ __forceinline__ float fma_sat(float a, float b, float c) {
  float r;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ F2 exp_below2_sat(F2 x, float m) {
  float ea, eb, ra, rb;
  F2 r;
  exp_parts2(f2_sum(x, f2_of(-m, -m)), ea, eb, r);
  f2_to(r, ra, rb);
  return f2_of(fma_sat(ea, ra, ea), fma_sat(eb, rb, eb));
}

// What a row's terms are taken under: its maximum m.  For sums, and for the
// gradient of 16-bit logits (which keeps 12 bits at most), they are 2^(x L - m L)
// for L = log2 e rounded to f32, with m L as `hi`, its f32 value, and the factor
// 2^-lo of the `lo` that leaves, by which a sum of terms or the gradient's
// multiplier is multiplied: one rounding of the exponent (|x - m| 2^-24 of the
// result), L's own (0.23 of that), the hardware's 2^y (2^-22), the factor's and
// the product's (2^-24 each; |lo| <= 2^-4, so five terms of its series are
// within 2^-29): within (0.62 |x - m| + 3.1) 2^-23 of e^(x - m).  In a sum a
// term's share e^(x - m) bounds what that gives.  Where lo could be larger (`wide`:
// |m| >= 2^20, or not a number) they are exp_below2's, and the factor is 1.  The
// gradient of f32 logits has exp_below2_sat's always, since there the error of
// an unlikely class would show (3.7e-6 at 80 below the maximum).
struct Under {
  float m, factor;
  F2 hi;
  bool wide;
};
__device__ __forceinline__ Under under(float m) {
  Under u;
  u.m = m;
  u.wide = !(fabsf(m) < 0x1p20f);
  const float hi = fmul(m, kLog2e);
  const float z = fmul(__fmaf_rn(m, kLog2e, -hi), -kLn2);   // -lo log 2
  const float tail = __fmaf_rn(__fmaf_rn(__fmaf_rn(z, 1.0f / 24, 1.0f / 6), z, 0.5f), z, 1.0f);
  u.factor = u.wide ? 1.0f : __fmaf_rn(tail, z, 1.0f);
  u.hi = f2_of(-hi, -hi);
  return u;
}
template <bool WIDE>
__device__ __forceinline__ F2 term2(F2 x, const Under& u) {
  if constexpr (WIDE) {
    return exp_below2(x, u.m);
  } else {
    float a, b;
    f2_to(f2_fma(x, f2_of(kLog2e, kLog2e), u.hi), a, b);
    return f2_of(exp2_approx(a), exp2_approx(b));
  }
}

// ---- 16 bytes of a row ----------------------------------------------------------

template <class T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
};

// Elements 2i and 2i + 1.
template <class T>
__device__ __forceinline__ F2 pair_of(const Vec<T>& v, int i) {
  if constexpr (sizeof(T) == 4) {
    return f2_of(u2f(v.w[2 * i]), u2f(v.w[2 * i + 1]));
  } else if constexpr (std::is_same<T, bf16>::value) {
    return f2_of(u2f(v.w[i] << 16), u2f(v.w[i] & 0xffff0000u));
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
    return f2_of(f.x, f.y);
  }
}
template <class T>
__device__ __forceinline__ void set_pair(Vec<T>& v, int i, F2 x) {
  float a, b;
  f2_to(x, a, b);
  if constexpr (sizeof(T) == 4) {
    v.w[2 * i] = f2u(a);
    v.w[2 * i + 1] = f2u(b);
  } else if constexpr (std::is_same<T, bf16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

// The largest elements so far, NaN passed over: in pairs for 16-bit types.
template <class T>
struct Top {
  float m = -INFINITY;
  __device__ __forceinline__ void see(const Vec<T>& v) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = fmaxf(m, u2f(v.w[i]));
  }
  __device__ __forceinline__ float get() const { return m; }
};
template <>
struct Top<bf16> {
  __nv_bfloat162 m = {__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80)};
  __device__ __forceinline__ void see(const Vec<bf16>& v) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&v.w[i]));
  }
  __device__ __forceinline__ float get() const { return fmaxf(to_f32(m.x), to_f32(m.y)); }
};
template <>
struct Top<f16> {
  __half2 m = {__ushort_as_half(0xfc00), __ushort_as_half(0xfc00)};
  __device__ __forceinline__ void see(const Vec<f16>& v) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = __hmax2(m, *reinterpret_cast<const __half2*>(&v.w[i]));
  }
  __device__ __forceinline__ float get() const { return fmaxf(to_f32(m.x), to_f32(m.y)); }
};

// Element e of v becomes -inf (under which its term is 0).
template <class T>
__device__ __forceinline__ void drop(Vec<T>& v, int e) {
  constexpr uint32_t kBits = sizeof(T) == 4 ? 0xff800000u
                             : std::is_same<T, bf16>::value ? 0xff80u : 0xfc00u;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      if (e == i) v.w[i] = kBits;
    } else {
      if (e == 2 * i) v.w[i] = (v.w[i] & 0xffff0000u) | kBits;
      if (e == 2 * i + 1) v.w[i] = (v.w[i] & 0xffffu) | kBits << 16;
    }
  }
}

// v's terms, added to `s` pair by pair.
template <bool WIDE, class T>
__device__ __forceinline__ void add_terms(const Vec<T>& v, const Under& u, F2& s) {
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; i++) s = f2_sum(s, term2<WIDE>(pair_of(v, i), u));
}
// v's terms times k (grad_factor), of a row whose k is NaN if it holds NaN or +inf.
template <bool WIDE, class T>
__device__ __forceinline__ Vec<T> scaled_terms(const Vec<T>& v, const Under& u, F2 k) {
  Vec<T> r;
#pragma unroll
  for (int i = 0; i < Vec<T>::N / 2; i++) {
    F2 e;
    if constexpr (sizeof(T) == 4) e = exp_below2_sat(pair_of(v, i), u.m);
    else e = term2<WIDE>(pair_of(v, i), u);
    set_pair(r, i, f2_mul(e, k));
  }
  return r;
}
// k with the factor that scaled_terms leaves out, in both halves.
template <class T>
__device__ __forceinline__ F2 grad_factor(float k, const Under& u) {
  if (sizeof(T) != 4) k = fmul(k, u.factor);
  return f2_of(k, k);
}

// Volatile, so that the compiler keeps the registers instead of loading twice.
template <class T>
__device__ __forceinline__ void load_vec(const T* p, Vec<T>& v) {
  asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3])
               : "l"(p));
}
template <class T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]));
}
// For a p that is not on a 16-byte boundary.
template <class T>
__device__ __forceinline__ void store_elements(T* p, const Vec<T>& v) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      p[i] = u2f(v.w[i]);
    } else {
      reinterpret_cast<uint16_t*>(p)[2 * i] = (uint16_t)v.w[i];
      reinterpret_cast<uint16_t*>(p)[2 * i + 1] = (uint16_t)(v.w[i] >> 16);
    }
  }
}

// A row as elements before its first 16-byte boundary, vectors, and the rest.
struct Split {
  unsigned head, vecs, tail;
};
template <class T>
__device__ __forceinline__ Split split_row(const T* row, unsigned vocab) {
  constexpr unsigned N = Vec<T>::N;
  Split s;
  const unsigned off = reinterpret_cast<uintptr_t>(row) & 15;
  s.head = min((16 - off) % 16 / (unsigned)sizeof(T), vocab);
  s.vecs = (vocab - s.head) / N;
  s.tail = vocab - s.head - s.vecs * N;
  return s;
}

// NaN passed over.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fadd(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// A maximum that terms may be taken against: 0 stands in for -inf, under which
// every term is e^-inf = 0.
__device__ __forceinline__ float against(float m) { return m == -INFINITY ? 0.0f : m; }

// The element of a row's head or tail that thread `self` takes (~0: none).
template <class T>
__device__ __forceinline__ unsigned edge_of(const Split& sp, unsigned self) {
  return self < 8 ? (self < sp.head ? self : ~0u)
         : self < 16 && self - 8 < sp.tail ? sp.head + sp.vecs * Vec<T>::N + (self - 8)
                                           : ~0u;
}

// One thread: a row's loss and statistics.
__device__ __forceinline__ void finish_row(const LossArgs& a, const Target& tg, size_t row,
                                           float top, float sum, float others, float xt) {
  if (tg.bad) atomicExch(a.bad, 1);
  if (a.row_losses)
    a.row_losses[row] = !tg.counted ? 0.0f : tg.bad ? nan_f() : row_loss(top, sum, others, xt);
  if (a.stats) {
    a.stats[3 * row] = top;
    a.stats[3 * row + 1] = sum;
    a.stats[3 * row + 2] = others;
  }
}

// Rows on chip.  A cluster of `blocks` blocks of TH threads (or one block)
// takes a row, and then the next that falls to it; each block has an equal run
// of the row's vectors in shared memory.  Thread 0 asks for the next row's run
// before work on this one begins, into the other of two buffers.
//
// Three walks over the run, a thread always at the same vectors: the maximum
// (then the thread that has the target replaces it by -inf, so that no walk
// asks for it), the sum of the terms, and their gradient.  Between the last two
// every warp's (maximum, sum) goes to every block of the cluster, as
// asynchronous stores that count their bytes at the receiving block's mbarrier:
// no block waits for more than the pairs themselves, where a cluster barrier
// would also drain every warp's memory accesses.  A block can be at most one
// row ahead of another (it needs the other's pairs), so two mbarriers and two
// tables in turn are enough.
template <class T, bool GRAD, int TH, int PER_SM>
__global__ void __launch_bounds__(TH, PER_SM)
row_kernel(const T* logits, LossArgs a, unsigned each) {
  constexpr int N = Vec<T>::N;
  constexpr unsigned kWarps = TH / 32;
  extern __shared__ __align__(128) uint4 runs[];        // [2][run_vecs(PER_SM)]
  __shared__ float2 pairs[2][kMaxCluster * kWarps];
  __shared__ uint64_t arrived[2], loaded[2];
  let_next_kernel_start();
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t clusters = gridDim.x / blocks;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(&arrived[i], 1);
      mbar_init(&loaded[i], 1);
    }
    mbar_fence_init();
  }
  __syncthreads();
  if (blocks > 1) {
    cluster_arrive_relaxed();   // the fence above orders what it has to
    cluster_wait();             // every block runs and its mbarriers are set up
  }

  // A row, and this block's run of it: `each` vectors to a block.
  struct Asked {
    Target tg;
    bool taken;                    // not an ignored one
    unsigned head, begin, count;   // in vectors, behind `head` elements
    unsigned edge;                 // this thread's element of the head or tail, or ~0
    float xe;                      // that element, or -inf
    float xt;                      // the target's logit, or 0
  };
  unsigned asked = 0, seen_loads = 0, turns = 0;
  auto ask = [&](size_t row, long long target) {
    Asked r;
    const T* x = logits + row * (size_t)a.vocab;
    const Split sp = split_row(x, a.vocab);
    r.tg = target_of(target, a.vocab, a.ignore);
    r.taken = r.tg.counted || a.stats;
    r.head = sp.head;
    r.begin = min(rank * each, sp.vecs);
    r.count = min(each, sp.vecs - r.begin);
    r.edge = rank == 0 ? edge_of<T>(sp, threadIdx.x) : ~0u;
    r.xe = -INFINITY;
    r.xt = 0.0f;
    if (!r.taken) return r;
    if (threadIdx.x == 0) {
      uint64_t* bar = &loaded[asked & 1];
      mbar_arrive_expect_tx(bar, r.count * 16);
      if (r.count)
        bulk_load(runs + (asked & 1) * run_vecs(PER_SM), x + sp.head + (size_t)r.begin * N,
                  r.count * 16, bar);
    }
    asked++;
    if (r.edge != ~0u) r.xe = to_f32(x[r.edge]);
    if (r.tg.t >= 0) r.xt = to_f32(x[r.tg.t]);
    return r;
  };

  // Nothing that comes from memory is waited for where it is asked for: the
  // target is read two rows ahead, a row's run and its odd elements one.
  size_t row = blockIdx.x / blocks;
  auto target_at = [&](size_t r) { return r < a.rows ? a.targets[r] : 0; };
  Asked next = {};
  if (row < a.rows) next = ask(row, target_at(row));
  long long ahead = target_at(row + clusters);
  bool fine = true, counted = false;
  float scale = a.grad_scale;
  if (a.count_here && (GRAD || blockIdx.x == 0)) {
    const Count c = count_rows<TH>(a.targets, a.rows, a.ignore);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = c;
    scale = fmul(scale, c.inverse);
    counted = true;
  }
  auto scale_by_count = [&] {
    if (!counted && a.count) {
      wait_for_previous_kernel();
      scale = fmul(scale, a.count->inverse);
    }
    counted = true;
  };
  for (; row < a.rows && fine; row += clusters) {
    const Asked now = next;
    if (row + clusters < a.rows) next = ask(row + clusters, ahead);
    ahead = target_at(row + 2 * clusters);
    const Target tg = now.tg;
    const unsigned count = now.count, edge = now.edge;
    T* g = GRAD ? static_cast<T*>(a.grad) + row * (size_t)a.vocab : nullptr;
    T* gv = GRAD ? g + now.head + (size_t)now.begin * N : nullptr;
    if (!now.taken) {
      // an ignored row: loss and gradient 0
      if (rank == 0 && threadIdx.x == 0 && a.row_losses) a.row_losses[row] = 0.0f;
      if constexpr (GRAD) {
        scale_by_count();
        for (unsigned i = threadIdx.x; i < count; i += TH) {
          if (a.alike) store_vec(gv + (size_t)i * N, Vec<T>{{0, 0, 0, 0}});
          else store_elements(gv + (size_t)i * N, Vec<T>{{0, 0, 0, 0}});
        }
        if (edge != ~0u) g[edge] = from_f32<T>(0.0f);
      }
      continue;
    }
    Vec<T>* run = reinterpret_cast<Vec<T>*>(runs + (seen_loads & 1) * run_vecs(PER_SM));
    fine = mbar_wait(&loaded[seen_loads & 1], (seen_loads >> 1) & 1);
    seen_loads++;
    const float xt = now.xt;

    Top<T> seen;
#pragma unroll 2
    for (unsigned i = threadIdx.x; i < count; i += TH) seen.see(run[i]);
    // The target's logit goes in with every warp, so that it has been read by
    // all of them before a block of the cluster, which needs this warp's pair,
    // may write its gradient in its place.
    const float m = warp_max(fmaxf(fmaxf(seen.get(), now.xe), tg.t >= 0 ? xt : -INFINITY));
    // the target's place: a vector of this thread's, or its odd element
    float xe = now.xe;
    bool owner = false;
    if (tg.t >= 0) {
      const unsigned t = (unsigned)tg.t, vec = (t - now.head) / N;
      if (t == edge) {
        owner = true;
        xe = -INFINITY;
      } else if (t >= now.head && vec - now.begin < count &&
                 (vec - now.begin) % TH == threadIdx.x) {
        owner = true;
        reinterpret_cast<T*>(run + (vec - now.begin))[(t - now.head) % N] = from_f32<T>(-INFINITY);
      }
    }
    const Under um = under(against(m));
    F2 s2 = f2_of(0.0f, 0.0f);
    if (!um.wide) {
#pragma unroll 2
      for (unsigned i = threadIdx.x; i < count; i += TH) add_terms<false>(run[i], um, s2);
    } else {
#pragma unroll 1
      for (unsigned i = threadIdx.x; i < count; i += TH) add_terms<true>(run[i], um, s2);
    }
    float sa, sb;
    f2_to(s2, sa, sb);
    const float s = warp_sum(__fmaf_rn(fadd(sa, sb), um.factor, exp_below(xe, um.m)));

    float top = m, others = s;
    if (TH > 32 || blocks > 1) {
      float2* table = pairs[turns & 1];
      if (blocks > 1) {
        uint64_t* bar = &arrived[turns & 1];
        if (threadIdx.x == 0)
          mbar_arrive_expect_tx(bar, blocks * kWarps * (unsigned)sizeof(float2));
        __syncwarp();
        if (lane < blocks) store_async(&table[rank * kWarps + warp], make_float2(m, s), bar, lane);
        if (!mbar_wait(bar, (turns >> 1) & 1)) fine = false;
      } else {
        if (lane == 0) table[warp] = make_float2(m, s);
        __syncthreads();
      }
      turns++;
      top = -INFINITY;
      others = 0.0f;
      for (unsigned j = lane; j < blocks * kWarps; j += 32) top = fmaxf(top, table[j].x);
      __syncwarp();
      top = warp_max(top);
      for (unsigned j = lane; j < blocks * kWarps; j += 32)
        others = fadd(others, fmul(table[j].y, exp_below(table[j].x, against(top))));
      __syncwarp();
      others = warp_sum(others);
    }
    if (top == -INFINITY) others = nan_f();    // nothing but -inf: terms of e^(-inf + inf)
    const float sum = tg.t >= 0 ? fadd(others, exp_below(xt, top)) : others;
    if (rank == 0 && threadIdx.x == 0) finish_row(a, tg, row, top, sum, others, xt);
    if constexpr (GRAD) {
      scale_by_count();
      // the quotient's roundings (of 1/sum and of the products) are common to
      // the row
      const float k = tg.bad ? nan_f() : fmul(scale, rcp_rn(sum));
      const Under ut = under(top);
      const F2 k2 = grad_factor<T>(k, ut);
      if (a.alike && (sizeof(T) == 4 || !ut.wide) && tg.counted) {
#pragma unroll 2
        for (unsigned i = threadIdx.x; i < count; i += TH)
          store_vec(gv + (size_t)i * N, scaled_terms<false>(run[i], ut, k2));
      } else {
#pragma unroll 1
        for (unsigned i = threadIdx.x; i < count; i += TH) {
          Vec<T> r = Vec<T>{{0, 0, 0, 0}};
          if (tg.counted)
            r = ut.wide ? scaled_terms<true>(run[i], ut, k2) : scaled_terms<false>(run[i], ut, k2);
          if (a.alike) store_vec(gv + (size_t)i * N, r);
          else store_elements(gv + (size_t)i * N, r);
        }
      }
      if (edge != ~0u)
        g[edge] = from_f32<T>(tg.counted ? fmul(exp_below(xe, top), k) : 0.0f);
      // behind this thread's own store of the target's vector
      if (owner) g[tg.t] = from_f32<T>(fmul(-others, k));
    }
    // The buffer is free for the bulk copy after next; a wait that ran out ends
    // the block's rows, for all its threads alike.
    fence_proxy_async_smem();
    fine = __syncthreads_and(fine);
  }
  // the sum, which waits for this kernel alone, reads the count
  if (!GRAD && a.count) wait_for_previous_kernel();
  if (!fine) {
    if (threadIdx.x == 0) atomicExch(a.gave_up, 1);
    // what may still be on its way into this block's shared memory
    for (; seen_loads < asked; seen_loads++)
      mbar_wait(&loaded[seen_loads & 1], (seen_loads >> 1) & 1);
    mbar_wait(&arrived[turns & 1], (turns >> 1) & 1);
  }
}

// Statistics alone: a block of TH walks a row with a running maximum and sum, in
// steps of NV vectors a thread.  (8192 x 50257 bf16: 147 us, 5.6 TB/s; 1024 x
// 600000 f32: 418 us, 5.9 TB/s; 8192 x 50257 with 512 threads: 166 us.)
template <class T, int TH>
__global__ void __launch_bounds__(TH) walk_kernel(const T* logits, LossArgs a) {
  constexpr int N = Vec<T>::N;
  constexpr int kWarps = TH / 32;
  constexpr int NV = 4;
  __shared__ float2 pairs[kWarps];
  let_next_kernel_start();
  const size_t row = blockIdx.x;
  const T* x = logits + row * (size_t)a.vocab;
  const Split sp = split_row(x, a.vocab);
  const Target tg = target_of(a.targets[row], a.vocab, a.ignore);
  const unsigned self = threadIdx.x;
  const unsigned edge = edge_of<T>(sp, self);
  const bool has_edge = edge != ~0u;
  const float xe = has_edge ? to_f32(x[edge]) : -INFINITY;
  const float xt = tg.t >= 0 ? to_f32(x[tg.t]) : 0.0f;
  float m = xe;
  float s = has_edge && (long long)edge != tg.t ? exp_below(xe, against(xe)) : 0.0f;
  for (unsigned i0 = 0; i0 < sp.vecs; i0 += NV * TH) {
    Vec<T> v[NV];
    Top<T> seen;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const unsigned i = i0 + k * TH + self;
      if (i < sp.vecs) load_vec(x + sp.head + (size_t)i * N, v[k]);
    }
#pragma unroll
    for (int k = 0; k < NV; k++)
      if (i0 + k * TH + self < sp.vecs) seen.see(v[k]);
    const float nm = fmaxf(m, seen.get());
    const Under u = under(against(nm));
    const float shrink = exp_below(m, u.m);
    F2 part = f2_of(0.0f, 0.0f);
    m = nm;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const unsigned i = i0 + k * TH + self;
      if (i < sp.vecs) {
        const long long t = tg.t - (long long)sp.head - (long long)i * N;
        if (t >= 0 && t < N) drop(v[k], (int)t);
        if (u.wide) add_terms<true>(v[k], u, part);
        else add_terms<false>(v[k], u, part);
      }
    }
    float pa, pb;
    f2_to(part, pa, pb);
    s = __fmaf_rn(s, shrink, fmul(fadd(pa, pb), u.factor));
  }
  const float wm = warp_max(m);
  const float ws = warp_sum(fmul(s, exp_below(m, against(wm))));
  if ((self & 31) == 0) pairs[self >> 5] = make_float2(wm, ws);
  __syncthreads();
  if (a.count) wait_for_previous_kernel();   // the sum, which waits for this kernel alone, reads it
  if (self >= 32) return;
  const float2 p = self < kWarps ? pairs[self] : make_float2(-INFINITY, 0.0f);
  const float top = warp_max(p.x);
  float others = warp_sum(fmul(p.y, exp_below(p.x, against(top))));
  if (self == 0) {
    if (top == -INFINITY) others = nan_f();
    const float sum = tg.t >= 0 ? fadd(others, exp_below(xt, top)) : others;
    finish_row(a, tg, row, top, sum, others, xt);
  }
}

// The gradient from the statistics: G threads to a row, or `parts` blocks, each
// thread's loads
// under way before the statistics arrive.  HBM bounds it (4096 x 32768 f32:
// 170 us, 6.3 TB/s; 8192 x 50257 bf16: 277 us, 6.0).
template <class T, unsigned G>
__global__ void __launch_bounds__(kThreads)
token_grad_kernel(const T* logits, IndexArray targets, size_t rows, unsigned vocab,
                  long long ignore, const float* stats, const float* upstream, bool per_row,
                  float grad_scale, const Count* count, bool count_here, T* grad, bool alike,
                  unsigned parts, bool chained, int* bad) {
  constexpr int N = Vec<T>::N;
  constexpr int U = 4;
  const size_t row0 = (size_t)(blockIdx.x / parts) * (kThreads / G) + threadIdx.x / G;
  const bool live = G == kThreads || row0 < rows;
  const size_t row = live ? row0 : rows - 1;     // a thread without a row takes part in the count
  const unsigned part = blockIdx.x % parts, self = threadIdx.x % G;
  const T* x = logits + row * (size_t)vocab;
  T* g = grad + row * (size_t)vocab;
  const Split sp = split_row(x, vocab);
  const Target tg = target_of(targets[row], vocab, ignore);
  const unsigned i0 = part * (U * G) + self;
  Vec<T> v[U];
  if (live && tg.counted) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i0 + u * G < sp.vecs) load_vec(x + sp.head + (size_t)(i0 + u * G) * N, v[u]);
  }
  if (chained) wait_for_previous_kernel();
  const float top = stats[3 * row], sum = stats[3 * row + 1], others = stats[3 * row + 2];
  float k = upstream ? upstream[per_row ? row : 0] : grad_scale;
  if (count_here) k = fmul(k, count_rows<kThreads>(targets, rows, ignore).inverse);
  else if (count) k = fmul(k, count->inverse);
  if (!live) return;
  k = tg.bad ? nan_f() : fmul(k, rcp_rn(sum));
  if (tg.bad && part == 0 && self == 0) atomicExch(bad, 1);
  const Under ut = under(top);
  const F2 k2 = grad_factor<T>(k, ut);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const unsigned i = i0 + u * G;
    if (i < sp.vecs) {
      T* p = g + sp.head + (size_t)i * N;
      Vec<T> r = Vec<T>{{0, 0, 0, 0}};
      if (tg.counted)
        r = ut.wide ? scaled_terms<true>(v[u], ut, k2) : scaled_terms<false>(v[u], ut, k2);
      if (alike) store_vec(p, r);
      else store_elements(p, r);
      // the target, behind the store of its vector
      const long long t = tg.t - (long long)sp.head - (long long)i * N;
      if (t >= 0 && t < N) p[t] = from_f32<T>(fmul(-others, k));
    }
  }
  if (part == 0 && self < sp.head + sp.tail) {
    const unsigned j = self < sp.head ? self : sp.vecs * N + self;
    g[j] = from_f32<T>(!tg.counted            ? 0.0f
                       : (long long)j == tg.t ? fmul(-others, k)
                                              : fmul(exp_below(to_f32(x[j]), top), k));
  }
}

template <class T, bool GRAD, int TH, int PER_SM>
cudaError_t rows_of(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  const auto kernel = row_kernel<T, GRAD, TH, PER_SM>;
  const unsigned vecs = (unsigned)vecs_of(t);
  const unsigned blocks = (unsigned)((vecs + run_vecs(PER_SM) - 1) / run_vecs(PER_SM));
  const unsigned each = (vecs + blocks - 1) / blocks;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.stream = s;
  cfg.attrs = attr;
  if (chained) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.blockDim = dim3(TH);
  cfg.dynamicSmemBytes = 2 * run_vecs(PER_SM) * 16;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)cfg.dynamicSmemBytes);
  if (e != cudaSuccess) return e;
  if (blocks > 1) {
    cudaLaunchAttribute& cluster = attr[cfg.numAttrs++];
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = blocks;
    cluster.val.clusterDim.y = 1;
    cluster.val.clusterDim.z = 1;
  }
  // As many clusters as can be resident (asked for once: it depends on how
  // the device's SMs are grouped).
  static std::atomic<int> resident[64][kMaxCluster + 1];
  int most = device < 64 ? resident[device][blocks].load(std::memory_order_relaxed) : 0;
  if (most == 0) {
    if (blocks > 1) {
      cfg.gridDim = dim3(blocks);
      e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
    } else {
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kernel, TH, cfg.dynamicSmemBytes);
      most *= sm_count(device);
    }
    if (e != cudaSuccess) return e;
    most = std::max(1, most);
    if (device < 64) resident[device][blocks].store(most, std::memory_order_relaxed);
  }
  cfg.gridDim = dim3((unsigned)(std::min<size_t>(a.rows, (size_t)most) * blocks));
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(t.logits), a, each);
}

// The fewest threads that hold the row alone; longer rows go to clusters of
// two blocks to an SM, and of one where eight of those are too few.
template <class T, bool GRAD>
cudaError_t rows_by_size(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  switch (row_threads(t)) {
    case 32: return rows_of<T, GRAD, 32, 16>(t, a, chained, s);
    case 64: return rows_of<T, GRAD, 64, 8>(t, a, chained, s);
    case 128: return rows_of<T, GRAD, 128, 4>(t, a, chained, s);
    case 256: {
      // Three blocks to an SM where that puts more rows on it than two do, for
      // 16-bit types (8192 x 32768 bf16: 207 us for 239; at 50257 both put one
      // there, and three take 322 us for 312).  f32, whose time is HBM's, stays
      // with two (4096 x 32768: 178 us for 190 with three, a call).
      const size_t two = (vecs_of(t) + run_vecs(2) - 1) / run_vecs(2);
      const size_t three = (vecs_of(t) + run_vecs(3) - 1) / run_vecs(3);
      if (sizeof(T) == 2 && three <= kMaxCluster && 3 * two > 2 * three)
        return rows_of<T, GRAD, 256, 3>(t, a, chained, s);
      return rows_of<T, GRAD, 256, 2>(t, a, chained, s);
    }
    default: return rows_of<T, GRAD, 512, 1>(t, a, chained, s);
  }
}

template <class T>
cudaError_t walk_rows(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  if (t.rows > kMaxGrid) return cudaErrorInvalidValue;
  const size_t vecs = vecs_of(t);
  // threads for two steps at least
  const auto kernel = vecs <= 4096    ? walk_kernel<T, 128>
                      : vecs <= 16384 ? walk_kernel<T, 256> : walk_kernel<T, 512>;
  const unsigned threads = vecs <= 4096 ? 128 : vecs <= 16384 ? 256 : 512;
  const T* x = static_cast<const T*>(t.logits);
  if (chained) return launch_after(kernel, (unsigned)t.rows, threads, 0, s, x, a);
  kernel<<<(unsigned)t.rows, threads, 0, s>>>(x, a);
  return cudaGetLastError();
}

// Statistics and losses of every row, and the gradient unless it is null.
template <class T>
cudaError_t rows_any(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  if (walks_rows(t, a.grad)) return walk_rows<T>(t, a, chained, s);
  return a.grad ? rows_by_size<T, true>(t, a, chained, s)
                : rows_by_size<T, false>(t, a, chained, s);
}

template <class T, unsigned G>
cudaError_t grad_by(const TokenLoss& a, const float* stats, const float* upstream,
                    float grad_scale, const Count* count, bool count_here, void* grad,
                    bool chained, cudaStream_t s) {
  const size_t parts = std::max<size_t>(1, (vecs_of(a) + 4 * G - 1) / (4 * G));
  const size_t step = std::max<size_t>(1, kMaxGrid / parts);
  const bool alike =
      ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(a.logits)) & 15) == 0;
  for (size_t r0 = 0; r0 < a.rows; r0 += step) {
    const size_t rows = std::min(a.rows - r0, step);
    const size_t off = r0 * a.vocab;
    const size_t tsize = a.wide ? 8 : 4;
    const bool per_row = a.reduction == RTC_REDUCE_NONE;
    const IndexArray targets{static_cast<const char*>(a.targets) + r0 * tsize, a.wide};
    const T* x = static_cast<const T*>(a.logits) + off;
    T* g = static_cast<T*>(grad) + off;
    const float* up = upstream && per_row ? upstream + r0 : upstream;
    const unsigned grid = (unsigned)((rows + kThreads / G - 1) / (kThreads / G) * parts);
    cudaError_t e;
    if (chained && r0 == 0) {
      e = launch_after(token_grad_kernel<T, G>, grid, kThreads, 0, s, x, targets, rows,
                       (unsigned)a.vocab, a.ignore, stats, up, per_row, grad_scale, count,
                       count_here, g, alike, (unsigned)parts, true, a.bad);
    } else {
      token_grad_kernel<T, G><<<grid, kThreads, 0, s>>>(
          x, targets, rows, (unsigned)a.vocab, a.ignore, stats + 3 * r0, up, per_row, grad_scale,
          count, count_here, g, alike, (unsigned)parts, false, a.bad);
      e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Four vectors a thread; a warp at least to a row (16384 x 200 f32: 14 us, and
// 39 us with a block to each).
template <class T>
cudaError_t grad_of(const TokenLoss& a, const float* stats, const float* upstream,
                    float grad_scale, const Count* count, bool count_here, void* grad,
                    bool chained, cudaStream_t s) {
  const size_t vecs = vecs_of(a);
  const auto by = vecs <= 128   ? grad_by<T, 32>
                  : vecs <= 256 ? grad_by<T, 64>
                  : vecs <= 512 ? grad_by<T, 128> : grad_by<T, kThreads>;
  return by(a, stats, upstream, grad_scale, count, count_here, grad, chained, s);
}

}  // namespace

// The instances for one storage type are compiled in a file of their own.
#define RT_TOKEN_LOSS_TYPE(T, NAME)                                                             \
  cudaError_t token_rows_##NAME(const TokenLoss& t, const LossArgs& a, bool chained,            \
                                cudaStream_t s) {                                               \
    return rows_any<T>(t, a, chained, s);                                                       \
  }                                                                                             \
  cudaError_t token_grad_##NAME(const TokenLoss& t, const float* stats, const float* upstream,  \
                                float grad_scale, const Count* count, bool count_here,          \
                                void* grad, bool chained, cudaStream_t s) {                     \
    return grad_of<T>(t, stats, upstream, grad_scale, count, count_here, grad, chained, s);     \
  }

}  // namespace rt
