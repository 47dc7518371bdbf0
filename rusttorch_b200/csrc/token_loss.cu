// token_loss.cu — softmax cross entropy of logits against token ids, and its
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
// a row stays in registers between its statistics and its gradient: up to
// kMaxVec 16-byte vectors a thread, over a warp, a block or a cluster of up to
// eight blocks, whichever holds the row.  Each warp reduces its own part to a
// maximum and a sum under that maximum; one exchange of these pairs through
// (distributed) shared memory gives every warp M and o, in the same order.
#include "../../include/rusttorch_cuda.h"
#include "rt_chain.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_types.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace rt {
namespace {

namespace cg = cooperative_groups;

struct Target {
  long long t;     // the class, or -1: none of the row's elements is it
  bool counted;    // takes part in the loss
  bool bad;        // outside the vocabulary
};

__device__ __forceinline__ Target target_of(const IndexArray& targets, size_t row, long long vocab,
                                            long long ignore) {
  const long long t = targets[row];
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

// e^(x - m), m >= x: the difference, its product with log2 e and the
// hardware's 2^y (2 ulp) each round once, so the result is within
// (|x - m| + 2) 2^-23 of itself; results below 2^-126 are 0.
__device__ __forceinline__ float exp_below(float x, float m) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmul(fsub(x, m), 1.44269504f)));
  return r;
}

// ---- 16 bytes of a row ----------------------------------------------------------

template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
};

template <class T>
__device__ __forceinline__ void unpack(const Vec<T>& v, float (&x)[Vec<T>::N]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      x[i] = u2f(v.w[i]);
    } else if constexpr (std::is_same<T, bf16>::value) {
      x[2 * i] = u2f(v.w[i] << 16);
      x[2 * i + 1] = u2f(v.w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

template <class T>
__device__ __forceinline__ Vec<T> pack(const float (&x)[Vec<T>::N]) {
  Vec<T> v;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if constexpr (sizeof(T) == 4) {
      v.w[i] = f2u(x[i]);
    } else if constexpr (std::is_same<T, bf16>::value) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      v.w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return v;
}

// The largest element of v and of m, NaN passed over.
template <class T>
__device__ __forceinline__ float max_of(const Vec<T>& v, float m) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; i++) m = fmaxf(m, u2f(v.w[i]));
    return m;
  } else {
    float x[Vec<T>::N];
    unpack<T>(v, x);
#pragma unroll
    for (int i = 0; i < Vec<T>::N; i++) m = fmaxf(m, x[i]);
    return m;
  }
}

template <class T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
  return {{v.x, v.y, v.z, v.w}};
}
template <class T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]));
}

// A row as elements before its first 16-byte boundary, vectors, and the rest.
struct Split {
  unsigned head, vecs, tail;
};
template <class T>
__device__ __forceinline__ Split split_row(const T* row, unsigned vocab) {
  constexpr unsigned N = Vec<T>::N;
  Split s;
  s.head = min((unsigned)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (unsigned)sizeof(T),
               vocab);
  s.vecs = (vocab - s.head) / N;
  s.tail = vocab - s.head - s.vecs * N;
  return s;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fadd(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// A maximum that terms may be taken against: 0 stands in for -inf, under which
// every term is e^-inf = 0.
__device__ __forceinline__ float against(float m) { return m == -INFINITY ? 0.0f : m; }

struct LossArgs {
  IndexArray targets;
  size_t row0, rows;
  unsigned vocab;
  long long ignore;
  float* row_losses;                   // [rows of the call]
  float* stats;                        // null, or [rows, 3]
  void* grad;                          // null, or the gradient
  float grad_scale;
  const unsigned long long* count;     // null, or what a mean divides by
  int* bad;
  bool alike;                          // grad's rows start where logits' do, modulo 16 bytes
};

constexpr int kMaxVec = 8;

// One row over all the threads that hold it: `threads` of them, this one
// `self`; `exchange` turns a warp's (maximum, sum) into the row's.
template <class T, int NV, bool GRAD, class X>
__device__ __forceinline__ void row_in_registers(const T* logits, const LossArgs& a, size_t row,
                                                 unsigned threads, unsigned self, X exchange) {
  constexpr int N = Vec<T>::N;
  const T* x = logits + row * (size_t)a.vocab;
  const Split sp = split_row(x, a.vocab);
  const Target tg = target_of(a.targets, row, a.vocab, a.ignore);
  const bool skip = !tg.counted && !a.stats;      // nothing but zeros to write
  Vec<T> v[NV];
#pragma unroll
  for (int k = 0; k < NV; k++) {
    const unsigned i = k * threads + self;
    if (i < sp.vecs && !skip) v[k] = load_vec(x + sp.head + (size_t)i * N);
  }
  // head and tail: an element each for the first threads
  const unsigned edge = self < 8 ? (self < sp.head ? self : ~0u)
                        : self < 16 && self - 8 < sp.tail ? sp.head + sp.vecs * N + (self - 8)
                                                          : ~0u;
  const bool has_edge = edge != ~0u;
  const float xe = has_edge ? to_f32(x[edge]) : -INFINITY;
  const float xt = tg.t >= 0 ? to_f32(x[tg.t]) : 0.0f;
  // which of this thread's vectors holds the target, and where
  const unsigned tv = (unsigned)tg.t - sp.head;
  const bool t_in_vec = tg.t >= (long long)sp.head && tv / N < sp.vecs;
  const int t_slot = t_in_vec && tv / N % threads == self ? (int)(tv / N / threads) : -1;
  const int t_elem = (int)(tv % N);
  const bool t_edge = has_edge && (long long)edge == tg.t;

  float m = -INFINITY, s = 0.0f;
  if (!skip) {
    m = xe;
#pragma unroll
    for (int k = 0; k < NV; k++)
      if (k * threads + self < sp.vecs) m = max_of<T>(v[k], m);
    m = warp_max(m);
    const float ms = against(m);
#pragma unroll
    for (int k = 0; k < NV; k++) {
      if (k * threads + self < sp.vecs) {
        float f[N];
        unpack<T>(v[k], f);
        if (k == t_slot) {
#pragma unroll
          for (int e = 0; e < N; e++)
            if (e == t_elem) f[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < N; e++) s = fadd(s, exp_below(f[e], ms));
      }
    }
    if (has_edge && !t_edge) s = fadd(s, exp_below(xe, ms));
    s = warp_sum(s);
  }
  const float2 r = exchange(m, s);
  const float top = r.x;
  // nothing but -inf: the sums are of e^(-inf + inf)
  const float others = top == -INFINITY ? nan_f() : r.y;
  const float sum = tg.t >= 0 ? fadd(others, exp_below(xt, top)) : others;
  if (self == 0) {
    if (tg.bad) atomicExch(a.bad, 1);
    if (a.row_losses)
      a.row_losses[row] = !tg.counted ? 0.0f : tg.bad ? nan_f() : row_loss(top, sum, others, xt);
    if (a.stats) {
      a.stats[3 * row] = top;
      a.stats[3 * row + 1] = sum;
      a.stats[3 * row + 2] = others;
    }
  }
  if constexpr (GRAD) {
    float k = a.grad_scale;
    if (a.count) {
      wait_for_previous_kernel();
      k = fdiv(k, (float)*a.count);
    }
    k = tg.bad ? nan_f() : fdiv(k, sum);
    const float at_target = fmul(-others, k);
    T* g = static_cast<T*>(a.grad) + row * (size_t)a.vocab;
#pragma unroll
    for (int j = 0; j < NV; j++) {
      const unsigned i = j * threads + self;
      if (i < sp.vecs) {
        float f[N];
        if (tg.counted) {
          unpack<T>(v[j], f);
#pragma unroll
          for (int e = 0; e < N; e++) f[e] = fmul(exp_below(f[e], top), k);
          if (j == t_slot) {
#pragma unroll
            for (int e = 0; e < N; e++)
              if (e == t_elem) f[e] = at_target;
          }
        } else {
#pragma unroll
          for (int e = 0; e < N; e++) f[e] = 0.0f;
        }
        T* p = g + sp.head + (size_t)i * N;
        if (a.alike) {
          store_vec(p, pack<T>(f));
        } else {
#pragma unroll
          for (int e = 0; e < N; e++) p[e] = from_f32<T>(f[e]);
        }
      }
    }
    if (has_edge)
      g[edge] = from_f32<T>(!tg.counted ? 0.0f
                            : t_edge    ? at_target
                                        : fmul(exp_below(xe, top), k));
  }
}

// A warp to a row: rows of at most 32 * NV vectors.
template <class T, int NV, bool GRAD>
__global__ void __launch_bounds__(kThreads) warp_row_kernel(const T* logits, LossArgs a) {
  let_next_kernel_start();
  const size_t i = (size_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (i >= a.rows) return;
  row_in_registers<T, NV, GRAD>(logits, a, a.row0 + i, 32, threadIdx.x & 31,
                                [](float m, float s) { return make_float2(m, s); });
}

// A cluster of `blocks` blocks (or one block) to a row.
constexpr int kRowThreads = 512;
constexpr int kMaxCluster = 8;
template <class T, int NV, bool GRAD>
__global__ void __launch_bounds__(kRowThreads, 2) cluster_row_kernel(const T* logits, LossArgs a) {
  constexpr int kWarps = kRowThreads / 32;
  __shared__ float2 pairs[kMaxCluster * kWarps];
  let_next_kernel_start();
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (blocks > 1) cluster.barrier_arrive();
  auto exchange = [&](float m, float s) {
    // every warp's pair into every block's table, once every block runs
    if (blocks > 1) cluster.barrier_wait();
    if (lane < blocks)
      *cluster.map_shared_rank(&pairs[rank * kWarps + warp], lane) = make_float2(m, s);
    if (blocks > 1) cluster.sync();
    else __syncthreads();
    float2 p[kMaxCluster * kWarps / 32];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMaxCluster * kWarps / 32; k++) {
      const unsigned j = k * 32 + lane;
      p[k] = j < blocks * kWarps ? pairs[j] : make_float2(-INFINITY, 0.0f);
      top = fmaxf(top, p[k].x);
    }
    top = warp_max(top);
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kMaxCluster * kWarps / 32; k++)
      sum = fadd(sum, fmul(p[k].y, exp_below(p[k].x, against(top))));
    return make_float2(top, warp_sum(sum));
  };
  row_in_registers<T, NV, GRAD>(logits, a, a.row0 + blockIdx.x / blocks, blocks * kRowThreads,
                                rank * kRowThreads + threadIdx.x, exchange);
}

// Rows that no cluster holds: a block walks the row with a running maximum and
// sum, in steps of kMaxVec vectors a thread.
template <class T>
__global__ void __launch_bounds__(kRowThreads) long_row_kernel(const T* logits, LossArgs a) {
  constexpr int N = Vec<T>::N;
  constexpr int kWarps = kRowThreads / 32;
  constexpr int NV = 4;
  __shared__ float2 pairs[kWarps];
  let_next_kernel_start();
  const size_t row = a.row0 + blockIdx.x;
  const T* x = logits + row * (size_t)a.vocab;
  const Split sp = split_row(x, a.vocab);
  const Target tg = target_of(a.targets, row, a.vocab, a.ignore);
  const unsigned self = threadIdx.x;
  const unsigned edge = self < 8 ? (self < sp.head ? self : ~0u)
                        : self < 16 && self - 8 < sp.tail ? sp.head + sp.vecs * N + (self - 8)
                                                          : ~0u;
  const bool has_edge = edge != ~0u;
  const float xe = has_edge ? to_f32(x[edge]) : -INFINITY;
  const float xt = tg.t >= 0 ? to_f32(x[tg.t]) : 0.0f;
  float m = xe, s = has_edge && (long long)edge != tg.t ? exp_below(xe, against(xe)) : 0.0f;
  for (unsigned i0 = 0; i0 < sp.vecs; i0 += NV * kRowThreads) {
    Vec<T> v[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const unsigned i = i0 + k * kRowThreads + self;
      if (i < sp.vecs) v[k] = load_vec(x + sp.head + (size_t)i * N);
    }
    float nm = m;
#pragma unroll
    for (int k = 0; k < NV; k++)
      if (i0 + k * kRowThreads + self < sp.vecs) nm = max_of<T>(v[k], nm);
    const float ms = against(nm);
    s = fmul(s, exp_below(m, ms));
    m = nm;
#pragma unroll
    for (int k = 0; k < NV; k++) {
      const unsigned i = i0 + k * kRowThreads + self;
      if (i < sp.vecs) {
        float f[N];
        unpack<T>(v[k], f);
        const long long j = (long long)sp.head + (long long)i * N;
        if (tg.t >= j && tg.t < j + N) {
#pragma unroll
          for (int e = 0; e < N; e++)
            if (j + e == tg.t) f[e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < N; e++) s = fadd(s, exp_below(f[e], ms));
      }
    }
  }
  const float wm = warp_max(m);
  const float ws = warp_sum(fmul(s, exp_below(m, against(wm))));
  if ((self & 31) == 0) pairs[self >> 5] = make_float2(wm, ws);
  __syncthreads();
  if (self >= 32) return;
  const float2 p = self < kWarps ? pairs[self] : make_float2(-INFINITY, 0.0f);
  const float top = warp_max(p.x);
  float others = warp_sum(fmul(p.y, exp_below(p.x, against(top))));
  if (self == 0) {
    if (top == -INFINITY) others = nan_f();
    const float sum = tg.t >= 0 ? fadd(others, exp_below(xt, top)) : others;
    if (tg.bad) atomicExch(a.bad, 1);
    if (a.row_losses)
      a.row_losses[row] = !tg.counted ? 0.0f : tg.bad ? nan_f() : row_loss(top, sum, others, xt);
    if (a.stats) {
      a.stats[3 * row] = top;
      a.stats[3 * row + 1] = sum;
      a.stats[3 * row + 2] = others;
    }
  }
}

// The gradient from the statistics: `parts` blocks to a row.
template <class T>
__global__ void __launch_bounds__(kThreads)
token_grad_kernel(const T* logits, IndexArray targets, size_t rows, unsigned vocab,
                  long long ignore, const float* stats, const float* upstream, bool per_row,
                  float grad_scale, const unsigned long long* count, T* grad, bool alike,
                  unsigned parts, bool chained, int* bad) {
  constexpr int N = Vec<T>::N;
  constexpr int U = 4;
  const size_t row = blockIdx.x / parts;
  const unsigned part = blockIdx.x % parts;
  const T* x = logits + row * (size_t)vocab;
  T* g = grad + row * (size_t)vocab;
  const Split sp = split_row(x, vocab);
  const Target tg = target_of(targets, row, vocab, ignore);
  const unsigned i0 = part * (U * kThreads) + threadIdx.x;
  Vec<T> v[U];
  if (tg.counted) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (i0 + u * kThreads < sp.vecs) v[u] = load_vec(x + sp.head + (size_t)(i0 + u * kThreads) * N);
  }
  if (chained) wait_for_previous_kernel();
  const float top = stats[3 * row], sum = stats[3 * row + 1], others = stats[3 * row + 2];
  float k = upstream ? upstream[per_row ? row : 0] : grad_scale;
  if (count) k = fdiv(k, (float)*count);
  k = tg.bad ? nan_f() : fdiv(k, sum);
  const float at_target = fmul(-others, k);
  if (tg.bad && part == 0 && threadIdx.x == 0) atomicExch(bad, 1);
#pragma unroll
  for (int u = 0; u < U; u++) {
    const unsigned i = i0 + u * kThreads;
    if (i < sp.vecs) {
      float f[N];
      if (tg.counted) {
        unpack<T>(v[u], f);
        const long long j = (long long)sp.head + (long long)i * N;
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = fmul(exp_below(f[e], top), k);
        if (tg.t >= j && tg.t < j + N) {
#pragma unroll
          for (int e = 0; e < N; e++)
            if (j + e == tg.t) f[e] = at_target;
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; e++) f[e] = 0.0f;
      }
      T* p = g + sp.head + (size_t)i * N;
      if (alike) {
        store_vec(p, pack<T>(f));
      } else {
#pragma unroll
        for (int e = 0; e < N; e++) p[e] = from_f32<T>(f[e]);
      }
    }
  }
  if (part == 0 && threadIdx.x < sp.head + sp.tail) {
    const unsigned j =
        threadIdx.x < sp.head ? threadIdx.x : sp.vecs * N + threadIdx.x;
    g[j] = from_f32<T>(!tg.counted           ? 0.0f
                       : (long long)j == tg.t ? at_target
                                              : fmul(exp_below(to_f32(x[j]), top), k));
  }
}

// One block: how many rows count, at least 1 (a mean over none is 0).
__global__ void __launch_bounds__(1024)
token_count_kernel(IndexArray targets, size_t rows, long long ignore, unsigned long long* count) {
  __shared__ unsigned long long part[32];
  let_next_kernel_start();
  unsigned long long c = 0;
#pragma unroll 8
  for (size_t i = threadIdx.x; i < rows; i += 1024) c += targets[i] != ignore;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x < 32) {
    c = part[threadIdx.x];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
    if (threadIdx.x == 0) *count = c ? c : 1;
  }
}

// One block: the rows' losses summed in f64 in a fixed order, over `count`.
__global__ void __launch_bounds__(1024)
token_loss_sum_kernel(const float* row_losses, size_t rows, const unsigned long long* count,
                      float* loss) {
  __shared__ double part[32];
  wait_for_previous_kernel();
  double a = 0.0;
#pragma unroll 8
  for (size_t i = threadIdx.x; i < rows; i += 1024) a += (double)row_losses[i];
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x < 32) {
    a = part[threadIdx.x];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
    if (threadIdx.x == 0) *loss = (float)(count ? a / (double)*count : a);
  }
}

struct Scratch {
  float* row_losses;
  float* stats;
  unsigned long long* count;
};
size_t up256(size_t b) { return (b + 255) & ~size_t(255); }
Scratch scratch_of(const TokenLoss& a, void* p) {
  char* c = static_cast<char*>(p);
  Scratch s;
  s.count = reinterpret_cast<unsigned long long*>(c);
  c += 256;
  s.row_losses = reinterpret_cast<float*>(c);
  c += up256(a.rows * 4);
  s.stats = reinterpret_cast<float*>(c);
  return s;
}

constexpr size_t kMaxGrid = 0x7fffffff;

// The vectors that a row may have.
size_t vecs_of(const TokenLoss& a) { return (a.vocab * store_bytes(a.type) + 15) / 16; }
bool fits_cluster(const TokenLoss& a) {
  return vecs_of(a) <= (size_t)kMaxCluster * kRowThreads * kMaxVec;
}

template <class T, int NV, bool GRAD>
cudaError_t rows_of(const TokenLoss& t, LossArgs a, unsigned blocks, bool chained,
                    cudaStream_t s) {
  const T* x = static_cast<const T*>(t.logits);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.stream = s;
  cfg.attrs = attr;
  const size_t step = blocks ? kMaxGrid / blocks : kMaxGrid;
  for (size_t r0 = 0; r0 < t.rows; r0 += step) {
    a.row0 = r0;
    a.rows = std::min<size_t>(t.rows - r0, step);
    cfg.numAttrs = 0;
    if (chained) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    cudaError_t e;
    if (blocks == 0) {
      cfg.gridDim = dim3((unsigned)((a.rows + kThreads / 32 - 1) / (kThreads / 32)));
      cfg.blockDim = dim3(kThreads);
      e = cudaLaunchKernelEx(&cfg, warp_row_kernel<T, NV, GRAD>, x, a);
    } else {
      cfg.gridDim = dim3((unsigned)(a.rows * blocks));
      cfg.blockDim = dim3(kRowThreads);
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = blocks;
      attr[cfg.numAttrs].val.clusterDim.y = 1;
      attr[cfg.numAttrs++].val.clusterDim.z = 1;
      e = cudaLaunchKernelEx(&cfg, cluster_row_kernel<T, NV, GRAD>, x, a);
    }
    if (e != cudaSuccess) return e;
    // a later launch's wait covers only its predecessor: from the second on,
    // each starts when the one before has ended
    chained = false;
  }
  return cudaSuccess;
}

template <class T, bool GRAD>
cudaError_t rows_by_size(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  const size_t vecs = vecs_of(t);
  // a warp up to 4 KB, then as few blocks as hold the row in kMaxVec vectors a
  // thread
  unsigned blocks = 0;
  size_t threads = 32;
  if (vecs > 32 * kMaxVec) {
    blocks = 1;
    while (blocks < kMaxCluster && (size_t)blocks * kRowThreads * kMaxVec < vecs) blocks *= 2;
    threads = (size_t)blocks * kRowThreads;
  }
  const size_t nv = (vecs + threads - 1) / threads;
  if (nv <= 1) return rows_of<T, 1, GRAD>(t, a, blocks, chained, s);
  if (nv <= 2) return rows_of<T, 2, GRAD>(t, a, blocks, chained, s);
  if (nv <= 4) return rows_of<T, 4, GRAD>(t, a, blocks, chained, s);
  if (nv <= 6) return rows_of<T, 6, GRAD>(t, a, blocks, chained, s);
  if (nv <= 7) return rows_of<T, 7, GRAD>(t, a, blocks, chained, s);
  return rows_of<T, 8, GRAD>(t, a, blocks, chained, s);
}

template <class T>
cudaError_t long_rows(const TokenLoss& t, LossArgs a, cudaStream_t s) {
  for (size_t r0 = 0; r0 < t.rows; r0 += kMaxGrid) {
    a.row0 = r0;
    const size_t rows = std::min<size_t>(t.rows - r0, kMaxGrid);
    long_row_kernel<T><<<(unsigned)rows, kRowThreads, 0, s>>>(
        static_cast<const T*>(t.logits), a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Statistics and losses of every row, and the gradient unless it is null.
template <class T>
cudaError_t rows_any(const TokenLoss& t, const LossArgs& a, bool chained, cudaStream_t s) {
  if (!fits_cluster(t)) return long_rows<T>(t, a, s);
  return a.grad ? rows_by_size<T, true>(t, a, chained, s)
                : rows_by_size<T, false>(t, a, chained, s);
}

cudaError_t launch_rows(const TokenLoss& t, float* row_losses, float* stats, void* grad,
                        float grad_scale, const unsigned long long* count, bool chained,
                        cudaStream_t s) {
  if (t.rows == 0) return cudaSuccess;
  LossArgs a = {};
  a.targets = IndexArray{t.targets, t.wide};
  a.vocab = (unsigned)t.vocab;
  a.ignore = t.ignore;
  a.row_losses = row_losses;
  a.stats = stats;
  a.grad = grad;
  a.grad_scale = grad_scale;
  a.count = count;
  a.bad = t.bad;
  a.alike = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(t.logits)) & 15) == 0;
  switch (t.type) {
    case kF32: return rows_any<float>(t, a, chained, s);
    case kBF16: return rows_any<bf16>(t, a, chained, s);
    case kF16: return rows_any<f16>(t, a, chained, s);
  }
  return cudaErrorInvalidValue;
}

template <class T>
cudaError_t grad_of(const TokenLoss& a, const float* stats, const float* upstream,
                    float grad_scale, const unsigned long long* count, void* grad, bool chained,
                    cudaStream_t s) {
  const size_t parts = std::max<size_t>(1, (vecs_of(a) + 4 * kThreads - 1) / (4 * kThreads));
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
    const unsigned grid = (unsigned)(rows * parts);
    cudaError_t e;
    if (chained && r0 == 0) {
      e = launch_after(token_grad_kernel<T>, grid, kThreads, 0, s, x, targets, rows,
                       (unsigned)a.vocab, a.ignore, stats, up, per_row, grad_scale, count, g,
                       alike, (unsigned)parts, true, a.bad);
    } else {
      token_grad_kernel<T><<<grid, kThreads, 0, s>>>(
          x, targets, rows, (unsigned)a.vocab, a.ignore, stats + 3 * r0, up, per_row, grad_scale,
          count, g, alike, (unsigned)parts, false, a.bad);
      e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

cudaError_t grad_any(const TokenLoss& a, const float* stats, const float* upstream,
                     float grad_scale, const unsigned long long* count, void* grad, bool chained,
                     cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return grad_of<float>(a, stats, upstream, grad_scale, count, grad, chained, s);
    case kBF16: return grad_of<bf16>(a, stats, upstream, grad_scale, count, grad, chained, s);
    case kF16: return grad_of<f16>(a, stats, upstream, grad_scale, count, grad, chained, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t count_rows(const TokenLoss& a, unsigned long long* count, cudaStream_t s) {
  token_count_kernel<<<1, 1024, 0, s>>>(IndexArray{a.targets, a.wide}, a.rows, a.ignore, count);
  return cudaGetLastError();
}

}  // namespace

size_t token_loss_scratch(const TokenLoss& a) { return 256 + up256(a.rows * 4) + a.rows * 12; }

cudaError_t launch_token_loss(const TokenLoss& a, float* loss, float* stats, void* scratch,
                              cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool none = a.reduction == RTC_REDUCE_NONE, mean = a.reduction == RTC_REDUCE_MEAN;
  cudaError_t e = mean ? count_rows(a, sc.count, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_rows(a, none ? loss : sc.row_losses, stats, nullptr, 1.0f, nullptr, false, s);
  if (e != cudaSuccess || none) return e;
  return launch_after(token_loss_sum_kernel, 1u, 1024u, 0, s, (const float*)sc.row_losses, a.rows,
                      (const unsigned long long*)(mean ? sc.count : nullptr), loss);
}

cudaError_t launch_token_loss_backward(const TokenLoss& a, const float* upstream,
                                       const float* stats, void* grad, void* scratch,
                                       cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool mean = a.reduction == RTC_REDUCE_MEAN;
  const cudaError_t e = mean ? count_rows(a, sc.count, s) : cudaSuccess;
  return e != cudaSuccess ? e
                          : grad_any(a, stats, upstream, 1.0f, mean ? sc.count : nullptr, grad,
                                     mean, s);
}

cudaError_t launch_token_loss_grad(const TokenLoss& a, float grad_scale, float* loss, void* grad,
                                   void* scratch, cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool none = a.reduction == RTC_REDUCE_NONE, mean = a.reduction == RTC_REDUCE_MEAN;
  unsigned long long* count = mean ? sc.count : nullptr;
  const bool one_pass = fits_cluster(a);
  cudaError_t e = mean ? count_rows(a, count, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_rows(a, none ? loss : sc.row_losses, one_pass ? nullptr : sc.stats,
                    one_pass ? grad : nullptr, grad_scale, count, mean && one_pass, s);
  if (e == cudaSuccess && !one_pass)
    e = grad_any(a, sc.stats, nullptr, grad_scale, count, grad, false, s);
  if (e != cudaSuccess || none) return e;
  return launch_after(token_loss_sum_kernel, 1u, 1024u, 0, s, (const float*)sc.row_losses, a.rows,
                      (const unsigned long long*)count, loss);
}

}  // namespace rt
