// token_loss.cu — softmax cross entropy of logits against token ids, and its
// gradient.
//
// With M = max_j x_j, o = sum_{j != t} e^(x_j - M) and s = o + e^(x_t - M):
//   loss = log s - (x_t - M), which is log1p(o) where x_t = M,
//   gradient = k e^(x_j - M)/s for j != t and -k o/s for j = t,
// k the upstream gradient (over the count of rows for a mean).  The target's
// term stays out of o, so a token that the model is sure of keeps the digits
// of its small loss and gradient, which 1 - p_t would lose.
#include "../../include/rusttorch_cuda.h"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_types.cuh"

#include <algorithm>

namespace rt {
namespace {

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

// The maximum of the block's values, NaN if any is NaN.
__device__ __forceinline__ float nan_max(float a, float b) {
  return a != a ? a : (b != b ? b : fmaxf(a, b));
}

template <class F>
__device__ __forceinline__ float block_reduce(float v, float* smem, F f, float none) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < blockDim.x / 32 ? smem[threadIdx.x] : none;
  if (threadIdx.x < 32) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
    if (threadIdx.x == 0) smem[0] = v;
  }
  __syncthreads();
  return smem[0];
}

// One block per row: its maximum, then its sums.
template <class T>
__global__ void __launch_bounds__(kThreads)
token_stats_kernel(const T* x, IndexArray targets, size_t rows, long long vocab, long long ignore,
                   float* row_losses, float* stats, int* bad) {
  __shared__ float smem[kThreads / 32];
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * (size_t)vocab;
    const Target tg = target_of(targets, row, vocab, ignore);
    float top = -INFINITY;
    for (long long j = threadIdx.x; j < vocab; j += kThreads) top = nan_max(top, to_f32(xr[j]));
    top = block_reduce(top, smem, nan_max, -INFINITY);
    float others = 0.0f;
    for (long long j = threadIdx.x; j < vocab; j += kThreads)
      if (j != tg.t) others = fadd(others, expf(fsub(to_f32(xr[j]), top)));
    others = block_reduce(others, smem, fadd, 0.0f);
    if (threadIdx.x == 0) {
      const float xt = tg.t >= 0 ? to_f32(xr[tg.t]) : 0.0f;
      const float sum = tg.t >= 0 ? fadd(others, expf(fsub(xt, top))) : others;
      if (tg.bad) atomicExch(bad, 1);
      row_losses[row] = !tg.counted ? 0.0f : tg.bad ? nan_f() : row_loss(top, sum, others, xt);
      if (stats) {
        stats[3 * row] = top;
        stats[3 * row + 1] = sum;
        stats[3 * row + 2] = others;
      }
    }
  }
}

// One block: how many rows count.
__global__ void __launch_bounds__(1024)
token_count_kernel(IndexArray targets, size_t rows, long long ignore, unsigned long long* count) {
  __shared__ unsigned long long part[32];
  unsigned long long c = 0;
  for (size_t i = threadIdx.x; i < rows; i += 1024) c += targets[i] != ignore;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) c += __shfl_xor_sync(0xffffffffu, c, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    c = 0;
    for (int k = 0; k < 32; k++) c += part[k];
    *count = c;
  }
}

// One block: the rows' losses summed in f64 in a fixed order, over `count`.
__global__ void __launch_bounds__(1024)
token_loss_sum_kernel(const float* row_losses, size_t rows, const unsigned long long* count,
                      float* loss) {
  __shared__ double part[1024];
  double a = 0.0;
  for (size_t i = threadIdx.x; i < rows; i += 1024) a += (double)row_losses[i];
  part[threadIdx.x] = a;
  __syncthreads();
  for (int d = 512; d > 0; d >>= 1) {
    if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const unsigned long long c = count ? *count : 1;
    *loss = (float)(part[0] / (double)(c ? c : 1));
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads)
token_grad_kernel(const T* x, IndexArray targets, size_t rows, long long vocab, long long ignore,
                  const float* stats, const float* upstream, bool per_row, float grad_scale,
                  const unsigned long long* count, T* grad, int* bad) {
  for (size_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const Target tg = target_of(targets, row, vocab, ignore);
    if (tg.bad && threadIdx.x == 0) atomicExch(bad, 1);
    const float top = stats[3 * row], sum = stats[3 * row + 1], others = stats[3 * row + 2];
    float k = upstream ? upstream[per_row ? row : 0] : grad_scale;
    if (count) k = fdiv(k, (float)*count);
    if (tg.bad) k = nan_f();
    k = fdiv(k, sum);
    for (long long j = (long long)blockIdx.x * kThreads + threadIdx.x; j < vocab;
         j += (long long)gridDim.x * kThreads) {
      const size_t i = row * (size_t)vocab + j;
      const float e = j == tg.t ? -others : expf(fsub(to_f32(x[i]), top));
      grad[i] = from_f32<T>(tg.counted ? fmul(e, k) : 0.0f);
    }
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

template <class T>
cudaError_t stats_of(const TokenLoss& a, float* row_losses, float* stats, cudaStream_t s) {
  const unsigned grid = (unsigned)std::min<size_t>(a.rows, 1u << 20);
  token_stats_kernel<T><<<grid, kThreads, 0, s>>>((const T*)a.logits, IndexArray{a.targets, a.wide},
                                                  a.rows, (long long)a.vocab, a.ignore, row_losses,
                                                  stats, a.bad);
  return cudaGetLastError();
}

template <class T>
cudaError_t grad_of(const TokenLoss& a, const float* stats, const float* upstream,
                    float grad_scale, const unsigned long long* count, void* grad,
                    cudaStream_t s) {
  const dim3 grid((unsigned)std::min<size_t>((a.vocab + kThreads - 1) / kThreads, 64),
                  (unsigned)std::min<size_t>(a.rows, 65535));
  token_grad_kernel<T><<<grid, kThreads, 0, s>>>(
      (const T*)a.logits, IndexArray{a.targets, a.wide}, a.rows, (long long)a.vocab, a.ignore,
      stats, upstream, a.reduction == RTC_REDUCE_NONE, grad_scale, count, (T*)grad, a.bad);
  return cudaGetLastError();
}

cudaError_t stats_any(const TokenLoss& a, float* row_losses, float* stats, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return stats_of<float>(a, row_losses, stats, s);
    case kBF16: return stats_of<bf16>(a, row_losses, stats, s);
    case kF16: return stats_of<f16>(a, row_losses, stats, s);
  }
  return cudaErrorInvalidValue;
}
cudaError_t grad_any(const TokenLoss& a, const float* stats, const float* upstream,
                     float grad_scale, const unsigned long long* count, void* grad,
                     cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return grad_of<float>(a, stats, upstream, grad_scale, count, grad, s);
    case kBF16: return grad_of<bf16>(a, stats, upstream, grad_scale, count, grad, s);
    case kF16: return grad_of<f16>(a, stats, upstream, grad_scale, count, grad, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t count_rows(const TokenLoss& a, unsigned long long* count, cudaStream_t s) {
  token_count_kernel<<<1, 1024, 0, s>>>(IndexArray{a.targets, a.wide}, a.rows, a.ignore, count);
  return cudaGetLastError();
}

cudaError_t sum_rows(const TokenLoss& a, const Scratch& sc, float* loss, cudaStream_t s) {
  token_loss_sum_kernel<<<1, 1024, 0, s>>>(
      sc.row_losses, a.rows, a.reduction == RTC_REDUCE_MEAN ? sc.count : nullptr, loss);
  return cudaGetLastError();
}

}  // namespace

size_t token_loss_scratch(const TokenLoss& a) { return 256 + up256(a.rows * 4) + a.rows * 12; }

cudaError_t launch_token_loss(const TokenLoss& a, float* loss, float* stats, void* scratch,
                              cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool none = a.reduction == RTC_REDUCE_NONE;
  cudaError_t e = stats_any(a, none ? loss : sc.row_losses, stats, s);
  if (e != cudaSuccess || none) return e;
  if (a.reduction == RTC_REDUCE_MEAN) e = count_rows(a, sc.count, s);
  return e != cudaSuccess ? e : sum_rows(a, sc, loss, s);
}

cudaError_t launch_token_loss_backward(const TokenLoss& a, const float* upstream,
                                       const float* stats, void* grad, void* scratch,
                                       cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool mean = a.reduction == RTC_REDUCE_MEAN;
  const cudaError_t e = mean ? count_rows(a, sc.count, s) : cudaSuccess;
  return e != cudaSuccess
             ? e
             : grad_any(a, stats, upstream, 1.0f, mean ? sc.count : nullptr, grad, s);
}

cudaError_t launch_token_loss_grad(const TokenLoss& a, float grad_scale, float* loss, void* grad,
                                   void* scratch, cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const cudaError_t e = launch_token_loss(a, loss, sc.stats, scratch, s);
  return e != cudaSuccess
             ? e
             : grad_any(a, sc.stats, nullptr, grad_scale,
                        a.reduction == RTC_REDUCE_MEAN ? sc.count : nullptr, grad, s);
}

}  // namespace rt
