// token_loss.cu — softmax cross entropy of logits against token ids: the
// kernels around the rows' (token_loss.cuh), and the launchers.
#include "../../include/rusttorch_cuda.h"
#include "rt_chain.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_types.cuh"
#include "token_loss.h"

namespace rt {
namespace {

// One block.
__global__ void __launch_bounds__(1024)
token_count_kernel(IndexArray targets, size_t rows, long long ignore, Count* count) {
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
    if (threadIdx.x == 0) *count = {c ? c : 1, frcp((float)(c ? c : 1))};
  }
}

// One block: the rows' losses summed in f64 in a fixed order, over `count`.
__global__ void __launch_bounds__(1024)
token_loss_sum_kernel(const float* row_losses, size_t rows, const Count* count, float* loss) {
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
    if (threadIdx.x == 0) *loss = (float)(count ? a / (double)count->rows : a);
  }
}

struct Scratch {
  float* row_losses;
  float* stats;
  Count* count;
};
size_t up256(size_t b) { return (b + 255) & ~size_t(255); }
Scratch scratch_of(const TokenLoss& a, void* p) {
  char* c = static_cast<char*>(p);
  Scratch s;
  s.count = reinterpret_cast<Count*>(c);
  c += 256;
  s.row_losses = reinterpret_cast<float*>(c);
  c += up256(a.rows * 4);
  s.stats = reinterpret_cast<float*>(c);
  return s;
}

cudaError_t launch_rows(const TokenLoss& t, float* row_losses, float* stats, void* grad,
                        float grad_scale, const Count* count, bool chained,
                        cudaStream_t s) {
  if (t.rows == 0) return cudaSuccess;
  LossArgs a = {};
  a.targets = IndexArray{t.targets, t.wide};
  a.rows = t.rows;
  a.vocab = (unsigned)t.vocab;
  a.ignore = t.ignore;
  a.row_losses = row_losses;
  a.stats = stats;
  a.grad = grad;
  a.grad_scale = grad_scale;
  a.count = count;
  a.bad = t.bad;
  a.gave_up = t.gave_up;
  a.alike = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(t.logits)) & 15) == 0;
  switch (t.type) {
    case kF32: return token_rows_f32(t, a, chained, s);
    case kBF16: return token_rows_bf16(t, a, chained, s);
    case kF16: return token_rows_f16(t, a, chained, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t grad_any(const TokenLoss& a, const float* stats, const float* upstream,
                     float grad_scale, const Count* count, void* grad, bool chained,
                     cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case kF32: return token_grad_f32(a, stats, upstream, grad_scale, count, grad, chained, s);
    case kBF16: return token_grad_bf16(a, stats, upstream, grad_scale, count, grad, chained, s);
    case kF16: return token_grad_f16(a, stats, upstream, grad_scale, count, grad, chained, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t count_rows(const TokenLoss& a, Count* count, cudaStream_t s) {
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
                      (const Count*)(mean ? sc.count : nullptr), loss);
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
  Count* count = mean ? sc.count : nullptr;
  const bool one_pass = fits_cluster(a);
  cudaError_t e = mean ? count_rows(a, count, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_rows(a, none ? loss : sc.row_losses, one_pass ? nullptr : sc.stats,
                    one_pass ? grad : nullptr, grad_scale, count, mean && one_pass, s);
  if (e == cudaSuccess && !one_pass)
    e = grad_any(a, sc.stats, nullptr, grad_scale, count, grad, false, s);
  if (e != cudaSuccess || none) return e;
  return launch_after(token_loss_sum_kernel, 1u, 1024u, 0, s, (const float*)sc.row_losses, a.rows,
                      (const Count*)count, loss);
}

}  // namespace rt
