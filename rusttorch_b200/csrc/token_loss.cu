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
  let_next_kernel_start();
  const Count c = count_rows<1024>(targets, rows, ignore);
  if (threadIdx.x == 0) *count = c;
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
                        float grad_scale, Count* count, bool count_here, bool chained,
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
  a.count_here = count_here;
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
                     float grad_scale, const Count* count, bool count_here, void* grad,
                     bool chained, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  switch (a.type) {
    case kF32:
      return token_grad_f32(a, stats, upstream, grad_scale, count, count_here, grad, chained, s);
    case kBF16:
      return token_grad_bf16(a, stats, upstream, grad_scale, count, count_here, grad, chained, s);
    case kF16:
      return token_grad_f16(a, stats, upstream, grad_scale, count, count_here, grad, chained, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t launch_count(const TokenLoss& a, Count* count, cudaStream_t s) {
  token_count_kernel<<<1, 1024, 0, s>>>(IndexArray{a.targets, a.wide}, a.rows, a.ignore, count);
  return cudaGetLastError();
}

}  // namespace

size_t token_loss_scratch(const TokenLoss& a) { return 256 + up256(a.rows * 4) + a.rows * 12; }

namespace {

cudaError_t launch_sum(const TokenLoss& a, const Scratch& sc, const Count* count, float* loss,
                       cudaStream_t s) {
  return launch_after(token_loss_sum_kernel, 1u, 1024u, 0, s, (const float*)sc.row_losses, a.rows,
                      count, loss);
}

// Few rows are counted by the blocks that work on them, 32 to a thread at
// most: a kernel less, 2 us of the 12 that 32 rows of 1000 took.  For more rows
// a kernel of one block counts while the first rows arrive.
bool counts_itself(const TokenLoss& a, const void* grad) {
  return !walks_rows(a, grad) && a.rows <= (size_t)32 * row_threads(a);
}

}  // namespace

cudaError_t launch_token_loss(const TokenLoss& a, float* loss, float* stats, void* scratch,
                              cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool none = a.reduction == RTC_REDUCE_NONE;
  Count* count = a.reduction == RTC_REDUCE_MEAN && a.rows ? sc.count : nullptr;
  const bool here = count && counts_itself(a, nullptr);
  cudaError_t e = count && !here ? launch_count(a, count, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_rows(a, none ? loss : sc.row_losses, stats, nullptr, 1.0f, count, here,
                    count && !here, s);
  return e != cudaSuccess || none ? e : launch_sum(a, sc, count, loss, s);
}

cudaError_t launch_token_loss_backward(const TokenLoss& a, const float* upstream,
                                       const float* stats, void* grad, void* scratch,
                                       cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  Count* count = a.reduction == RTC_REDUCE_MEAN && a.rows ? sc.count : nullptr;
  const bool here = count && a.rows <= (size_t)kThreads;   // a target a thread
  const bool chained = count && !here;
  const cudaError_t e = chained ? launch_count(a, count, s) : cudaSuccess;
  return e != cudaSuccess ? e : grad_any(a, stats, upstream, 1.0f, count, here, grad, chained, s);
}

cudaError_t launch_token_loss_grad(const TokenLoss& a, float grad_scale, float* loss, void* grad,
                                   void* scratch, cudaStream_t s) {
  const Scratch sc = scratch_of(a, scratch);
  const bool none = a.reduction == RTC_REDUCE_NONE;
  Count* count = a.reduction == RTC_REDUCE_MEAN && a.rows ? sc.count : nullptr;
  const bool one_pass = fits_cluster(a);
  const bool here = count && counts_itself(a, grad);
  const bool ahead = count && !here;
  cudaError_t e = ahead ? launch_count(a, count, s) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_rows(a, none ? loss : sc.row_losses, one_pass ? nullptr : sc.stats,
                    one_pass ? grad : nullptr, grad_scale, count, here, ahead, s);
  if (e == cudaSuccess && !one_pass)
    e = grad_any(a, sc.stats, nullptr, grad_scale, count, false, grad, false, s);
  return e != cudaSuccess || none ? e : launch_sum(a, sc, count, loss, s);
}

}  // namespace rt
