// token_loss.h — what the token loss's kernels (token_loss.cuh, one file per
// storage type) and its launchers (token_loss.cu) share.
#pragma once
#include "rt_internal.h"
#include "rt_types.cuh"

namespace rt {

// How many rows count, at least 1 (a mean over none is 0), and its inverse.
struct Count {
  unsigned long long rows;
  float inverse;
};

struct LossArgs {
  IndexArray targets;
  size_t rows;
  unsigned vocab;
  long long ignore;
  float* row_losses;                   // [rows of the call]
  float* stats;                        // null, or [rows, 3]
  void* grad;                          // null, or the gradient
  float grad_scale;
  Count* count;                        // null, or what a mean divides by
  bool count_here;                     // the row kernel counts, and writes it
  int* bad;
  int* gave_up;                        // the flag of a wait that ran out
  bool alike;                          // grad's rows start where logits' do, modulo 16 bytes
};

// Statistics and losses of every row, and the gradient unless it is null and
// the rows fit on chip.
#define RT_TOKEN_LOSS_DECL(NAME)                                                                \
  cudaError_t token_rows_##NAME(const TokenLoss& t, const LossArgs& a, bool chained,            \
                                cudaStream_t s);                                                \
  cudaError_t token_grad_##NAME(const TokenLoss& t, const float* stats, const float* upstream,  \
                                float grad_scale, const Count* count, bool count_here,          \
                                void* grad, bool chained, cudaStream_t s);
RT_TOKEN_LOSS_DECL(f32)
RT_TOKEN_LOSS_DECL(bf16)
RT_TOKEN_LOSS_DECL(f16)
#undef RT_TOKEN_LOSS_DECL

constexpr size_t kMaxGrid = 0x7fffffff;
constexpr int kMaxCluster = 8;        // blocks to a row
// 16-byte vectors of a row that a block holds: two buffers of them in each of
// per_sm blocks fill an SM's shared memory (less 1 KB and the tables of each).
__host__ __device__ constexpr unsigned run_vecs(int per_sm) {
  return per_sm == 16 ? 400 : per_sm == 8 ? 840 : 6912 / per_sm;
}

// The vectors that a row may have.
inline size_t vecs_of(const TokenLoss& a) { return (a.vocab * store_bytes(a.type) + 15) / 16; }
// Whether a row fits on chip, so that one pass gives its gradient too.
inline bool fits_cluster(const TokenLoss& a) {
  return vecs_of(a) <= kMaxCluster * run_vecs(1);
}

// Whether a block walks a row (walk_kernel) where clusters would hold it: for
// statistics alone, with rows enough for all SMs, since nothing then has to stay
// on chip (8192 x 50257 bf16: 147 us for 201, 4096 x 32768 f32: 96 for 117), but
// not for rows that a warp holds (16384 x 1000 f32: 35 us for 23).
constexpr size_t kWalkRows = 296;
inline bool walks_rows(const TokenLoss& a, const void* grad) {
  return !fits_cluster(a) || (!grad && a.rows >= kWalkRows && vecs_of(a) > run_vecs(16));
}

// Threads of the blocks that take such rows (rows_by_size).
inline int row_threads(const TokenLoss& a) {
  const size_t vecs = vecs_of(a);
  return vecs <= run_vecs(16)                 ? 32
         : vecs <= run_vecs(8)                ? 64
         : vecs <= run_vecs(4)                ? 128
         : vecs <= kMaxCluster * run_vecs(2) ? 256 : 512;
}

// How many of `rows` targets are not `ignore`, at least 1, in all threads of a
// block of TH; every thread calls it.
template <int TH>
__device__ __forceinline__ Count count_rows(const IndexArray& targets, size_t rows,
                                            long long ignore) {
  __shared__ unsigned part[TH / 32];
  unsigned c = 0;
#pragma unroll 8
  for (size_t i = threadIdx.x; i < rows; i += TH) c += targets[i] != ignore;
  c = __reduce_add_sync(0xffffffffu, c);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
  __syncthreads();
  unsigned long long n = 0;
#pragma unroll
  for (int k = 0; k < TH / 32; k++) n += part[k];
  n = n ? n : 1;
  return {n, __frcp_rn((float)n)};
}

}  // namespace rt
