// embedding.cu — rows of a table by token id, and the table's gradient.
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_types.cuh"

#include <algorithm>

namespace rt {

size_t store_bytes(StoreType t) { return t == kF32 ? 4 : 2; }

namespace {

template <class T>
__global__ void __launch_bounds__(kThreads)
embedding_kernel(const T* w, IndexArray ids, size_t n, long long vocab, size_t width, float scale,
                 T* out, int* bad) {
  for (size_t i = blockIdx.x; i < n; i += gridDim.x) {
    const long long id = ids[i];
    const bool good = id >= 0 && id < vocab;
    if (!good && threadIdx.x == 0) atomicExch(bad, 1);
    for (size_t c = threadIdx.x; c < width; c += kThreads)
      out[i * width + c] =
          from_f32<T>(good ? fmul(to_f32(w[(size_t)id * width + c]), scale) : u2f(0x7fc00000u));
  }
}

// One block per table row: it looks through all ids for its own.
template <class T, class G>
__global__ void __launch_bounds__(kThreads)
embedding_backward_kernel(const T* g, IndexArray ids, size_t n, long long vocab, size_t width,
                          float scale, long long padding, bool accumulate, G* gw, int* bad) {
  __shared__ int hits[kThreads];
  __shared__ int count;
  const size_t col = (size_t)blockIdx.y * kThreads + threadIdx.x;
  for (long long v = blockIdx.x; v < vocab; v += gridDim.x) {
    float acc = 0.0f;
    bool any = false;
    for (size_t base = 0; base < n; base += kThreads) {
      const size_t i = base + threadIdx.x;
      const long long id = i < n ? ids[i] : -1;
      if (i < n && (id < 0 || id >= vocab)) atomicExch(bad, 1);
      hits[threadIdx.x] = id == v && v != padding;
      const int found = __syncthreads_count(hits[threadIdx.x]);
      if (found) {
        any = true;
        if (threadIdx.x == 0) {
          count = 0;
          for (int k = 0; k < kThreads; k++)
            if (hits[k]) hits[count++] = k;
        }
        __syncthreads();
        if (col < width)
          for (int k = 0; k < found; k++)
            acc = fadd(acc, to_f32(g[(base + hits[k]) * width + col]));
      }
      __syncthreads();
    }
    if (col < width) {
      G* o = gw + (size_t)v * width + col;
      const float r = fmul(acc, scale);
      if (!accumulate) *o = from_f32<G>(r);
      else if (any) *o = from_f32<G>(fadd(to_f32(*o), r));
    }
  }
}

}  // namespace

cudaError_t launch_embedding(StoreType t, const void* weight, const void* ids, bool wide,
                             size_t n, size_t vocab, size_t width, float scale, void* out,
                             int* bad, cudaStream_t s) {
  if (n == 0 || width == 0) return cudaSuccess;
  const unsigned grid = (unsigned)std::min<size_t>(n, 1u << 20);
  const IndexArray ia{ids, wide};
  switch (t) {
    case kF32:
      embedding_kernel<float><<<grid, kThreads, 0, s>>>((const float*)weight, ia, n, vocab, width,
                                                        scale, (float*)out, bad);
      break;
    case kBF16:
      embedding_kernel<bf16><<<grid, kThreads, 0, s>>>((const bf16*)weight, ia, n, vocab, width,
                                                       scale, (bf16*)out, bad);
      break;
    case kF16:
      embedding_kernel<f16><<<grid, kThreads, 0, s>>>((const f16*)weight, ia, n, vocab, width,
                                                      scale, (f16*)out, bad);
      break;
  }
  return cudaGetLastError();
}

size_t embedding_backward_scratch(size_t, size_t, size_t) { return 256; }

namespace {
template <class T, class G>
cudaError_t backward_of(const void* g, IndexArray ids, size_t n, size_t vocab, size_t width,
                        float scale, long long padding, bool accumulate, void* gw, int* bad,
                        cudaStream_t s) {
  const dim3 grid((unsigned)std::min<size_t>(vocab, 1u << 20),
                  (unsigned)((width + kThreads - 1) / kThreads));
  embedding_backward_kernel<T, G><<<grid, kThreads, 0, s>>>(
      (const T*)g, ids, n, vocab, width, scale, padding, accumulate, (G*)gw, bad);
  return cudaGetLastError();
}
}  // namespace

cudaError_t launch_embedding_backward(StoreType t, const void* grad_output, const void* ids,
                                      bool wide, size_t n, size_t vocab, size_t width,
                                      float scale, long long padding, bool accumulate,
                                      void* grad_weight, bool narrow, void*, int* bad,
                                      cudaStream_t s) {
  if (vocab == 0 || width == 0) return cudaSuccess;
  const IndexArray ia{ids, wide};
  if (t == kF32)
    return backward_of<float, float>(grad_output, ia, n, vocab, width, scale, padding, accumulate,
                                     grad_weight, bad, s);
  if (t == kBF16)
    return narrow ? backward_of<bf16, bf16>(grad_output, ia, n, vocab, width, scale, padding,
                                            accumulate, grad_weight, bad, s)
                  : backward_of<bf16, float>(grad_output, ia, n, vocab, width, scale, padding,
                                             accumulate, grad_weight, bad, s);
  return narrow ? backward_of<f16, f16>(grad_output, ia, n, vocab, width, scale, padding,
                                        accumulate, grad_weight, bad, s)
                : backward_of<f16, float>(grad_output, ia, n, vocab, width, scale, padding,
                                          accumulate, grad_weight, bad, s);
}

}  // namespace rt
