// embedding.cu — rows of a table by token id, and the table's gradient.
//
// Forward: out[i, :] = T(scale * weight[ids[i], :]), one f32 product and one
// rounding per element, 16 bytes of a row a thread.  HBM bounds it (32768 x 4096
// bf16 of 131072 rows: 68 us, 5.4 TB/s).
//
// Gradient: grad_weight[v, :] (+)= scale * sum over {i : ids[i] = v} of
// grad_output[i, :].  The sums of a row are wherever its tokens are, so:
//  1. sort_ids_kernel sorts the positions by id (stable radix sort) in one
//     cluster of thread blocks; few_ids_kernel few of them by counting,
//     sort_tiles_kernel and place_kernel some by counting and searching;
//  2. segment_kernel cuts the sorted list into pieces of equal length, so
//     that a frequent id costs no block more than a rare one; a group sums its
//     piece's rows in order, writes each id's sum that begins and ends in the
//     piece, and leaves partial sums of those that cross its ends; in the same
//     launch other blocks write the zeros of the ids that do not occur;
//  3. join_kernel adds up the partial sums.
// No floating-point atomics: the order of every sum follows from ids alone.
#include "rt_chain.cuh"
#include "rt_internal.h"
#include "rt_libm.cuh"
#include "rt_tma.cuh"
#include "rt_types.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace rt {

size_t store_bytes(StoreType t) { return t == kF32 ? 4 : 2; }

namespace {

namespace cg = cooperative_groups;

// ---- rows, 16 bytes to a thread ---------------------------------------------
// A group of G threads covers G * 16 bytes of a row: each thread N / VW chunks
// of VW elements, G chunks apart.  VW is the widest access that every row's
// start allows (16 bytes down to one element).
template <class T, int VW>
struct alignas(VW * sizeof(T)) Chunk {
  T x[VW];
};

template <class T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  T x[N];
};

template <int VW, class T>
__device__ __forceinline__ void load_row(const T* row, size_t first, unsigned G, size_t width,
                                         Row<T>& r) {
  constexpr int N = Row<T>::N;
#pragma unroll
  for (int k = 0; k < N / VW; k++) {
    const size_t c = first + (size_t)k * G * VW;
    if (c < width) {
      const T* p = row + c;
      if constexpr (VW * sizeof(T) == 16) {
        const uint4* q = reinterpret_cast<const uint4*>(p);
        *reinterpret_cast<uint4*>(&r.x[k * VW]) = __ldcs(q);
      } else {
        const auto v = *reinterpret_cast<const Chunk<T, VW>*>(p);
#pragma unroll
        for (int e = 0; e < VW; e++) r.x[k * VW + e] = v.x[e];
      }
    }
  }
}

// Stores values laid out as load_row<VW> gave them.
template <int VW, class G_, int N>
__device__ __forceinline__ void store_row(G_* row, size_t first, unsigned G, size_t width,
                                          const float (&v)[N]) {
  // as many elements of G_ as fit 16 bytes at a time
  constexpr int SW = VW * sizeof(G_) > 16 ? 16 / sizeof(G_) : VW;
#pragma unroll
  for (int k = 0; k < N / VW; k++) {
    const size_t c = first + (size_t)k * G * VW;
    if (c < width) {
#pragma unroll
      for (int h = 0; h < VW / SW; h++) {
        Chunk<G_, SW> o;
#pragma unroll
        for (int e = 0; e < SW; e++) o.x[e] = from_f32<G_>(v[k * VW + h * SW + e]);
        if constexpr (SW * sizeof(G_) == 16)
          __stcs(reinterpret_cast<uint4*>(row + c + h * SW), *reinterpret_cast<const uint4*>(&o));
        else
          *reinterpret_cast<Chunk<G_, SW>*>(row + c + h * SW) = o;
      }
    }
  }
}

// v[e] = old + v[e].
template <int VW, class G_, int N>
__device__ __forceinline__ void add_row(const G_* row, size_t first, unsigned G, size_t width,
                                        float (&v)[N]) {
  constexpr int SW = VW * sizeof(G_) > 16 ? 16 / sizeof(G_) : VW;
#pragma unroll
  for (int k = 0; k < N / VW; k++) {
    const size_t c = first + (size_t)k * G * VW;
    if (c < width) {
#pragma unroll
      for (int h = 0; h < VW / SW; h++) {
        const auto o = *reinterpret_cast<const Chunk<G_, SW>*>(row + c + h * SW);
#pragma unroll
        for (int e = 0; e < SW; e++) {
          float& x = v[k * VW + h * SW + e];
          x = fadd(to_f32(o.x[e]), x);
        }
      }
    }
  }
}

// ---- forward -------------------------------------------------------------------

// Rows that all start on 16 bytes: a thread takes the same 16 bytes of R rows.
template <class T, int R>
__global__ void __launch_bounds__(kThreads)
embedding_kernel(const T* w, IndexArray ids, size_t n, long long vocab, size_t width, float scale,
                 T* out, int* bad, unsigned vecs) {
  constexpr int N = Row<T>::N;
  const size_t unit = (size_t)blockIdx.x * kThreads + threadIdx.x;
  const size_t i0 = unit / vecs * R;
  const size_t first = unit % vecs * N;
  Row<T> x[R];
  bool good[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    good[r] = false;
    if (i0 + r < n) {
      const long long id = ids[i0 + r];
      good[r] = id >= 0 && id < vocab;
      if (good[r])
        *reinterpret_cast<uint4*>(x[r].x) =
            __ldg(reinterpret_cast<const uint4*>(w + (size_t)id * width + first));
      else if (first == 0) atomicExch(bad, 1);
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (i0 + r < n) {
      Row<T> o;
#pragma unroll
      for (int e = 0; e < N; e++)
        o.x[e] = from_f32<T>(good[r] ? fmul(to_f32(x[r].x[e]), scale) : u2f(0x7fc00000u));
      *reinterpret_cast<uint4*>(out + (i0 + r) * width + first) =
          *reinterpret_cast<const uint4*>(o.x);
    }
  }
}

// Rows that do not all start on 16 bytes: a thread takes 16 aligned bytes of the
// output and reads them as two aligned 16-byte accesses, of which it shifts
// together what it needs; elements beyond a row's ends are not stored.  Nothing
// outside the table is read.  (32768 rows of 1023 bf16, 50257 in the table:
// 31 us, and 53 us with an access for each element.)
template <class T>
__device__ __forceinline__ uint4 load_anywhere(const char* p) {
  const unsigned off = reinterpret_cast<uintptr_t>(p) & 15;
  const uint4* q = reinterpret_cast<const uint4*>(p - off);
  uint4 a = __ldg(q);
  if (off == 0) return a;
  uint4 b = __ldg(q + 1);
  if (off & 8) {
    a = make_uint4(a.z, a.w, b.x, b.y);
    b.x = b.z;
    b.y = b.w;
  }
  if (off & 4) {
    a = make_uint4(a.y, a.z, a.w, b.x);
    b.x = b.y;
  }
  if (sizeof(T) == 2 && (off & 2))
    a = make_uint4(__funnelshift_r(a.x, a.y, 16), __funnelshift_r(a.y, a.z, 16),
                   __funnelshift_r(a.z, a.w, 16), __funnelshift_r(a.w, b.x, 16));
  return a;
}

template <class T, int R>
__global__ void __launch_bounds__(kThreads)
embedding_anywhere_kernel(const T* w, IndexArray ids, size_t n, long long vocab, size_t width,
                          float scale, T* out, int* bad, unsigned vecs) {
  constexpr int N = Row<T>::N;
  const size_t unit = (size_t)blockIdx.x * kThreads + threadIdx.x;
  const size_t i0 = unit / vecs * R;
  const unsigned vec = (unsigned)(unit % vecs);
  const char* const begin = reinterpret_cast<const char*>(w);
  const char* const end = reinterpret_cast<const char*>(w + (size_t)vocab * width);
  Row<T> x[R];
  long long e[R];        // the row's element that the 16 bytes begin with
  bool good[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    good[r] = false;
    e[r] = 0;
    if (i0 + r >= n) continue;
    const long long id = ids[i0 + r];
    const uintptr_t to = reinterpret_cast<uintptr_t>(out + (i0 + r) * width);
    e[r] = (long long)vec * N - (long long)((to & 15) / sizeof(T));
    good[r] = id >= 0 && id < vocab;
    if (good[r]) {
      const long long at = id * (long long)width + e[r];   // in the table
      const char* p = begin + at * (long long)sizeof(T);
      const unsigned off = reinterpret_cast<uintptr_t>(p) & 15;
      if (p - off >= begin && p + (off ? 32 - off : 16) <= end) {
        *reinterpret_cast<uint4*>(x[r].x) = load_anywhere<T>(p);
      } else {
#pragma unroll
        for (int k = 0; k < N; k++)
          if (e[r] + k >= 0 && e[r] + k < (long long)width) x[r].x[k] = w[at + k];
      }
    } else if (vec == 0) {
      atomicExch(bad, 1);
    }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    if (i0 + r >= n) continue;
    T* to = out + (i0 + r) * width + e[r];
    Row<T> o;
#pragma unroll
    for (int k = 0; k < N; k++)
      o.x[k] = from_f32<T>(good[r] ? fmul(to_f32(x[r].x[k]), scale) : u2f(0x7fc00000u));
    if (e[r] >= 0 && e[r] + N <= (long long)width) {
      *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(o.x);
    } else {
#pragma unroll
      for (int k = 0; k < N; k++)
        if (e[r] + k >= 0 && e[r] + k < (long long)width) to[k] = o.x[k];
    }
  }
}

// Threads that share a row: as many as it has 16-byte parts, at most a block.
unsigned group_of(size_t width, int n_per_thread) {
  unsigned g = 8;
  while (g < (unsigned)kThreads && (size_t)g * n_per_thread < width) g *= 2;
  return g;
}

// The widest chunk (in elements, at most 16 bytes) that every row start of
// these tensors allows.
template <class T>
int chunk_of(size_t width, const void* a, size_t a_size, const void* b, size_t b_size) {
  int vw = 16 / (int)sizeof(T);
  while (vw > 1 && (width % vw ||
                    reinterpret_cast<uintptr_t>(a) % std::min<size_t>(16, vw * a_size) ||
                    reinterpret_cast<uintptr_t>(b) % std::min<size_t>(16, vw * b_size)))
    vw /= 2;
  return vw;
}

template <class T>
cudaError_t embedding_any(const void* weight, IndexArray ids, size_t n, size_t vocab, size_t width,
                          float scale, void* out, int* bad, cudaStream_t s) {
  constexpr int N = Row<T>::N;
  const T* w = static_cast<const T*>(weight);
  T* o = static_cast<T*>(out);
  const bool aligned = chunk_of<T>(width, w, sizeof(T), o, sizeof(T)) == N;
  // the 16 bytes that a row may touch: one more where it starts inside some
  const size_t vecs = aligned ? width / N : (width + 2 * N - 2) / N;
  // Four rows a thread keep 64 bytes of each in flight (two where each takes two
  // accesses and more registers: 1001 f32 43 us, 58 with four, 52 with one); with
  // few rows one each spreads them over more SMs.
  int device = 0;
  cudaGetDevice(&device);
  const bool many = n * vecs >= (size_t)8 * sm_count(device) * kThreads;
  const size_t rows = !many ? 1 : aligned ? 4 : 2;
  const size_t blocks = ((n + rows - 1) / rows * vecs + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffull || vecs > 0xffffffffull) return cudaErrorInvalidValue;
  const auto kernel = aligned ? (many ? embedding_kernel<T, 4> : embedding_kernel<T, 1>)
                              : (many ? embedding_anywhere_kernel<T, 2>
                                      : embedding_anywhere_kernel<T, 1>);
  kernel<<<(unsigned)blocks, kThreads, 0, s>>>(w, ids, n, (long long)vocab, width, scale, o, bad,
                                               (unsigned)vecs);
  return cudaGetLastError();
}

// ---- sorting ---------------------------------------------------------------------

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxCluster = 8;
constexpr int kSortMaxBits = 9;

// Bytes of the gradient that other blocks zero while one cluster sorts.
struct Shadow {
  char* begin;
  size_t bytes;          // a multiple of 2, as begin is
};

struct Sorted {
  uint2* pair[2];       // [n] each: key, and where in ids it was; sorted in pair[passes & 1]
  unsigned* count;      // [2]: of the sums that cross pieces, zeroed here
};

__device__ __forceinline__ unsigned key_of(const IndexArray& ids, size_t i, long long vocab,
                                           long long padding, int* bad) {
  const long long id = ids[i];
  if (id < 0 || id >= vocab) {
    atomicExch(bad, 1);
    return (unsigned)vocab;
  }
  return id == padding ? (unsigned)vocab : (unsigned)id;
}

constexpr unsigned kShadowBytes = 16384;   // zeros that they copy at a time

// `block` of `blocks`, a warp's first lane at a time: the 16-byte-aligned inside
// by bulk copies of shared zeros, the ends two bytes at a time.
__device__ __forceinline__ void write_shadow(const Shadow& z, uint4* zeros, unsigned block,
                                             unsigned blocks) {
  for (unsigned i = threadIdx.x; i < kShadowBytes / 16; i += kSortThreads)
    zeros[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  char* end = z.begin + z.bytes;
  char* a0 = z.begin + (-reinterpret_cast<intptr_t>(z.begin) & 15);
  char* a1 = end - (reinterpret_cast<intptr_t>(end) & 15);
  if (a0 > a1) a0 = a1 = end;
  if (block == 0 && threadIdx.x < 16) {
    uint16_t* h = reinterpret_cast<uint16_t*>(threadIdx.x < 8 ? z.begin : a1) + threadIdx.x % 8;
    if (reinterpret_cast<char*>(h) < (threadIdx.x < 8 ? a0 : end)) *h = 0;
  }
  if ((threadIdx.x & 31) == 0) {
    const size_t step = (size_t)blocks * kSortWarps * kShadowBytes;
    for (char* q = a0 + ((size_t)block * kSortWarps + (threadIdx.x >> 5)) * kShadowBytes; q < a1;
         q += step)
      bulk_store(q, zeros, (unsigned)min((ptrdiff_t)kShadowBytes, (ptrdiff_t)(a1 - q)));
    bulk_store_done();
  }
}

// Stable least-significant-digit radix sort of n keys below 2^(bits * passes)
// by one cluster.  Every warp owns a contiguous range of the list.  A pass
// ranks each key among its warp's keys of the same digit (ballots over the
// digit's bits give a lane its equals), turns the warps' counts into where
// each warp's first key of each digit goes (over warps, then the cluster's
// blocks through distributed shared memory, then digits), and moves the keys.
// Latency bounds it, not bytes: with HELD a warp's 32 * K keys at most stay in
// registers between ranking and moving, all of them loaded at once; longer
// ranges are read twice.  A scattered store takes the SM a cycle for each
// lane, so key and position travel as one, over all the blocks of a cluster.
// Ids that have no row (outside the vocabulary, or padding) get key = vocab,
// which sorts last.
// The grid's further clusters write zeros (Shadow) meanwhile.  (32768 ids below
// 131072, two passes: 21 us; 16384 below 50257: 14 us.)
template <int K, bool HELD>
__global__ void __launch_bounds__(kSortThreads)
sort_ids_kernel(IndexArray ids, unsigned n, long long vocab, long long padding, int bits,
                int passes, Sorted out, Shadow shadow, int* bad) {
  extern __shared__ __align__(16) unsigned hist[];       // [kSortWarps][bins]
  __shared__ unsigned block_total[1 << kSortMaxBits];    // read by the cluster
  __shared__ unsigned base[1 << kSortMaxBits];           // where the block's digits go
  __shared__ unsigned warp_sum[kSortWarps];
  let_next_kernel_start();
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned rank = cluster.block_rank(), blocks = cluster.num_blocks();
  if (blockIdx.x >= blocks) {
    write_shadow(shadow, reinterpret_cast<uint4*>(hist), blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const unsigned bins = 1u << bits;
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned warps = blocks * kSortWarps;
  const unsigned per_warp = ((n + warps - 1) / warps + 31) & ~31u;
  const unsigned long long begin64 = (unsigned long long)(rank * kSortWarps + warp) * per_warp;
  const unsigned begin = (unsigned)min(begin64, (unsigned long long)n);
  const unsigned end = (unsigned)min(begin64 + per_warp, (unsigned long long)n);
  unsigned* mine = hist + warp * bins;
  if (rank == 0 && threadIdx.x < 2) out.count[threadIdx.x] = 0;

  auto clear_mine = [&] {
    __syncwarp();
    for (unsigned b = lane; b < bins; b += 32) mine[b] = 0;
    __syncwarp();
  };
  clear_mine();
  unsigned key[K], pos[K], to[K];
  for (int pass = 0; pass < passes; pass++) {
    const int shift = pass * bits;
    const uint2* in = out.pair[pass & 1];
    uint2* moved = out.pair[(pass + 1) & 1];
    auto load = [&](unsigned from) {
#pragma unroll
      for (int j = 0; j < K; j++) {
        const unsigned i = from + j * 32 + lane;
        key[j] = 0;
        if (i < end) {
          const uint2 x =
              pass ? __ldcg(in + i) : make_uint2(key_of(ids, i, vocab, padding, bad), i);
          key[j] = x.x;
          pos[j] = x.y;
        }
      }
    };
    // to[j]: how many of the warp's keys before this one have its digit, on
    // top of what `mine` starts with
    auto rank_keys = [&](unsigned from) {
      unsigned same[K];                 // the lanes with this one's digit
#pragma unroll
      for (int j = 0; j < K; j++) {
        const unsigned digit = (key[j] >> shift) & (bins - 1);
        same[j] = __ballot_sync(0xffffffffu, from + j * 32 + lane < end);
#pragma unroll
        for (int d = 0; d < kSortMaxBits; d++) {   // bits above `bits` are 0 in every lane
          const unsigned m = __ballot_sync(0xffffffffu, (digit >> d) & 1u);
          same[j] &= (digit >> d) & 1u ? m : ~m;
        }
      }
#pragma unroll
      for (int j = 0; j < K; j++) {
        if (from + j * 32 >= end) break;        // the warp's lanes agree
        const bool live = from + j * 32 + lane < end;
        const unsigned digit = (key[j] >> shift) & (bins - 1);
        const unsigned before = __popc(same[j] & ((1u << lane) - 1));
        if (live) to[j] = mine[digit] + before;
        __syncwarp();
        if (live && before == 0) mine[digit] += __popc(same[j]);
        __syncwarp();
      }
    };
    for (unsigned i0 = begin; i0 < end; i0 += 32 * K) {
      load(i0);
      rank_keys(i0);
    }
    __syncthreads();
    // over the block's warps: exclusive prefix of each digit
    const unsigned b = threadIdx.x;
    if (b < bins) {
      unsigned sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; w++) {
        const unsigned c = hist[w * bins + b];
        hist[w * bins + b] = sum;
        sum += c;
      }
      block_total[b] = sum;
    }
    cluster.sync();
    // over the cluster's blocks, then over digits
    unsigned before = 0, all = 0;
    if (b < bins) {
#pragma unroll
      for (unsigned r = 0; r < kSortMaxCluster; r++) {
        if (r < blocks) {
          const unsigned c = *cluster.map_shared_rank(&block_total[b], r);
          if (r < rank) before += c;
          all += c;
        }
      }
    }
    unsigned scan = all;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned o = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= (unsigned)d) scan += o;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    if (b < bins) {
      unsigned at = scan - all + before;
#pragma unroll
      for (unsigned w = 0; w < (1u << kSortMaxBits) / 32; w++)
        if (w < warp) at += warp_sum[w];
      base[b] = at;
    }
    __syncthreads();
    for (unsigned i0 = begin; i0 < end; i0 += 32 * K) {
      if (!HELD) {
        load(i0);
        rank_keys(i0);
      }
#pragma unroll
      for (int j = 0; j < K; j++) {
        if (i0 + j * 32 + lane < end) {
          const unsigned digit = (key[j] >> shift) & (bins - 1);
          // HELD: to[] counts from 0, the prefix over warps is in mine[]
          const unsigned at = base[digit] + to[j] + (HELD ? mine[digit] : 0);
          moved[at] = make_uint2(key[j], pos[j]);
        }
      }
    }
    // the keys have arrived, and block_total may be overwritten; a warp's
    // counts are its own by now
    cluster.barrier_arrive();
    clear_mine();
    cluster.barrier_wait();
  }
}

// The same for at most 4096 without passes: a key's place is how many come
// before it, which a warp counts for each key, 32 keys to a block.  The blocks
// do not wait for one another.  (With the rest of the gradient of 1000
// ids of 512 bf16: 17 us, and 27 us with the passes; of 4000: 24 and 31 us.)
constexpr unsigned kFewIds = kShadowBytes / 4;
__global__ void __launch_bounds__(kSortThreads)
few_ids_kernel(IndexArray ids, unsigned n, long long vocab, long long padding, Sorted out,
               unsigned sorting, Shadow shadow, int* bad) {
  __shared__ uint4 buffer[kShadowBytes / 16];
  let_next_kernel_start();
  if (blockIdx.x >= sorting) {
    write_shadow(shadow, buffer, blockIdx.x - sorting, gridDim.x - sorting);
    return;
  }
  unsigned* key = reinterpret_cast<unsigned*>(buffer);
  if (blockIdx.x == 0 && threadIdx.x < 2) out.count[threadIdx.x] = 0;
#pragma unroll 4
  for (unsigned j = threadIdx.x; j < n; j += kSortThreads)
    key[j] = key_of(ids, j, vocab, padding, bad);
  __syncthreads();
  const unsigned i = blockIdx.x * kSortWarps + (threadIdx.x >> 5);
  if (i >= n) return;
  const unsigned k = key[i];
  unsigned place = 0;
#pragma unroll 4
  for (unsigned j = threadIdx.x & 31; j < n; j += 32) place += key[j] < k + (j < i);
  place = __reduce_add_sync(0xffffffffu, place);
  if ((threadIdx.x & 31) == 0) out.pair[0][place] = make_uint2(k, i);
}

// Up to kTiledIds ids in two kernels, one block to 256 of them: sort_tiles_kernel
// places each within its tile of 512 by counting, then place_kernel, which has
// every tile's keys in shared memory, adds how many of each other tile's come
// before it, by binary search.  That leaves the other SMs no time for zeros, so
// it is for sums that are added to what is there: 32768 x 4096 bf16 149 us, and
// 154 us with sort_ids_kernel; 8000 x 300 f32 27 and 31 us.
constexpr unsigned kTile = 512, kTiledIds = 96 * kTile, kPerBlock = 256;
constexpr unsigned kTileStride = kTile + 4;    // words: tiles searched together, in other banks

// The sum over 4 adjacent lanes.
__device__ __forceinline__ unsigned sum4(unsigned x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

__global__ void __launch_bounds__(kSortThreads)
sort_tiles_kernel(IndexArray ids, unsigned n, long long vocab, long long padding, unsigned* keys,
                  unsigned* where, unsigned* count, int* bad) {
  __shared__ uint4 tile[kTile / 4];
  let_next_kernel_start();
  const unsigned first = blockIdx.x / 2 * kTile;
  unsigned* key = reinterpret_cast<unsigned*>(tile);
  if (blockIdx.x == 0 && threadIdx.x < 2) count[threadIdx.x] = 0;
  if (threadIdx.x < kTile) {
    const unsigned i = first + threadIdx.x;
    key[threadIdx.x] = i < n ? key_of(ids, i, vocab, padding, bad) : ~0u;
  }
  __syncthreads();
  const unsigned self = blockIdx.x % 2 * kPerBlock + threadIdx.x / 4;
  const unsigned k = key[self];
  unsigned place = 0;
#pragma unroll 4
  for (unsigned j = threadIdx.x % 4; j < kTile / 4; j += 4) {
    const uint4 x = tile[j];
    place += x.x < k + (4 * j < self);
    place += x.y < k + (4 * j + 1 < self);
    place += x.z < k + (4 * j + 2 < self);
    place += x.w < k + (4 * j + 3 < self);
  }
  place = sum4(place);
  if (threadIdx.x % 4 == 0 && first + self < n) {
    keys[first + place] = k;
    where[first + place] = first + self;
  }
}

__global__ void __launch_bounds__(kSortThreads)
place_kernel(const unsigned* keys, const unsigned* where, unsigned n, uint2* sorted) {
  extern __shared__ uint4 tiles[];      // [number of tiles][kTileStride / 4]
  let_next_kernel_start();
  const unsigned count = (n + kTile - 1) / kTile;
  wait_for_previous_kernel();
#pragma unroll 4
  for (unsigned v = threadIdx.x; v < count * (kTile / 4); v += kSortThreads) {
    uint4 x = make_uint4(~0u, ~0u, ~0u, ~0u);
    if (4 * v + 3 < n) {
      x = __ldcg(reinterpret_cast<const uint4*>(keys) + v);
    } else {
      if (4 * v < n) x.x = __ldcg(keys + 4 * v);
      if (4 * v + 1 < n) x.y = __ldcg(keys + 4 * v + 1);
      if (4 * v + 2 < n) x.z = __ldcg(keys + 4 * v + 2);
    }
    tiles[v / (kTile / 4) * (kTileStride / 4) + v % (kTile / 4)] = x;
  }
  __syncthreads();
  const unsigned* key = reinterpret_cast<const unsigned*>(tiles);
  const unsigned i = blockIdx.x * kPerBlock + threadIdx.x / 4;
  const unsigned mine = i / kTile;
  unsigned place = 0, k = 0;
  if (i < n) {
    k = key[mine * kTileStride + i % kTile];
#pragma unroll 4
    for (unsigned t = threadIdx.x % 4; t < count; t += 4) {
      const unsigned below = k + (t < mine);
      const unsigned* tile = key + t * kTileStride;
      unsigned lo = 0;
#pragma unroll
      for (unsigned step = kTile / 2; step > 0; step /= 2)
        if (tile[lo + step - 1] < below) lo += step;
      lo += tile[lo] < below;
      place += t == mine ? i % kTile : lo;
    }
  }
  place = sum4(place);
  if (i < n && threadIdx.x % 4 == 0) sorted[place] = make_uint2(k, __ldcg(where + i));
}

// ---- sums -------------------------------------------------------------------------

constexpr int kSub = 16;             // sorted positions whose ids are staged at a time
constexpr int kPiece = 32;           // positions to a piece, unless there are few or very many
constexpr size_t kMaxPieces = 2048;
constexpr size_t kFewPieces = 2048;  // at most, where pieces are cut shorter than kPiece
constexpr unsigned kLong = 16;       // a sum over more pieces than this is a long one
constexpr int kZeroRows = 64;        // at most, to a block that writes zeros
constexpr int kZeroBytes = 4096;     // zeros that it copies at a time

struct Plan {
  unsigned n, piece, pieces;
  const uint2* pair;      // sorted keys (.x) and positions
  unsigned* count;        // [2]: sums that cross pieces, and of those the long ones apart
  uint2* crossing;        // [pieces]: the piece where one begins, and its id
  uint2* crossing_long;   // [pieces / kLong + 1]
  float* partial;         // [pieces][2][ld]: a sum that began before the piece; one that ends later
  size_t ld;
  long long vocab;
  size_t width;
  float scale;
  bool accumulate;
  unsigned G, tiles, per_block;
  unsigned sum_blocks;    // then blocks that write zeros
  unsigned zero_rows;     // rows of the table for each of those
  long long zeroed;       // rows that have their zeros already
};

__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

template <int VW, class W, int N>
__device__ __forceinline__ void write_sum(const Plan& a, W* gw, unsigned id, size_t first,
                                          const float (&acc)[N]) {
  float v[N];
#pragma unroll
  for (int e = 0; e < N; e++) v[e] = fmul(acc[e], a.scale);
  W* row = gw + (size_t)id * a.width;
  if (a.accumulate) add_row<VW>(row, first, a.G, a.width, v);
  store_row<VW>(row, first, a.G, a.width, v);
}

// How many of the n sorted keys are below v: a warp looks at 32 places at a
// time.
__device__ __forceinline__ unsigned lower_bound(const uint2* key, unsigned n, unsigned v) {
  const unsigned lane = threadIdx.x & 31;
  unsigned lo = 0, hi = n;             // the answer is in [lo, hi]
  while (lo < hi) {
    const unsigned step = (hi - lo + 31) / 32;
    const unsigned at = lo + lane * step;      // below 2^31 + 2^31
    const unsigned below =
        __popc(__ballot_sync(0xffffffffu, at < hi && key[at].x < v));   // a prefix of the lanes
    if (below == 0) return lo;
    const unsigned last = lo + (below - 1) * step;
    hi = min(hi, last + step);
    lo = last + 1;
  }
  return lo;
}

template <class W>
__device__ __forceinline__ void write_zeros(const Plan& a, W* gw) {
  __shared__ unsigned here[kZeroRows / 32];      // the block's rows that have tokens
  __shared__ unsigned range[2];
  __shared__ uint4 zeros[kZeroBytes / 16];
  for (int i = threadIdx.x; i < kZeroBytes / 16; i += kThreads) zeros[i] = make_uint4(0, 0, 0, 0);
  const long long v0 = a.zeroed + (long long)(blockIdx.x - a.sum_blocks) * a.zero_rows;
  const int rows = (int)min((long long)a.zero_rows, a.vocab - v0);
  if (threadIdx.x < kZeroRows / 32) here[threadIdx.x] = 0;
  if (threadIdx.x < 64) {
    const unsigned w = threadIdx.x >> 5;
    const unsigned p = lower_bound(a.pair, a.n, (unsigned)v0 + (w ? rows : 0));
    if ((threadIdx.x & 31) == 0) range[w] = p;
  }
  __syncthreads();
  for (unsigned p = range[0] + threadIdx.x; p < range[1]; p += kThreads) {
    const unsigned r = a.pair[p].x - (unsigned)v0;
    atomicOr(&here[r >> 5], 1u << (r & 31));
  }
  fence_proxy_async_smem();
  __syncthreads();
  // Runs of rows without tokens, an eighth of the block's rows to a warp: the
  // 16-byte-aligned inside of a run as bulk copies of a block of zeros (one
  // instruction where stores would take one for each 512 bytes of a warp), the
  // ends element by element.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (rows + kThreads / 32 - 1) / (kThreads / 32);
  const int last = min((warp + 1) * each, rows);
  auto taken = [&](int r) { return (here[r >> 5] >> (r & 31)) & 1u; };
  for (int r = warp * each; r < last;) {
    if (taken(r)) {
      r++;
      continue;
    }
    int e = r + 1;
    while (e < last && !taken(e)) e++;
    char* b0 = reinterpret_cast<char*>(gw + (size_t)(v0 + r) * a.width);
    char* b1 = reinterpret_cast<char*>(gw + (size_t)(v0 + e) * a.width);
    char* a0 = b0 + (-reinterpret_cast<intptr_t>(b0) & 15);
    char* a1 = b1 - (reinterpret_cast<intptr_t>(b1) & 15);
    if (a0 >= a1) a0 = a1 = b1;
    for (W* q = reinterpret_cast<W*>(b0) + lane; reinterpret_cast<char*>(q) < a0; q += 32)
      *q = from_f32<W>(0.0f);
    for (W* q = reinterpret_cast<W*>(a1) + lane; reinterpret_cast<char*>(q) < b1; q += 32)
      *q = from_f32<W>(0.0f);
    for (char* q = a0 + (size_t)lane * sizeof zeros; q < a1; q += 32 * sizeof zeros)
      bulk_store(q, zeros, (unsigned)min((ptrdiff_t)sizeof zeros, (ptrdiff_t)(a1 - q)));
    r = e;
  }
  bulk_store_wait();   // `zeros` has been read
}

// The sums of pieces of the sorted list, a group of G threads to a piece (and to
// a tile of the row, where that is longer than a block covers), the rows added in
// the list's order in f32.  HBM bounds it: each gradient is read once, each row
// with tokens written (or added to) once, the others zeroed (32768 x 4096 bf16
// into 131072 rows f32: 119 us for 102 at the copy's rate).  U rows' loads in
// flight per thread (fewer where a row takes many narrow ones).
template <class T, class W, int VW>
__global__ void __launch_bounds__(kThreads)
segment_kernel(const T* g, W* gw, Plan a) {
  constexpr int N = Row<T>::N;
  constexpr int U = VW * sizeof(T) >= 8 ? 4 : 2;
  wait_for_previous_kernel();   // the sorted list
  let_next_kernel_start();
  if (blockIdx.x >= a.sum_blocks) {
    write_zeros(a, gw);
    return;
  }
  extern __shared__ unsigned staged[];   // per group: kSub keys, then kSub positions
  const unsigned group = threadIdx.x / a.G, lane = threadIdx.x % a.G;
  unsigned* skey = staged + group * 2 * kSub;
  unsigned* spos = skey + kSub;
  const size_t unit = (size_t)blockIdx.x * a.per_block + group;
  const unsigned piece = (unsigned)(unit / a.tiles);
  const size_t first = (size_t)(unit % a.tiles) * a.G * N + (size_t)lane * VW;
  const bool live = piece < a.pieces;
  const unsigned p0 = live ? piece * a.piece : a.n;
  const unsigned p1 = live ? min(p0 + a.piece, a.n) : a.n;
  const unsigned none = (unsigned)a.vocab;

  float acc[N];
#pragma unroll
  for (int e = 0; e < N; e++) acc[e] = 0.0f;
  unsigned cur = live ? a.pair[p0].x : none;
  bool head = live && p0 > 0 && a.pair[p0 - 1].x == cur;   // cur's sum began in an earlier piece
  float* part = a.partial + (size_t)piece * 2 * a.ld + first;

  auto put_partial = [&](int which) {
    float* o = part + which * a.ld;
#pragma unroll
    for (int k = 0; k < N / VW; k++)
#pragma unroll
      for (int e = 0; e < VW; e++) {
        const size_t c = (size_t)k * a.G * VW + e;
        if (first + c < a.width) o[c] = acc[k * VW + e];
      }
  };

  // every group of the block takes the same number of turns
  for (unsigned s0 = 0; s0 < a.piece; s0 += kSub) {
    __syncthreads();
    for (unsigned i = lane; i < kSub; i += a.G) {
      const unsigned p = p0 + s0 + i;
      const uint2 x = p < p1 ? a.pair[p] : make_uint2(none, 0);
      skey[i] = x.x;
      spos[i] = x.y;
    }
    __syncthreads();
    if (a.accumulate)
      for (unsigned i = 0; i < kSub; i++) {
        const unsigned k = skey[i];
        if (k != none && (i == 0 || skey[i - 1] != k) && first < a.width)
          prefetch_l2(gw + (size_t)k * a.width + first);
      }
    const unsigned turn = min((unsigned)kSub, a.piece);
    for (unsigned i = 0; i < turn; i += U) {
      Row<T> x[U];
#pragma unroll
      for (int u = 0; u < U; u++)
        if (skey[i + u] != none)
          load_row<VW>(g + (size_t)spos[i + u] * a.width, first, a.G, a.width, x[u]);
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (i + u >= turn) break;
        const unsigned k = skey[i + u];
        if (k != cur) {
          if (cur != none) {
            if (head) put_partial(0);
            else write_sum<VW>(a, gw, cur, first, acc);
          }
          head = false;
          cur = k;
#pragma unroll
          for (int e = 0; e < N; e++) acc[e] = 0.0f;
        }
        if (k != none) {
#pragma unroll
          for (int e = 0; e < N; e++) acc[e] = fadd(acc[e], to_f32(x[u].x[e]));
        }
      }
    }
  }
  // the last sum, unless padding or the end of the list closed it above
  if (cur != none) {
    const bool more = p1 < a.n && a.pair[p1].x == cur;
    if (head) put_partial(0);
    else if (more) put_partial(1);
    else write_sum<VW>(a, gw, cur, first, acc);
    if (!head && more && first == 0) {
      const size_t far = (size_t)(piece + kLong) * a.piece;
      const bool is_long = far < a.n && a.pair[far].x == cur;
      const unsigned e = atomicAdd(a.count + is_long, 1u);
      (is_long ? a.crossing_long : a.crossing)[e] = make_uint2(piece, cur);
    }
  }
}

// Joins the sums that cross pieces, 128 columns at a time.  Most take a few
// pieces: a warp adds the partial sums in order, four columns to a lane.  The
// long ones (at most pieces / kLong) get a block: its warps add an eighth of the
// pieces each, in order, then the eight are added in order.  Which block takes
// which sum does not matter.
template <class W>
__global__ void __launch_bounds__(kThreads)
join_kernel(W* gw, Plan a) {
  __shared__ float4 eighth[8][32];
  wait_for_previous_kernel();   // the partial sums
  const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t tiles = (a.width + 127) / 128;
  const size_t shorts = a.count[0] * tiles, longs = a.count[1] * tiles;
  for (size_t unit = blockIdx.x; unit < longs + (shorts + 7) / 8; unit += gridDim.x) {
    const bool is_long = unit < longs;
    const size_t u = is_long ? unit : (unit - longs) * 8 + warp;
    if (!is_long && u >= shorts) break;
    const uint2 which = (is_long ? a.crossing_long : a.crossing)[u / tiles];
    const unsigned piece = which.x;
    // the pieces after this one whose first key is still the id (keys are
    // sorted), 32 looked at together
    unsigned count = 1;   // partial sums: the first one's tail, then heads
    for (unsigned q = piece + 1; q < a.pieces; q += 32) {
      const bool more = q + lane < a.pieces && a.pair[(size_t)(q + lane) * a.piece].x == which.y;
      const unsigned m = __ballot_sync(0xffffffffu, more);
      count += __popc(m);
      if (m != 0xffffffffu) break;
    }
    const unsigned each = is_long ? (count + 7) / 8 : count;
    const unsigned j0 = is_long ? warp * each : 0, j1 = min(j0 + each, count);
    const size_t c = u % tiles * 128 + lane * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < a.width) {
#pragma unroll 8
      for (unsigned j = j0; j < j1; j++) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(
            a.partial + (size_t)(piece + j) * 2 * a.ld + (j == 0 ? a.ld : 0) + c));
        acc.x = fadd(acc.x, x.x);
        acc.y = fadd(acc.y, x.y);
        acc.z = fadd(acc.z, x.z);
        acc.w = fadd(acc.w, x.w);
      }
    }
    if (is_long) {
      eighth[warp][lane] = acc;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int k = 1; k < 8; k++) {
          const float4 x = eighth[k][lane];
          acc.x = fadd(acc.x, x.x);
          acc.y = fadd(acc.y, x.y);
          acc.z = fadd(acc.z, x.z);
          acc.w = fadd(acc.w, x.w);
        }
      }
    }
    if (!is_long || warp == 0) {
      const float v[4] = {acc.x, acc.y, acc.z, acc.w};
      W* row = gw + (size_t)which.y * a.width;
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (c + k < a.width) {
          const float r = fmul(v[k], a.scale);
          row[c + k] = from_f32<W>(a.accumulate ? fadd(to_f32(row[c + k]), r) : r);
        }
    }
    if (is_long) __syncthreads();   // `eighth` is free
  }
}

size_t up256(size_t b) { return (b + 255) & ~size_t(255); }

struct Layout {
  unsigned piece, pieces;
  unsigned G, tiles, per_block;
  size_t ld, list, crossing, partial, total;
};
size_t sum_blocks_of(size_t pieces, const Layout& l) {
  return (pieces * l.tiles + l.per_block - 1) / l.per_block;
}
Layout layout_of(StoreType t, size_t n, size_t width) {
  Layout l;
  const int N = 16 / (int)store_bytes(t);
  l.G = group_of(width, N);
  l.tiles = (unsigned)((width + (size_t)l.G * N - 1) / ((size_t)l.G * N));
  l.per_block = kThreads / l.G;
  size_t piece = kPiece;
  while ((n + piece - 1) / piece > kMaxPieces) piece *= 2;
  // Shorter ones where the blocks would leave SMs idle: a group's positions
  // come one after the other (1000 ids of 512 bf16, added to a table: 27 us, and
  // 37 us with 32 positions to a piece).
  constexpr size_t kBlocks = 2 * 148;
  while (piece > 1 && sum_blocks_of((n + piece - 1) / piece, l) < kBlocks &&
         (n + piece / 2 - 1) / (piece / 2) <= kFewPieces)
    piece /= 2;
  l.piece = (unsigned)piece;
  l.pieces = (unsigned)((n + piece - 1) / piece);
  l.ld = (width + 3) & ~size_t(3);
  l.list = up256(n * 8);
  l.crossing = up256(((size_t)l.pieces + l.pieces / kLong + 1) * 8);
  l.partial = (size_t)l.pieces * 2 * l.ld * 4;
  l.total = 256 + 2 * l.list + l.crossing + l.partial;
  return l;
}

cudaError_t sort_ids(IndexArray ids, unsigned n, size_t vocab, long long padding,
                     const Sorted& out, const Shadow& shadow, int* bad, int* passes_out,
                     cudaStream_t s) {
  int device = 0;
  cudaGetDevice(&device);
  const unsigned sms = (unsigned)sm_count(device);
  if (n <= kFewIds) {
    *passes_out = 0;
    const unsigned sorting = (n + kSortWarps - 1) / kSortWarps;
    const unsigned others = shadow.bytes ? std::max(sms > sorting ? sms - sorting : 0, sms / 2) : 0;
    few_ids_kernel<<<sorting + others, kSortThreads, 0, s>>>(ids, n, (long long)vocab, padding, out,
                                                           sorting, shadow, bad);
    return cudaGetLastError();
  }
  if (n <= kTiledIds && !shadow.bytes) {
    *passes_out = 0;
    unsigned* keys = reinterpret_cast<unsigned*>(out.pair[1]);
    unsigned* where = keys + n;
    const unsigned sorting = (n + kPerBlock - 1) / kPerBlock;
    cudaError_t e = cudaFuncSetAttribute(place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kTiledIds / kTile * kTileStride * 4);
    if (e != cudaSuccess) return e;
    sort_tiles_kernel<<<sorting, kSortThreads, 0, s>>>(ids, n, (long long)vocab, padding, keys,
                                                       where, out.count, bad);
    e = cudaGetLastError();
    return e != cudaSuccess ? e
                            : launch_after(place_kernel, sorting, kSortThreads,
                                           (n + kTile - 1) / kTile * kTileStride * 4, s, keys,
                                           where, n, out.pair[0]);
  }
  int total_bits = 1;
  while (total_bits < 32 && (vocab >> total_bits)) total_bits++;
  const int passes = (total_bits + kSortMaxBits - 1) / kSortMaxBits;
  const int bits = (total_bits + passes - 1) / passes;
  // a key a thread before another block joins
  unsigned blocks = 1;
  while (blocks < kSortMaxCluster && blocks * kSortThreads < n) blocks *= 2;
  const size_t smem = std::max<size_t>((size_t)kSortWarps * (1u << bits) * 4, kShadowBytes);
  const size_t per_warp = (n + (size_t)blocks * kSortWarps - 1) / ((size_t)blocks * kSortWarps);
  const auto kernel = per_warp <= 128 ? sort_ids_kernel<4, true> : sort_ids_kernel<4, false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kSortWarps * (1 << kSortMaxBits) * 4);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  unsigned others = 0;       // whole clusters, an SM to a block
  if (shadow.bytes) others = sms > 2 * blocks ? (sms - blocks) / blocks * blocks : blocks;
  cfg.gridDim = dim3(blocks + others);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  *passes_out = passes;
  return cudaLaunchKernelEx(&cfg, kernel, ids, n, (long long)vocab, padding, bits, passes,
                            out, shadow, bad);
}

template <class T, class W, int VW>
cudaError_t sums_of(const void* g, void* gw, Plan a, cudaStream_t s) {
  int device = 0;
  cudaGetDevice(&device);
  const unsigned sms = (unsigned)sm_count(device);
  const size_t sum_blocks = ((size_t)a.pieces * a.tiles + a.per_block - 1) / a.per_block;
  size_t zero_blocks = 0;
  if (!a.accumulate) {
    // 128 KB of the table to a block that writes zeros
    const size_t row = a.width * sizeof(W);
    a.zero_rows = (unsigned)std::max<size_t>(1, std::min<size_t>((size_t)131072 / row, kZeroRows));
    zero_blocks = ((size_t)(a.vocab - a.zeroed) + a.zero_rows - 1) / a.zero_rows;
  }
  if (sum_blocks + zero_blocks > 0x7fffffffull) return cudaErrorInvalidValue;
  a.sum_blocks = (unsigned)sum_blocks;
  const size_t smem = (size_t)a.per_block * 2 * kSub * 4;
  cudaError_t e = launch_after(segment_kernel<T, W, VW>, (unsigned)(sum_blocks + zero_blocks),
                               kThreads, smem, s, static_cast<const T*>(g), static_cast<W*>(gw),
                               a);
  if (e != cudaSuccess || a.pieces < 2) return e;
  const size_t tiles = (a.width + 127) / 128;
  const size_t blocks = std::min(a.pieces / 8 * tiles + (a.pieces / kLong + 1) * tiles,
                                 (size_t)16 * sms);
  return launch_after(join_kernel<W>, (unsigned)blocks, kThreads, 0, s, static_cast<W*>(gw), a);
}

template <class T, class W>
cudaError_t sums_any(const void* g, void* gw, const Plan& a, cudaStream_t s) {
  switch (chunk_of<T>(a.width, g, sizeof(T), gw, sizeof(W))) {
    case 8:
      if constexpr (sizeof(T) == 2) return sums_of<T, W, 8>(g, gw, a, s);
    case 4: return sums_of<T, W, 4>(g, gw, a, s);
    case 2: return sums_of<T, W, 2>(g, gw, a, s);
    default: return sums_of<T, W, 1>(g, gw, a, s);
  }
}

}  // namespace

cudaError_t launch_embedding(StoreType t, const void* weight, const void* ids, bool wide,
                             size_t n, size_t vocab, size_t width, float scale, void* out,
                             int* bad, cudaStream_t s) {
  if (n == 0 || width == 0) return cudaSuccess;
  const IndexArray ia{ids, wide};
  switch (t) {
    case kF32: return embedding_any<float>(weight, ia, n, vocab, width, scale, out, bad, s);
    case kBF16: return embedding_any<bf16>(weight, ia, n, vocab, width, scale, out, bad, s);
    case kF16: return embedding_any<f16>(weight, ia, n, vocab, width, scale, out, bad, s);
  }
  return cudaErrorInvalidValue;
}

size_t embedding_backward_scratch(StoreType t, size_t n, size_t width) {
  return layout_of(t, n, width).total;
}

cudaError_t launch_embedding_backward(StoreType t, const void* grad_output, const void* ids,
                                      bool wide, size_t n, size_t vocab, size_t width,
                                      float scale, long long padding, bool accumulate,
                                      void* grad_weight, bool narrow, void* scratch, int* bad,
                                      cudaStream_t s) {
  if (vocab == 0 || width == 0) return cudaSuccess;
  if (n == 0)
    return accumulate ? cudaSuccess
                      : cudaMemsetAsync(grad_weight, 0,
                                        vocab * width * (narrow ? store_bytes(t) : 4), s);
  const Layout l = layout_of(t, n, width);
  char* p = static_cast<char*>(scratch);
  Sorted sorted;
  sorted.count = reinterpret_cast<unsigned*>(p);
  p += 256;
  sorted.pair[0] = reinterpret_cast<uint2*>(p);
  sorted.pair[1] = reinterpret_cast<uint2*>(p + l.list);
  p += 2 * l.list;
  // What the other SMs can zero while one cluster sorts, which takes about 8 us
  // and 0.4 us for each 1000 ids.  Rows with tokens among it are written again,
  // which costs less than the wait (16384 x 1024 f32 into 50257 rows: 64 us for
  // 71).
  const size_t row = width * (narrow ? store_bytes(t) : 4);
  size_t zeroed = 0;
  Shadow shadow = {static_cast<char*>(grad_weight), 0};
  if (!accumulate) {
    zeroed = std::min(vocab, (((size_t)48 << 20) + std::min<size_t>(n, 32768) * 2048) / row);
    shadow.bytes = zeroed * row;
  }
  int passes = 0;
  const cudaError_t e = sort_ids(IndexArray{ids, wide}, (unsigned)n, vocab, padding, sorted,
                                 shadow, bad, &passes, s);
  if (e != cudaSuccess) return e;
  Plan a = {};
  a.n = (unsigned)n;
  a.piece = l.piece;
  a.pieces = l.pieces;
  a.G = l.G;
  a.tiles = l.tiles;
  a.per_block = l.per_block;
  a.pair = sorted.pair[passes & 1];
  a.count = sorted.count;
  a.crossing = reinterpret_cast<uint2*>(p);
  a.crossing_long = a.crossing + l.pieces;
  a.partial = reinterpret_cast<float*>(p + l.crossing);
  a.ld = l.ld;
  a.vocab = (long long)vocab;
  a.width = width;
  a.scale = scale;
  a.accumulate = accumulate;
  a.zeroed = (long long)zeroed;
  switch (t) {
    case kF32: return sums_any<float, float>(grad_output, grad_weight, a, s);
    case kBF16:
      return narrow ? sums_any<bf16, bf16>(grad_output, grad_weight, a, s)
                    : sums_any<bf16, float>(grad_output, grad_weight, a, s);
    case kF16:
      return narrow ? sums_any<f16, f16>(grad_output, grad_weight, a, s)
                    : sums_any<f16, float>(grad_output, grad_weight, a, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace rt
