// Scaled embedding lookup and its gradient by sorted tokens.
//   out[i] = scale * W[ids[i]]               dW[v] = scale * sum over i with ids[i] = v of dout[i]
// The lookup copies rows (bound by memory; one rounding, none when the scale is 1).  The gradient sorts the
// (id, position) pairs with a stable radix sort, so that each table row's tokens form one run in token order, and
// sums every run in fp32 in that order: no atomics on values, the same bits every time.
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

// ---- lookup ----------------------------------------------------------------------------------------
template <int BYTES>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<2> { using type = uint16_t; };

template <typename T, int BYTES>
__device__ __forceinline__ typename Word<BYTES>::type scale_word(typename Word<BYTES>::type w, float scale) {
  constexpr int N = BYTES / static_cast<int>(sizeof(T));
  T v[N];
  memcpy(v, &w, BYTES);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = from_f32<T>(to_f32(v[i]) * scale);
  memcpy(&w, v, BYTES);
  return w;
}

// One warp per (token, chunk of 32 * 4 words of the row).  An id outside the table gives a row of NaN.
template <typename T, int BYTES>
__global__ void __launch_bounds__(256) lookup_kernel(IntList ids, int64_t n, const T* __restrict__ table,
                                                     int64_t vocab, int64_t hidden, int64_t ld, float scale, T* out,
                                                     int chunks) {
  using W = typename Word<BYTES>::type;
  constexpr int N = BYTES / static_cast<int>(sizeof(T));
  const int lane = threadIdx.x & 31;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t i = item / chunks;
  if (i >= n) return;
  const int64_t words = hidden / N;
  const int64_t c0 = (item - i * chunks) * 128 + lane;
  const int64_t id = ids[i];
  W* dst = reinterpret_cast<W*>(out + i * hidden);
  if (id < 0 || id >= vocab) {
    for (int u = 0; u < 4; ++u) {
      const int64_t c = c0 + u * 32;
      if (c < words)
        for (int e = 0; e < N; ++e) out[i * hidden + c * N + e] = from_f32<T>(NAN);
    }
    return;
  }
  const W* src = reinterpret_cast<const W*>(table + id * ld);
  W v[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (c0 + u * 32 < words) v[u] = __ldg(src + c0 + u * 32);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (c0 + u * 32 < words) dst[c0 + u * 32] = scale == 1.0f ? v[u] : scale_word<T, BYTES>(v[u], scale);
}

template <typename T, int BYTES>
cudaError_t lookup_words(IntList ids, int64_t n, const void* table, int64_t vocab, int64_t hidden, int64_t ld,
                         float scale, void* out, cudaStream_t stream) {
  const int64_t words = hidden * static_cast<int64_t>(sizeof(T)) / BYTES;
  const int64_t chunks = (words + 127) / 128;
  lookup_kernel<T, BYTES><<<static_cast<unsigned>((n * chunks + 7) / 8), 256, 0, stream>>>(
      ids, n, static_cast<const T*>(table), vocab, hidden, ld, scale, static_cast<T*>(out), static_cast<int>(chunks));
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t lookup_t(IntList ids, int64_t n, const void* table, int64_t vocab, int64_t hidden, int64_t ld, float scale,
                     void* out, cudaStream_t stream) {
  // widest word that divides every row's start and length
  const uint64_t bits = reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out) |
                        static_cast<uint64_t>(ld) * sizeof(T) | static_cast<uint64_t>(hidden) * sizeof(T);
  if (bits % 16 == 0) return lookup_words<T, 16>(ids, n, table, vocab, hidden, ld, scale, out, stream);
  if (bits % 8 == 0) return lookup_words<T, 8>(ids, n, table, vocab, hidden, ld, scale, out, stream);
  if (bits % 4 == 0) return lookup_words<T, 4>(ids, n, table, vocab, hidden, ld, scale, out, stream);
  if constexpr (sizeof(T) == 2) return lookup_words<T, 2>(ids, n, table, vocab, hidden, ld, scale, out, stream);
  return cudaErrorMisalignedAddress;
}

// ---- stable radix sort of the ids --------------------------------------------------------------------
constexpr int kSortTile = 2048, kSortThreads = 256, kDigits = 256;

// Ids that add nothing (the padding row's, ids outside the table) take the key `vocab` and end up last.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t vocab, int64_t padding) {
  return static_cast<uint32_t>(id < 0 || id >= vocab || id == padding ? vocab : id);
}

__global__ void __launch_bounds__(kSortThreads) sort_keys_kernel(IntList ids, int64_t n, int64_t vocab, int64_t padding,
                                                                 uint32_t* __restrict__ keys,
                                                                 uint32_t* __restrict__ pos) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kSortThreads + threadIdx.x;
  if (i < n) {
    keys[i] = sort_key(ids[i], vocab, padding);
    pos[i] = static_cast<uint32_t>(i);
  }
}

__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(const uint32_t* __restrict__ keys, int64_t n, int shift,
                                                                 uint32_t* __restrict__ hist, int blocks) {
  __shared__ uint32_t h[kDigits];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kSortTile;
  for (int i = threadIdx.x; i < kSortTile; i += kSortThreads)
    if (lo + i < n) atomicAdd(&h[(keys[lo + i] >> shift) & (kDigits - 1)], 1u);
  __syncthreads();
  hist[static_cast<int64_t>(threadIdx.x) * blocks + blockIdx.x] = h[threadIdx.x];
}

// Exclusive scan of the (digit, block) counts by one block.
__global__ void __launch_bounds__(1024) sort_scan_kernel(uint32_t* hist, int64_t count) {
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t carry;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t base = 0; base < count; base += 1024) {
    const int64_t i = base + threadIdx.x;
    const uint32_t v = i < count ? hist[i] : 0;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[warp] = x;
    __syncthreads();
    uint32_t before = carry;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    if (i < count) hist[i] = before + x - v;
    __syncthreads();
    if (threadIdx.x == 1023) carry = before + x;
    __syncthreads();
  }
}

// Each warp ranks 256 consecutive keys of its tile, 32 at a time, in order.
__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(const uint32_t* __restrict__ keys,
                                                                    const uint32_t* __restrict__ pos, int64_t n,
                                                                    int shift, const uint32_t* __restrict__ hist,
                                                                    int blocks, uint32_t* __restrict__ keys_out,
                                                                    uint32_t* __restrict__ pos_out) {
  constexpr int kWarps = kSortThreads / 32, kPer = kSortTile / kWarps / 32;
  __shared__ uint32_t start[kWarps][kDigits];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = lane; d < kDigits; d += 32) start[warp][d] = 0;
  __syncwarp();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (kSortTile / kWarps);
  uint32_t key[kPer], rank[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int64_t i = lo + u * 32 + lane;
    key[u] = i < n ? keys[i] : 0xffffffffu;
    const uint32_t d = i < n ? (key[u] >> shift) & (kDigits - 1) : kDigits;
    const uint32_t peers = __match_any_sync(0xffffffffu, d);
    uint32_t base = 0;
    if (d < kDigits) base = start[warp][d];
    rank[u] = base + __popc(peers & ((1u << lane) - 1u));
    __syncwarp();
    if (d < kDigits && lane == 31 - __clz(peers)) start[warp][d] = base + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  {
    uint32_t x = hist[static_cast<int64_t>(threadIdx.x) * blocks + blockIdx.x];
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t c = start[w][threadIdx.x];
      start[w][threadIdx.x] = x;
      x += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const int64_t i = lo + u * 32 + lane;
    if (i < n) {
      const uint32_t to = start[warp][(key[u] >> shift) & (kDigits - 1)] + rank[u];
      keys_out[to] = key[u];
      pos_out[to] = pos[i];
    }
  }
}

// ---- gradient -----------------------------------------------------------------------------------------
struct EmbedGradArgs {
  const uint32_t *keys, *pos;  // sorted
  int64_t n, vocab, hidden, ld_grad, ld_out;
  float scale;
  int32_t accumulate;
};

// First sorted position whose key is >= v.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* __restrict__ keys, int64_t n, uint32_t v) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (__ldg(keys + mid) < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// One warp per table row: the run is summed in token order, a column at a time per lane.
template <typename G, typename O>
__global__ void __launch_bounds__(256) embed_grad_kernel(EmbedGradArgs a, const G* __restrict__ grad, O* out) {
  const int lane = threadIdx.x & 31;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (v >= a.vocab) return;
  const int64_t lo = lower_bound(a.keys, a.n, static_cast<uint32_t>(v));
  int64_t hi = lo;
  while (hi < a.n && __ldg(a.keys + hi) == static_cast<uint32_t>(v)) ++hi;
  O* o = out + v * a.ld_out;
  if (lo == hi && a.accumulate) return;
  for (int64_t c = lane; c < a.hidden; c += 32) {
    float s = 0.0f;
    for (int64_t i = lo; i < hi; ++i) s += to_f32(grad[static_cast<int64_t>(__ldg(a.pos + i)) * a.ld_grad + c]);
    s *= a.scale;
    if (a.accumulate) s += to_f32(o[c]);
    o[c] = from_f32<O>(s);
  }
}

struct EmbedPlan {
  int64_t n, blocks;
  int passes;
  size_t bytes;
};
EmbedPlan embed_plan(int64_t n, int64_t vocab) {
  EmbedPlan p;
  p.n = n;
  p.blocks = (n + kSortTile - 1) / kSortTile;
  p.passes = 1;
  while ((vocab >> (8 * p.passes)) > 0) ++p.passes;
  p.bytes = static_cast<size_t>(16 * n) + static_cast<size_t>(p.blocks) * kDigits * 4;
  return p;
}

template <typename G, typename O>
cudaError_t embed_grad_t(EmbedGradArgs a, const void* grad, void* out, cudaStream_t stream) {
  embed_grad_kernel<G, O><<<static_cast<unsigned>((a.vocab + 7) / 8), 256, 0, stream>>>(
      a, static_cast<const G*>(grad), static_cast<O*>(out));
  count_launch();
  return cudaGetLastError();
}

cudaError_t sort_ids(IntList ids, int64_t n, int64_t vocab, int64_t padding, void* workspace, EmbedGradArgs& a,
                     cudaStream_t stream) {
  const EmbedPlan p = embed_plan(n, vocab);
  uint32_t* k0 = static_cast<uint32_t*>(workspace);
  uint32_t *p0 = k0 + n, *k1 = p0 + n, *p1 = k1 + n, *hist = p1 + n;
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  sort_keys_kernel<<<static_cast<unsigned>((n + kSortThreads - 1) / kSortThreads), kSortThreads, 0, stream>>>(
      ids, n, vocab, padding, k0, p0);
  count_launch();
  for (int q = 0; q < p.passes; ++q) {
    sort_hist_kernel<<<blocks, kSortThreads, 0, stream>>>(k0, n, 8 * q, hist, static_cast<int>(p.blocks));
    sort_scan_kernel<<<1, 1024, 0, stream>>>(hist, p.blocks * kDigits);
    sort_scatter_kernel<<<blocks, kSortThreads, 0, stream>>>(k0, p0, n, 8 * q, hist, static_cast<int>(p.blocks), k1, p1);
    count_launch(3);
    std::swap(k0, k1);
    std::swap(p0, p1);
  }
  a.keys = k0;
  a.pos = p0;
  return cudaGetLastError();
}

}  // namespace mib
