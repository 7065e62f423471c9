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

// One warp per (token, chunk of 32 * 4 words of the row), four loads in flight a lane.  Bound by memory: 16384 tokens of
// 1024 fp32 in 14 us, 6.9 TB/s of distinct rows read and rows written.  An id outside the table gives a row of NaN.
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
  if (chunks > (int64_t(1) << 33) / n) return cudaErrorInvalidValue;
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

// ---- stable radix sort of the ids: up to 65536 tokens in one launch -------------------------------------
// The blocks of one cluster (8, or a single block for up to 2048 tokens) hold all (id, position) pairs in registers
// and sort them by up to 9 bits a pass, least significant first: ranks within a warp by match, counts of the warps
// and blocks added through (distributed) shared memory.  151936 rows take two passes (16384 tokens: 16 us).  The zeros
// of a dense gradient are written by a kernel that does not wait for the sort until it has written them.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kBins = 512, kSortCluster = 8;

struct SortArgs {
  IntList ids;
  int64_t n, vocab, padding;
  uint32_t *keys0, *keys1, *pos0, *pos1;  // scratch: even passes write 0, odd ones 1
  int32_t passes, bits;
  uint32_t* heads;             // [0]: number of split runs, zeroed here
};

// A dense gradient to be cleared.
struct ZeroArgs {
  void* p;
  int64_t rows, row_bytes, pitch;
};

// Ids that add nothing (the padding row's, ids outside the table) take the key `vocab` and end up last.
__device__ __forceinline__ uint32_t sort_key(int64_t id, int64_t vocab, int64_t padding) {
  return static_cast<uint32_t>(id < 0 || id >= vocab || id == padding ? vocab : id);
}

// One block per 32 KB of a dense table: 622 MB in 83 us, 7.5 TB/s.
__global__ void __launch_bounds__(512) zero_kernel(ZeroArgs a) {
  pdl_release();
  char* p = static_cast<char*>(a.p);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (a.pitch == a.row_bytes && reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    const int64_t bytes = a.rows * a.row_bytes, vecs = bytes / 16;
    uint4* v = reinterpret_cast<uint4*>(p);
    for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * 2048 + threadIdx.x; i0 < vecs; i0 += gridDim.x * 2048ll) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * 512 < vecs) v[i0 + u * 512] = make_uint4(0, 0, 0, 0);
    }
    for (int64_t i = vecs * 16 + first * 2; i < bytes; i += stride * 2) *reinterpret_cast<uint16_t*>(p + i) = 0;
  } else {
    const int64_t per = a.row_bytes / 2;
    for (int64_t i = first; i < a.rows * per; i += stride)
      *reinterpret_cast<uint16_t*>(p + i / per * a.pitch + i % per * 2) = 0;
  }
  pdl_wait();  // the kernel behind this one waits for this one alone, and needs the sort too
}

template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(SortArgs a) {
  __shared__ uint16_t count[kSortWarps][kBins];
  __shared__ uint16_t total[kSortCluster][kBins];
  __shared__ uint32_t base[kBins];
  __shared__ uint32_t warp_sum[kBins / 32];
  pdl_release();
  const uint32_t nranks = cluster_size(), rank = cluster_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (rank == 0 && threadIdx.x == 0) a.heads[0] = 0;
  if (nranks > 1) cluster_arrive();  // waited for in front of the first remote store
  const int64_t first = (static_cast<int64_t>(rank) * kSortWarps + warp) * (32 * ITEMS) + lane;
  for (int q = 0; q < a.passes; ++q) {
    const int shift = q * a.bits;
    const uint32_t* keys_in = (q & 1) ? a.keys0 : a.keys1;
    const uint32_t* pos_in = (q & 1) ? a.pos0 : a.pos1;
    uint32_t* keys_out = (q & 1) ? a.keys1 : a.keys0;
    uint32_t* pos_out = (q & 1) ? a.pos1 : a.pos0;
    const uint32_t mask = (1u << a.bits) - 1u;
    uint32_t key[ITEMS], val[ITEMS], rnk[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const int64_t i = first + u * 32;
      key[u] = 0;
      val[u] = static_cast<uint32_t>(i);
      if (i < a.n) {
        if (q == 0) {
          key[u] = sort_key(a.ids[i], a.vocab, a.padding);
        } else {
          key[u] = __ldcg(keys_in + i);
          val[u] = __ldcg(pos_in + i);
        }
      }
    }
    for (int d = lane; d < kBins; d += 32) count[warp][d] = 0;
    __syncwarp();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const uint32_t d = first + u * 32 < a.n ? (key[u] >> shift) & mask : kBins;
      const uint32_t peers = __match_any_sync(0xffffffffu, d);
      const uint32_t seen = d < kBins ? count[warp][d] : 0;
      rnk[u] = seen + __popc(peers & ((1u << lane) - 1u));
      __syncwarp();
      if (d < kBins && lane == 31 - __clz(peers)) count[warp][d] = static_cast<uint16_t>(seen + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    if (nranks > 1 && q == 0) cluster_wait();
    if (threadIdx.x < kBins) {  // counts of the warps in front, and the block's own total to every block
      const int d = threadIdx.x;
      uint32_t s = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = count[w][d];
        count[w][d] = static_cast<uint16_t>(s);
        s += c;
      }
      if (nranks > 1) {
        for (uint32_t b = 0; b < nranks; ++b) {
          uint32_t to;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(&total[rank][d])), "r"(b));
          asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(to), "h"(static_cast<uint16_t>(s)) : "memory");
        }
      } else {
        total[0][d] = static_cast<uint16_t>(s);
      }
    }
    if (nranks > 1) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();
    }
    uint32_t all = 0, before = 0, scan = 0;
    if (threadIdx.x < kBins) {
      for (uint32_t b = 0; b < nranks; ++b) {
        const uint32_t c = total[b][threadIdx.x];
        if (b < rank) before += c;
        all += c;
      }
      scan = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += y;
      }
      if (lane == 31) warp_sum[warp] = scan;
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      for (int w = 0; w < warp; ++w) scan += warp_sum[w];
      base[threadIdx.x] = scan - all + before;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      if (first + u * 32 < a.n) {
        const uint32_t d = (key[u] >> shift) & mask;
        const uint32_t to = base[d] + count[warp][d] + rnk[u];
        keys_out[to] = key[u];
        pos_out[to] = val[u];
      }
    }
    if (q + 1 < a.passes) {
      if (nranks > 1) {
        cluster_arrive();
        cluster_wait();
      } else {
        __threadfence();
        __syncthreads();
      }
    }
  }
}

// ---- the same sort for more tokens: 8 bits a pass, three launches each ------------------------------------
constexpr int kTile = 2048, kTileThreads = 256, kDigits = 256;


__global__ void __launch_bounds__(kTileThreads) sort_keys_kernel(IntList ids, int64_t n, int64_t vocab, int64_t padding,
                                                                 uint32_t* __restrict__ keys,
                                                                 uint32_t* __restrict__ pos, uint32_t* heads) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kTileThreads + threadIdx.x;
  if (i < n) {
    keys[i] = sort_key(ids[i], vocab, padding);
    pos[i] = static_cast<uint32_t>(i);
  }
  if (i == 0) heads[0] = 0;
}

__global__ void __launch_bounds__(kTileThreads) sort_hist_kernel(const uint32_t* __restrict__ keys, int64_t n, int shift,
                                                                 uint32_t* __restrict__ hist, int blocks) {
  __shared__ uint32_t h[kDigits];
  h[threadIdx.x] = 0;
  __syncthreads();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kTile;
  for (int i = threadIdx.x; i < kTile; i += kTileThreads)
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
__global__ void __launch_bounds__(kTileThreads) sort_scatter_kernel(const uint32_t* __restrict__ keys,
                                                                    const uint32_t* __restrict__ pos, int64_t n,
                                                                    int shift, const uint32_t* __restrict__ hist,
                                                                    int blocks, uint32_t* __restrict__ keys_out,
                                                                    uint32_t* __restrict__ pos_out) {
  constexpr int kWarps = kTileThreads / 32, kPer = kTile / kWarps / 32;
  __shared__ uint32_t start[kWarps][kDigits];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = lane; d < kDigits; d += 32) start[warp][d] = 0;
  __syncwarp();
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kTile + warp * (kTile / kWarps);
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
// The sorted positions are cut into chunks; a group of threads, one per column vector, walks its chunk's tokens in
// order, eight rows in flight in its part of shared memory, and writes each run that lies inside the chunk.  A run that crosses chunk borders
// leaves one partial sum per chunk (slot 0 of the chunks it enters, slot 1 of the one it starts in), and its first
// chunk goes on the list of split runs, which the join kernel adds up, in order.  The cut depends on the shape alone, so
// the bits are the same every time.  16384 tokens of 1024 fp32 (Zipf's law): sums 19 us, 4.8 TB/s, bound by the latency
// of a chunk's dependent loads (with the rows in registers, 64 of them or more, 27 - 40 us); the join 9 us.
struct EmbedGradArgs {
  const uint32_t *keys, *pos;  // sorted
  int64_t n, vocab, hidden, ld_grad, ld_out;
  float scale;
  int32_t accumulate, chunk;
  float* partial;              // [chunks][2][hidden]
  uint32_t* heads;             // [0] number, [1 ...] first chunks of the split runs
  const void* grad;
  void* out;
};

// V consecutive elements.
template <typename T, int V>
__device__ __forceinline__ void load_cols(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (V == kVec16<T>) {
    unpack16<T>(*reinterpret_cast<const uint4*>(p), v);
  } else {  // fp32 in vectors of 16-bit elements' length
    float a[4], b[4];
    unpack16<float>(*reinterpret_cast<const uint4*>(p), a);
    unpack16<float>(*(reinterpret_cast<const uint4*>(p) + 1), b);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[e + 4] = b[e];
    }
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_cols(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (V == kVec16<T>) {
    *reinterpret_cast<uint4*>(p) = pack16<T>(v);
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

template <typename O, int V>
__device__ __forceinline__ void write_run(const EmbedGradArgs& a, uint32_t row, int64_t col, float (&s)[V]) {
  O* o = static_cast<O*>(a.out) + static_cast<int64_t>(row) * a.ld_out + col;
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] *= a.scale;
  if (a.accumulate) {
    float old[V];
    load_cols<O, V>(o, old);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += old[e];
  }
  store_cols<O, V>(o, s);
}

// V columns of a row on their way through a thread's own places in shared memory: 16-byte asynchronous copies, or plain
// loads where rows are off that alignment.
template <typename G, int V>
struct Staged {
  using type = uint4;
  static __device__ __forceinline__ void start(uint4* to, const G* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  }
  static __device__ __forceinline__ void add(const uint4& u, float (&s)[V]) {
    float v[V];
    unpack16<G>(u, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] += v[e];
  }
};
template <typename G>
struct Staged<G, 1> {
  using type = G;
  static __device__ __forceinline__ void start(G* to, const G* from) { *to = *from; }
  static __device__ __forceinline__ void add(G u, float (&s)[1]) { s[0] += to_f32(u); }
};

template <typename G, typename O, int V>
__global__ void __launch_bounds__(256) embed_sum_kernel(EmbedGradArgs a) {
  constexpr int kAhead = 8;  // rows in flight
  using S = Staged<G, V>;
  __shared__ typename S::type stage[kAhead + 1][256];
  pdl_release();
  pdl_wait();
  const int64_t col = (static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x) * V;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t begin = c * a.chunk;
  if (begin >= a.n) return;  // the whole warp: a row of threads is a multiple of 32
  const int len = static_cast<int>(a.n - begin < a.chunk ? a.n - begin : a.chunk);  // at most 64
  const bool mine = col < a.hidden;
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, lane = tid & 31;
  const uint32_t none = static_cast<uint32_t>(a.vocab);
  // the chunk's keys and positions, two a lane, and the keys in front of it and behind it
  uint32_t key[2], pos[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = h * 32 + lane;
    key[h] = t < len ? __ldcg(a.keys + begin + t) : none;
    pos[h] = t < len ? __ldcg(a.pos + begin + t) : 0;
  }
  const uint32_t in = begin > 0 ? __ldcg(a.keys + begin - 1) : none;
  const uint32_t out = begin + len < a.n ? __ldcg(a.keys + begin + len) : none;
  const G* grad = static_cast<const G*>(a.grad) + (mine ? col : 0);
  auto key_at = [&](int t) { return __shfl_sync(0xffffffffu, t < 32 ? key[0] : key[1], t & 31); };
  auto start = [&](int t, int slot) {
    if (t < len) {
      const uint32_t p = __shfl_sync(0xffffffffu, t < 32 ? pos[0] : pos[1], t & 31);
      if (key_at(t) != none && mine) S::start(&stage[slot][tid], grad + static_cast<int64_t>(p) * a.ld_grad);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int t = 0; t < kAhead; ++t) start(t, t);
  uint32_t run = key_at(0);
  bool entered = run == in;  // the run began in an earlier chunk
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.0f;
  int slot = 0;
#pragma unroll 1
  for (int t = 0; t < len; ++t) {
    const uint32_t k = key_at(t);  // uniform over the chunk's threads
    if (k != run) {
      if (mine) {
        if (entered) store_cols<float, V>(a.partial + (2 * c) * a.hidden + col, s);
        else write_run<O, V>(a, run, col, s);
      }
      entered = false;
      run = k;
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] = 0.0f;
    }
    if (run == none) break;
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    if (mine) S::add(stage[slot][tid], s);
    start(t + kAhead, slot == 0 ? kAhead : slot - 1);  // the place that the row before had
    slot = slot == kAhead ? 0 : slot + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (run == none) return;
  if (!entered && run == out) {
    if (mine) store_cols<float, V>(a.partial + (2 * c + 1) * a.hidden + col, s);
    if (blockIdx.y == 0 && threadIdx.x == 0) a.heads[1 + atomicAdd(a.heads, 1u)] = static_cast<uint32_t>(c);
  } else if (mine) {
    if (entered) store_cols<float, V>(a.partial + (2 * c) * a.hidden + col, s);
    else write_run<O, V>(a, run, col, s);
  }
}

// Adds up the split runs: 32 column vectors and 8 stretches of a run's chunks per block, the stretches' sums joined
// in order.
template <typename O, int V>
__global__ void __launch_bounds__(256) embed_join_kernel(EmbedGradArgs a) {
  __shared__ float part[8][V][33];
  pdl_wait();
  const int lane = threadIdx.x & 31, g = threadIdx.x >> 5;
  const uint32_t tiles = static_cast<uint32_t>((a.hidden + 32 * V - 1) / (32 * V)), count = __ldcg(a.heads) * tiles;
  const int64_t chunks = (a.n + a.chunk - 1) / a.chunk;
  for (uint32_t h = blockIdx.x; h < count; h += gridDim.x) {
    const int64_t c = __ldcg(a.heads + 1 + h / tiles), col = (static_cast<int64_t>(h % tiles) * 32 + lane) * V;
    const uint32_t run = __ldcg(a.keys + (c + 1) * a.chunk);
    // chunks c + 1 .. c + m hold the rest, in their slot 0: those whose first key is still the run's
    int64_t m = 1;
    for (;;) {
      const int64_t at = c + 1 + m + lane;
      const uint32_t same = __ballot_sync(0xffffffffu, at < chunks && __ldcg(a.keys + at * a.chunk) == run);
      m += same == 0xffffffffu ? 32 : __ffs(~same) - 1;
      if (same != 0xffffffffu) break;
    }
    const int64_t per = (m + 7) / 8, first = g * per, last = first + per < m ? first + per : m;
    float s[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 0.0f;
    if (col < a.hidden) {
      const float* p = a.partial + col;
      if (g == 0) load_cols<float, V>(p + (2 * c + 1) * a.hidden, s);
#pragma unroll 4
      for (int64_t i = first; i < last; ++i) {
        float v[V];
        load_cols<float, V>(p + 2 * (c + 1 + i) * a.hidden, v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) part[g][e][lane] = s[e];
    __syncthreads();
    if (g == 0 && col < a.hidden) {
      for (int w = 1; w < 8; ++w)
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += part[w][e][lane];
      write_run<O, V>(a, run, col, s);
    }
    __syncthreads();
  }
}

struct EmbedPlan {
  int items, cluster, passes, bits;  // items 0: the multi-launch sort
  int64_t blocks, chunk, chunks;
  size_t keys, hist, heads, partial, bytes;
};
// Chunks of 8 to 64 tokens, for about 512 blocks of 256 threads, a thread per four columns.
EmbedPlan embed_plan(int64_t n, int64_t vocab, int64_t hidden) {
  EmbedPlan p{};
  int width = 1;
  while ((vocab >> width) > 0) ++width;  // keys are 0 .. vocab
  p.blocks = (n + kTile - 1) / kTile;
  if (n <= 65536) {
    p.cluster = n <= 2 * kSortThreads ? 1 : kSortCluster;
    const int64_t per = static_cast<int64_t>(p.cluster) * kSortThreads;
    p.items = n <= per ? 1 : (n <= 2 * per ? 2 : (n <= 4 * per ? 4 : 8));
    p.passes = (width + 8) / 9;
    p.bits = (width + p.passes - 1) / p.passes;
  } else {
    p.passes = (width + 7) / 8;
  }
  p.chunk = 8;
  const int64_t threads = (hidden + 127) / 128 * 32;
  while (p.chunk < 64 && n * threads > p.chunk * 512 * 256) p.chunk *= 2;
  p.chunks = (n + p.chunk - 1) / p.chunk;
  auto take = [&](size_t bytes) {
    const size_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.keys = take(16 * static_cast<size_t>(n));
  p.hist = take(p.items ? 0 : static_cast<size_t>(p.blocks) * kDigits * 4);
  p.heads = take(4 * static_cast<size_t>(p.chunks + 1));
  p.partial = take(8 * static_cast<size_t>(p.chunks) * static_cast<size_t>(hidden));
  return p;
}

cudaError_t sort_tiles(const SortArgs& s, const EmbedPlan& p, uint32_t* hist, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(p.blocks);
  const int b = static_cast<int>(p.blocks);
  sort_keys_kernel<<<static_cast<unsigned>((s.n + kTileThreads - 1) / kTileThreads), kTileThreads, 0, stream>>>(
      s.ids, s.n, s.vocab, s.padding, s.keys1, s.pos1, s.heads);
  count_launch();
  for (int q = 0; q < p.passes; ++q) {
    uint32_t *keys_in = s.keys1, *pos_in = s.pos1, *keys_out = s.keys0, *pos_out = s.pos0;
    if (q & 1) {
      std::swap(keys_in, keys_out);
      std::swap(pos_in, pos_out);
    }
    sort_hist_kernel<<<blocks, kTileThreads, 0, stream>>>(keys_in, s.n, 8 * q, hist, b);
    sort_scan_kernel<<<1, 1024, 0, stream>>>(hist, p.blocks * kDigits);
    sort_scatter_kernel<<<blocks, kTileThreads, 0, stream>>>(keys_in, pos_in, s.n, 8 * q, hist, b, keys_out, pos_out);
    count_launch(3);
  }
  return cudaGetLastError();
}

template <typename G, typename O, int V>
cudaError_t embed_sum_v(const EmbedGradArgs& a, const EmbedPlan& p, cudaStream_t stream) {
  const int64_t cols = a.hidden / V;
  int x = 32;
  while (x < 256 && x < cols) x *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(x, 256 / x);
  cfg.gridDim = dim3(static_cast<unsigned>((p.chunks + 256 / x - 1) / (256 / x)), static_cast<unsigned>((cols + x - 1) / x));
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  count_launch();
  cudaError_t e = cudaLaunchKernelEx(&cfg, embed_sum_kernel<G, O, V>, a);
  if (e != cudaSuccess || p.chunks == 1) return e;
  cfg.blockDim = dim3(256);
  constexpr int W = V == 1 ? 1 : kVec16<O>;
  const int64_t most = p.chunks * ((a.hidden + 32 * W - 1) / (32 * W));
  cfg.gridDim = dim3(static_cast<unsigned>(most < 148 * 8 ? most : 148 * 8));
  count_launch();
  return cudaLaunchKernelEx(&cfg, embed_join_kernel<O, W>, a);
}

template <typename G, typename O>
cudaError_t embed_grad_t(EmbedGradArgs a, SortArgs s, void* workspace, cudaStream_t stream) {
  const EmbedPlan p = embed_plan(a.n, a.vocab, a.hidden);
  char* ws = static_cast<char*>(workspace);
  uint32_t* scratch = reinterpret_cast<uint32_t*>(ws + p.keys);
  s.keys0 = scratch;
  s.pos0 = scratch + a.n;
  s.keys1 = scratch + 2 * a.n;
  s.pos1 = scratch + 3 * a.n;
  s.heads = a.heads = reinterpret_cast<uint32_t*>(ws + p.heads);
  a.partial = reinterpret_cast<float*>(ws + p.partial);
  a.chunk = static_cast<int32_t>(p.chunk);
  s.passes = p.passes;
  s.bits = p.bits;
  a.keys = (p.passes & 1) ? s.keys0 : s.keys1;
  a.pos = (p.passes & 1) ? s.pos0 : s.pos1;
  cudaError_t e;
  if (p.items == 0) {
    e = sort_tiles(s, p, reinterpret_cast<uint32_t*>(ws + p.hist), stream);
  } else {
    auto fn = p.items == 1 ? sort_kernel<1> : (p.items == 2 ? sort_kernel<2> : (p.items == 4 ? sort_kernel<4> : sort_kernel<8>));
    e = launch_kernel(fn, p.cluster, kSortThreads, p.cluster, false, s, stream);
  }
  if (e == cudaSuccess && !a.accumulate) {
    const ZeroArgs z{a.out, a.vocab, a.hidden * static_cast<int64_t>(sizeof(O)), a.ld_out * static_cast<int64_t>(sizeof(O))};
    const int64_t want = (z.rows * z.row_bytes + 32767) / 32768;  // 4 vectors a thread
    e = launch_kernel(zero_kernel, want < (1 << 20) ? want : (1 << 20), 512, 1, true, z, stream);
  }
  if (e != cudaSuccess) return e;
  constexpr int V = kVec16<G>;
  const uint64_t bits = reinterpret_cast<uintptr_t>(a.grad) | reinterpret_cast<uintptr_t>(a.out) |
                        static_cast<uint64_t>(a.ld_grad) * sizeof(G) | static_cast<uint64_t>(a.ld_out) * sizeof(O) |
                        static_cast<uint64_t>(a.hidden) * sizeof(G);
  if (bits % 16 == 0) return embed_sum_v<G, O, V>(a, p, stream);
  return embed_sum_v<G, O, 1>(a, p, stream);
}

}  // namespace mib
