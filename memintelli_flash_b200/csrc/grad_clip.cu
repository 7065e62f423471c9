// Global norm of a list of gradients, and clipping:
//   norm = (sum over all tensors of |g|^p)^(1/p), p = 1, 2 or infinity;   g <- g * min(1, max_norm / (norm + eps))
// The tensors' addresses travel as kernel arguments (no table in device memory to fill), up to kClipTensors per
// launch.  Both passes walk fixed-size chunks; the norm's partial sums, one per block, are added in a fixed order, by
// every block of the second pass for itself (at most 9.5 KB from L2, and one launch less).  The second pass walks the
// chunks backwards: what the first read last is still in L2.  Both are bound by memory: 3 GB of fp32 gradients are read
// at 6.8 TB/s (440 us), then scaled at 6.3 TB/s (957 us).
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

constexpr int kClipTensors = 512, kClipFew = 32;  // a short list has a kernel with less to pass
constexpr int64_t kClipChunk = 8192;  // elements

template <int N>
struct ClipList {
  int32_t count;
  const void* in[N];
  void* out[N];
  int64_t numel[N];
  int32_t first[N + 1];  // first chunk of each tensor
  uint8_t in_type[N], out_type[N];
};
using ClipTable = ClipList<kClipTensors>;
static_assert(sizeof(ClipTable) <= 32000, "kernel parameters");

inline ClipList<kClipFew> clip_few(const ClipTable& t) {
  ClipList<kClipFew> f;
  f.count = t.count;
  f.first[0] = 0;
  for (int i = 0; i < t.count; ++i) {
    f.in[i] = t.in[i];
    f.out[i] = t.out[i];
    f.numel[i] = t.numel[i];
    f.first[i + 1] = t.first[i + 1];
    f.in_type[i] = t.in_type[i];
    f.out_type[i] = t.out_type[i];
  }
  return f;
}

template <int N>
__device__ __forceinline__ int clip_find(const ClipList<N>& t, int32_t chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// One value into the running sum: |g|, g^2, or the maximum of |g| (a NaN stays).  Squares of fp32 and bf16 gradients are
// added in double: beyond 2^64 or below 2^-63 they have no fp32 value.  (800 M elements: fp32 norm 460 -> 470 us, bf16 235
// -> 264 us; clipping, whose second pass is the longer one, 1503 -> 1524 and 786 -> 787 us.)
template <int P, typename T>
using NormSum = typename std::conditional<P == 2 && !std::is_same<T, __half>::value, double, float>::type;
template <int P, typename S>
__device__ __forceinline__ S norm_add(S acc, float g) {
  if (P == 2) return fma(static_cast<S>(g), static_cast<S>(g), acc);
  if (P == 1) return acc + fabsf(g);
  const float x = fabsf(g);
  return (x > acc || isnan(x)) ? x : acc;
}

template <int P>
__device__ __forceinline__ double norm_join(double a, double b) {
  if (P != 0) return a + b;
  return (b > a || isnan(b)) ? b : a;
}

template <int P>
__device__ __forceinline__ double block_join(double v, double* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = norm_join<P>(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) v = norm_join<P>(v, smem[w]);
  return v;
}

template <int P, typename T>
__device__ __forceinline__ NormSum<P, T> norm_chunk(const T* p, int64_t n) {
  NormSum<P, T> acc = 0;
  const int64_t head0 = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
  const int64_t head = head0 < n ? head0 : n;
  const int64_t nvec = (n - head) / kVec16<T>;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  for (int64_t i = threadIdx.x; i < nvec; i += 256) {
    float v[kVec16<T>];
    unpack16<T>(__ldg(pv + i), v);
#pragma unroll
    for (int e = 0; e < kVec16<T>; ++e) acc = norm_add<P>(acc, v[e]);
  }
  if (threadIdx.x < head) acc = norm_add<P>(acc, to_f32(p[threadIdx.x]));
  const int64_t j = head + nvec * kVec16<T> + threadIdx.x;
  if (j < n) acc = norm_add<P>(acc, to_f32(p[j]));
  return acc;
}

struct ClipState {
  double* part;       // one per block of every launch of the pass
  int32_t part_first, part_total;
  float max_norm, eps;
  float* norm;        // out
};

// Blocks stride over the chunks; part[b] is the block's sum.
template <int P, int N>
__global__ void __launch_bounds__(256) clip_norm_kernel(const __grid_constant__ ClipList<N> t, ClipState s) {
  __shared__ double smem[8];
  pdl_release();
  double acc = 0.0;
  for (int32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = clip_find(t, c);
    const int64_t at = static_cast<int64_t>(c - t.first[k]) * kClipChunk;
    const int64_t n = t.numel[k] - at < kClipChunk ? t.numel[k] - at : kClipChunk;
    double v;
    if (t.in_type[k] == MIB_F32) v = norm_chunk<P>(static_cast<const float*>(t.in[k]) + at, n);
    else if (t.in_type[k] == MIB_BF16) v = norm_chunk<P>(static_cast<const __nv_bfloat16*>(t.in[k]) + at, n);
    else v = norm_chunk<P>(static_cast<const __half*>(t.in[k]) + at, n);
    acc = norm_join<P>(acc, v);
  }
  acc = block_join<P>(acc, smem);
  if (threadIdx.x == 0) s.part[s.part_first + blockIdx.x] = acc;
}

// The norm from the blocks' sums; every thread gets it.
template <int P>
__device__ __forceinline__ float clip_total(const ClipState& s, double* smem) {
  double acc = 0.0;
  for (int b = threadIdx.x; b < s.part_total; b += 256) acc = norm_join<P>(acc, __ldcg(s.part + b));
  acc = block_join<P>(acc, smem);
  return static_cast<float>(P == 2 ? sqrt(acc) : acc);
}

template <int P>
__global__ void __launch_bounds__(256) clip_finish_kernel(ClipState s) {
  __shared__ double smem[8];
  pdl_wait();
  const float norm = clip_total<P>(s, smem);
  if (threadIdx.x == 0) *s.norm = norm;
}

template <typename I, typename O>
__device__ __forceinline__ void scale_chunk(const I* p, O* o, int64_t n, float c) {
  constexpr int V = kVec16<I>;
  if constexpr (sizeof(I) == sizeof(O)) {
    if (((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
      const int64_t head0 = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(I);
      const int64_t head = head0 < n ? head0 : n;
      const int64_t nvec = (n - head) / V;
      for (int64_t i = threadIdx.x; i < nvec; i += 256) {
        float v[V];
        unpack16<I>(reinterpret_cast<const uint4*>(p + head)[i], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= c;
        reinterpret_cast<uint4*>(o + head)[i] = pack16<O>(v);
      }
      if (threadIdx.x < head) o[threadIdx.x] = from_f32<O>(to_f32(p[threadIdx.x]) * c);
      const int64_t j = head + nvec * V + threadIdx.x;
      if (j < n) o[j] = from_f32<O>(to_f32(p[j]) * c);
      return;
    }
  }
  for (int64_t i = threadIdx.x; i < n; i += 256) o[i] = from_f32<O>(to_f32(p[i]) * c);
}

template <typename I>
__device__ __forceinline__ void scale_to(const I* p, void* out, int type, int64_t at, int64_t n, float c) {
  if (type == MIB_F32) scale_chunk(p + at, static_cast<float*>(out) + at, n, c);
  else if (type == MIB_BF16) scale_chunk(p + at, static_cast<__nv_bfloat16*>(out) + at, n, c);
  else scale_chunk(p + at, static_cast<__half*>(out) + at, n, c);
}

// In place, a coefficient of exactly 1 leaves the gradients as they are.
template <int P, int N>
__global__ void __launch_bounds__(256) clip_scale_kernel(const __grid_constant__ ClipList<N> t, ClipState s, int in_place) {
  __shared__ double smem[8];
  pdl_release();
  pdl_wait();
  const float norm = clip_total<P>(s, smem);
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.norm = norm;
  const float k = s.max_norm / (norm + s.eps), c = k > 1.0f ? 1.0f : k;  // a NaN norm gives NaN gradients
  if (in_place && c == 1.0f) return;
  const int32_t chunks = t.first[t.count];
  for (int32_t i = blockIdx.x; i < chunks; i += gridDim.x) {
    const int32_t b = chunks - 1 - i;
    const int q = clip_find(t, b);
    const int64_t at = static_cast<int64_t>(b - t.first[q]) * kClipChunk;
    const int64_t n = t.numel[q] - at < kClipChunk ? t.numel[q] - at : kClipChunk;
    if (t.in_type[q] == MIB_F32) scale_to(static_cast<const float*>(t.in[q]), t.out[q], t.out_type[q], at, n, c);
    else if (t.in_type[q] == MIB_BF16)
      scale_to(static_cast<const __nv_bfloat16*>(t.in[q]), t.out[q], t.out_type[q], at, n, c);
    else scale_to(static_cast<const __half*>(t.in[q]), t.out[q], t.out_type[q], at, n, c);
  }
}

constexpr int kClipBlocks = 148 * 8;

inline unsigned clip_grid(const ClipTable& t) {
  const int32_t chunks = t.first[t.count];
  return static_cast<unsigned>(chunks < kClipBlocks ? chunks : kClipBlocks);
}

// `early`: the launch in front belongs to this call, and the kernel waits for it where it needs its results.
template <typename... Args, typename... Given>
cudaError_t clip_launch(void (*fn)(Args...), unsigned blocks, bool early, cudaStream_t stream, const Given&... given) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  count_launch();
  return cudaLaunchKernelEx(&cfg, fn, given...);
}

template <int P>
cudaError_t clip_norm_p(const ClipTable& t, const ClipState& s, cudaStream_t stream) {
  if (t.count <= kClipFew) return clip_launch(clip_norm_kernel<P, kClipFew>, clip_grid(t), false, stream, clip_few(t), s);
  return clip_launch(clip_norm_kernel<P, kClipTensors>, clip_grid(t), false, stream, t, s);
}

template <int P>
cudaError_t clip_finish_p(const ClipState& s, cudaStream_t stream) {
  return clip_launch(clip_finish_kernel<P>, 1, s.part_total > 0, stream, s);
}

template <int P>
cudaError_t clip_scale_p(const ClipTable& t, const ClipState& s, bool in_place, bool early, cudaStream_t stream) {
  const int keep = in_place ? 1 : 0;
  if (t.count <= kClipFew)
    return clip_launch(clip_scale_kernel<P, kClipFew>, clip_grid(t), early, stream, clip_few(t), s, keep);
  return clip_launch(clip_scale_kernel<P, kClipTensors>, clip_grid(t), early, stream, t, s, keep);
}

// A tensor list as kernel tables, `use` called with each (the same tables for both passes).
template <typename F>
int clip_tables(const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
                const int32_t* out_dtype, int32_t count, F use) {
  ClipTable t;
  int32_t i = 0;
  while (i < count) {
    t.count = 0;
    t.first[0] = 0;
    for (; i < count && t.count < kClipTensors; ++i) {
      if (numel[i] == 0) continue;
      const int64_t chunks = (numel[i] + kClipChunk - 1) / kClipChunk;
      if (t.first[t.count] + chunks > (int64_t(1) << 30)) break;
      const int k = t.count++;
      t.in[k] = in[i];
      t.out[k] = out ? out[i] : nullptr;
      t.numel[k] = numel[i];
      t.in_type[k] = static_cast<uint8_t>(in_dtype[i]);
      t.out_type[k] = static_cast<uint8_t>(out ? out_dtype[i] : 0);
      t.first[k + 1] = t.first[k] + static_cast<int32_t>(chunks);
    }
    if (t.count == 0) break;
    if (const int rc = use(t)) return rc;
  }
  return MIB_OK;
}

}  // namespace mib
