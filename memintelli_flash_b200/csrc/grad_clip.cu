// Global norm of a list of gradients, and clipping:
//   norm = (sum over all tensors of |g|^p)^(1/p), p = 1, 2 or infinity;   g <- g * min(1, max_norm / (norm + eps))
// The tensors' addresses travel as kernel arguments (no table in device memory to fill), up to kClipTensors per
// launch.  Both passes walk fixed-size chunks; the norm's partial sums are added in a fixed order.
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

constexpr int kClipTensors = 512;
constexpr int64_t kClipChunk = 8192;  // elements

struct ClipTable {
  int32_t count;
  const void* in[kClipTensors];
  void* out[kClipTensors];
  int64_t numel[kClipTensors];
  int32_t first[kClipTensors + 1];  // first chunk of each tensor
  uint8_t in_type[kClipTensors], out_type[kClipTensors];
};
static_assert(sizeof(ClipTable) <= 32000, "kernel parameters");

__device__ __forceinline__ int clip_find(const ClipTable& t, int32_t chunk) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// One value into the running sum: |g|, g^2, or the maximum of |g| (a NaN stays).
template <int P>
__device__ __forceinline__ float norm_add(float acc, float g) {
  if (P == 2) return fmaf(g, g, acc);
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
__device__ __forceinline__ float norm_chunk(const T* p, int64_t n) {
  float acc = 0.0f;
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
  float* coef;        // out
};

// Blocks stride over the chunks; part[b] is the block's sum.
template <int P>
__global__ void __launch_bounds__(256) clip_norm_kernel(const __grid_constant__ ClipTable t, ClipState s) {
  __shared__ double smem[8];
  double acc = 0.0;
  for (int32_t c = blockIdx.x; c < t.first[t.count]; c += gridDim.x) {
    const int k = clip_find(t, c);
    const int64_t at = static_cast<int64_t>(c - t.first[k]) * kClipChunk;
    const int64_t n = t.numel[k] - at < kClipChunk ? t.numel[k] - at : kClipChunk;
    float v;
    if (t.in_type[k] == MIB_F32) v = norm_chunk<P>(static_cast<const float*>(t.in[k]) + at, n);
    else if (t.in_type[k] == MIB_BF16) v = norm_chunk<P>(static_cast<const __nv_bfloat16*>(t.in[k]) + at, n);
    else v = norm_chunk<P>(static_cast<const __half*>(t.in[k]) + at, n);
    acc = norm_join<P>(acc, static_cast<double>(v));
  }
  acc = block_join<P>(acc, smem);
  if (threadIdx.x == 0) s.part[s.part_first + blockIdx.x] = acc;
}

template <int P>
__global__ void __launch_bounds__(256) clip_finish_kernel(ClipState s) {
  __shared__ double smem[8];
  double acc = 0.0;
  for (int b = threadIdx.x; b < s.part_total; b += 256) acc = norm_join<P>(acc, s.part[b]);
  acc = block_join<P>(acc, smem);
  if (threadIdx.x == 0) {
    const float norm = static_cast<float>(P == 2 ? sqrt(acc) : acc);
    *s.norm = norm;
    if (s.coef) {
      const float c = s.max_norm / (norm + s.eps);
      *s.coef = c > 1.0f ? 1.0f : c;  // a NaN norm gives NaN gradients
    }
  }
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
__global__ void __launch_bounds__(256) clip_scale_kernel(const __grid_constant__ ClipTable t, const float* coef,
                                                         int in_place) {
  const float c = *coef;
  if (in_place && c == 1.0f) return;
  for (int32_t b = blockIdx.x; b < t.first[t.count]; b += gridDim.x) {
    const int k = clip_find(t, b);
    const int64_t at = static_cast<int64_t>(b - t.first[k]) * kClipChunk;
    const int64_t n = t.numel[k] - at < kClipChunk ? t.numel[k] - at : kClipChunk;
    if (t.in_type[k] == MIB_F32) scale_to(static_cast<const float*>(t.in[k]), t.out[k], t.out_type[k], at, n, c);
    else if (t.in_type[k] == MIB_BF16)
      scale_to(static_cast<const __nv_bfloat16*>(t.in[k]), t.out[k], t.out_type[k], at, n, c);
    else scale_to(static_cast<const __half*>(t.in[k]), t.out[k], t.out_type[k], at, n, c);
  }
}

constexpr int kClipBlocks = 148 * 8;

inline unsigned clip_grid(const ClipTable& t) {
  const int32_t chunks = t.first[t.count];
  return static_cast<unsigned>(chunks < kClipBlocks ? chunks : kClipBlocks);
}

template <int P>
cudaError_t clip_norm_p(const ClipTable& t, const ClipState& s, cudaStream_t stream) {
  clip_norm_kernel<P><<<clip_grid(t), 256, 0, stream>>>(t, s);
  count_launch();
  return cudaGetLastError();
}

template <int P>
cudaError_t clip_finish_p(const ClipState& s, cudaStream_t stream) {
  clip_finish_kernel<P><<<1, 256, 0, stream>>>(s);
  count_launch();
  return cudaGetLastError();
}

cudaError_t clip_scale(const ClipTable& t, const float* coef, bool in_place, cudaStream_t stream) {
  clip_scale_kernel<<<clip_grid(t), 256, 0, stream>>>(t, coef, in_place ? 1 : 0);
  count_launch();
  return cudaGetLastError();
}

}  // namespace mib
