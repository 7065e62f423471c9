// Shared helpers of the language-model tuning operators (embedding, token losses, gradient clipping):
// element types, 16-byte vectors of them, and row addressing.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>

namespace mib {

// ---- element types ---------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T>
constexpr int kVec16 = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte vector

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float (&v)[kVec16<T>]) {
  if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&v)[kVec16<T>]) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// 2^x (hardware, flushes subnormal results to zero; 2 ulp).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- row addressing: row r of a block starts at (r / per_group) * group_stride + (r % per_group) * row_stride --
struct RowMap {
  int64_t per_group, group_stride, row_stride;
  __host__ __device__ __forceinline__ int64_t at(int64_t r) const {
    if (r < per_group) return r * row_stride;
    const int64_t g = r / per_group;
    return g * group_stride + (r - g * per_group) * row_stride;
  }
};

// Token or sequence indices, 32 or 64 bits wide.
struct IntList {
  const void* p;
  int32_t is64;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return is64 ? __ldg(static_cast<const long long*>(p) + i) : __ldg(static_cast<const int*>(p) + i);
  }
};

// Sum over a block in a fixed order (warp trees, then the warps in turn); every thread gets it.
template <typename V>
__device__ __forceinline__ V block_sum(V v, V* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[warp] = v;
  __syncthreads();
  V t = smem[0];
  for (int w = 1; w < nw; ++w) t += smem[w];
  return t;
}

// True in every thread of the block that is the last of `total` to arrive at `counter` (zero before the launch).
__device__ __forceinline__ bool last_block(uint32_t* counter, uint32_t total) {
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(counter, 1u) == total - 1;
  __syncthreads();
  if (last) __threadfence();
  return last;
}

}  // namespace mib
