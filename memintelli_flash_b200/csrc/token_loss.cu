// Token log-probabilities, the clipped policy loss and the paired preference loss over (rows, vocab) logits,
// with the gradient of the logits.  With x = logits / T, target t_r and
//   m_r = max_j logits[r, j],  s_r = sum_j exp(x[r, j] - m_r / T):
//   lp_r = x[r, t_r] - m_r / T - log s_r,     p[r, j] = exp(x[r, j] - m_r / T) / s_r
// and every loss here depends on the logits through lp alone, so
//   d loss / d logits[r, j] = c_r (1{j = t_r} - p[r, j]),   c_r = (d loss / d lp_r) / T.
//
// All are bound by memory: a few operations per 2- or 4-byte logit.  Three steps: row statistics (one read of the
// logits, a long row split over blocks when there are few rows), the losses' per-row coefficients (small), and
// the gradient (a second read, one write).
//
// The maximum starts at the lowest finite float, so a row of -inf, or of the type's lowest value, needs no special
// case: exp(-inf - m) = 0 and exp(lowest - lowest) = 1.  A row of -inf alone gives s = 0 and lp = NaN, as the
// formula does; a NaN or +inf logit makes its row's lp NaN.  Statistics are fp32; lp is formed in double from
// them (the difference lp - ref summed over a sequence would otherwise carry lp's fp32 rounding per token).
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f;

struct RowStat {
  float m, s;
};
__device__ __forceinline__ RowStat merge(RowStat a, RowStat b, float k) {
  const float m = fmaxf(a.m, b.m);
  return RowStat{m, a.s * ex2((a.m - m) * k) + b.s * ex2((b.m - m) * k)};
}

__device__ __forceinline__ RowStat block_merge(RowStat t, float k, RowStat* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    t = merge(t, RowStat{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o)}, k);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = t;
  __syncthreads();
  t = smem[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) t = merge(t, smem[w], k);
  return t;
}

template <int N>
__device__ __forceinline__ void stat_push(RowStat& t, const float (&v)[N], float k) {
  float mx = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) mx = fmaxf(mx, v[i]);
  if (mx > t.m) {
    t.s *= ex2((t.m - mx) * k);
    t.m = mx;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) t.s += ex2((v[i] - t.m) * k);
}

// Elements in front of the first 16-byte boundary of a row at p (all of them when there is none).
template <typename T>
__device__ __forceinline__ int64_t peel(const T* p, int64_t cols) {
  const int64_t h = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
  return h < cols ? h : cols;
}

constexpr int kStatThreads = 256;

// Partial statistics of a row's columns: block b handles part b % splits of row b / splits.  Ignored rows are
// not read.
template <typename T>
__global__ void __launch_bounds__(kStatThreads) row_stat_kernel(const T* __restrict__ logits, RowMap map, int64_t rows,
                                                                int64_t cols, IntList targets, int64_t ignore_index,
                                                                float k, int splits, RowStat* __restrict__ part) {
  __shared__ RowStat smem[kStatThreads / 32];
  const int64_t r = blockIdx.x / splits;
  const int sp = blockIdx.x % splits;
  if (targets[r] == ignore_index) return;
  const T* p = logits + map.at(r);
  const int64_t head = peel(p, cols);
  const int64_t nvec = (cols - head) / kVec16<T>;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  RowStat t{kLowest, 0.0f};
  const int64_t step = static_cast<int64_t>(splits) * kStatThreads;
  for (int64_t i = static_cast<int64_t>(sp) * kStatThreads + threadIdx.x; i < nvec; i += step) {
    float v[kVec16<T>];
    unpack16<T>(__ldg(pv + i), v);
    stat_push(t, v, k);
  }
  if (sp == 0) {
    const int64_t tail = head + nvec * kVec16<T>;
    for (int64_t j = threadIdx.x; j < head; j += kStatThreads) {
      float v[1] = {to_f32(p[j])};
      stat_push(t, v, k);
    }
    for (int64_t j = tail + threadIdx.x; j < cols; j += kStatThreads) {
      float v[1] = {to_f32(p[j])};
      stat_push(t, v, k);
    }
  }
  t = block_merge(t, k, smem);
  if (threadIdx.x == 0) part[blockIdx.x] = t;
}

struct TokenArgs {
  const void* logits;
  RowMap map;
  int64_t rows, cols;
  IntList targets;
  int64_t ignore_index;
  float k;             // log2(e) / T
  double inv_temp;
  int splits;
  const RowStat* part; // [rows][splits]
  float* logps;        // [rows]
  float4* row;         // [rows] {m, 1 / s, c, -}
};

template <typename T>
__device__ __forceinline__ double row_logp(const TokenArgs& a, int64_t r, int64_t t, RowStat& st) {
  st = a.part[r * a.splits];
  for (int i = 1; i < a.splits; ++i) st = merge(st, a.part[r * a.splits + i], a.k);
  if (t < 0 || t >= a.cols) return static_cast<double>(NAN);
  const double x = to_f32(__ldg(static_cast<const T*>(a.logits) + a.map.at(r) + t));
  return (x - static_cast<double>(st.m)) * a.inv_temp - log(static_cast<double>(st.s));
}

template <typename T>
__global__ void token_logps_kernel(TokenArgs a) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (r >= a.rows) return;
  const int64_t t = a.targets[r];
  RowStat st;
  const bool live = t != a.ignore_index;
  a.logps[r] = live ? static_cast<float>(row_logp<T>(a, r, t, st)) : 0.0f;
  if (a.row) a.row[r] = live ? make_float4(st.m, 1.0f / st.s, 0.0f, 0.0f) : make_float4(0.0f, 1.0f, 0.0f, 0.0f);
}

// Sequence s holds rows [cu[s], cu[s + 1]); both ends are held to [0, rows] whatever the list says.
struct SeqList {
  IntList cu;
  int64_t count;  // sequences; 0: no list
  int64_t uniform;  // > 0: no list, every sequence holds this many rows
  __device__ __forceinline__ int64_t begin(int64_t s, int64_t rows) const {
    const int64_t v = uniform > 0 ? s * uniform : cu[s];
    return v < 0 ? 0 : (v > rows ? rows : v);
  }
  // The sequence of row r, or -1: the last s with cu[s] <= r, if r < cu[s + 1].
  __device__ __forceinline__ int64_t of(int64_t r) const {
    if (uniform > 0) return r / uniform < count ? r / uniform : -1;
    int64_t lo = 0, hi = count;  // cu[lo] <= r < cu[hi], were the list's ends -inf and +inf
    if (cu[0] > r || cu[count] <= r) return -1;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (cu[mid] <= r) lo = mid; else hi = mid;
    }
    return lo;
  }
};

// ---- policy loss -----------------------------------------------------------------------------------
struct PolicyArgs {
  TokenArgs t;
  SeqList seq;
  const float *old_logps, *advantages, *ref_logps;
  int32_t adv_per_seq, reduction;  // reduction: 0 token mean, 1 mean over sequences of their token means, 2 sum
  float lo, hi, kl_coef;           // ratio bounds
  int32_t count_blocks;
  int32_t* counts;                 // [count_blocks] counted tokens (token mean) or non-empty sequences
  float* seq_w;                    // [sequences] 1 / counted tokens of the sequence (sequence mean)
  uint32_t* done;
  double* sums;                    // [blocks][3]
  float* out;                      // loss, kl, clip fraction
};

constexpr int kCountBlocks = 64;

// Counted tokens: all (token mean), or per sequence with the number of non-empty ones (sequence mean).
__global__ void __launch_bounds__(256) policy_count_kernel(PolicyArgs a) {
  __shared__ int smem[8];
  const int64_t rows = a.t.rows;
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.done = 0;
  int n = 0;
  if (a.reduction == 0) {
    int64_t lo = 0, hi = rows;
    if (a.seq.count > 0) {
      lo = a.seq.begin(0, rows);
      hi = a.seq.begin(a.seq.count, rows);
    }
    for (int64_t r = lo + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; r < hi; r += gridDim.x * 256)
      n += a.t.targets[r] != a.t.ignore_index;
  } else if (a.reduction == 1) {
    const int lane = threadIdx.x & 31;
    for (int64_t s = blockIdx.x * 8 + (threadIdx.x >> 5); s < a.seq.count; s += gridDim.x * 8) {
      const int64_t lo = a.seq.begin(s, rows), hi = a.seq.begin(s + 1, rows);
      int c = 0;
      for (int64_t r = lo + lane; r < hi; r += 32) c += a.t.targets[r] != a.t.ignore_index;
      c = __reduce_add_sync(0xffffffffu, c);
      if (lane == 0) {
        a.seq_w[s] = c > 0 ? 1.0f / static_cast<float>(c) : 0.0f;
        n += c > 0;
      }
    }
  }
  n = block_sum(n, smem);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

struct PolicyTerm {
  double loss, kl, clipped;
  float c;
};

// One token's terms, weighted by w.  kl = e^d - d - 1 with d = ref - lp (its estimate from one sample, >= 0).
__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& a, int64_t r, int64_t seq, double lp, double w) {
  const double adv = __ldg(a.advantages + (a.adv_per_seq ? seq : r));
  const double ratio = exp(lp - static_cast<double>(__ldg(a.old_logps + r)));
  const double held = fmin(fmax(ratio, static_cast<double>(a.lo)), static_cast<double>(a.hi));
  const double gain = ratio * adv, gain_held = held * adv;
  const bool clipped = gain_held < gain;
  PolicyTerm o{-(clipped ? gain_held : gain), 0.0, clipped ? w : 0.0, 0.0f};
  double slope = clipped ? 0.0 : -gain;
  if (a.ref_logps) {
    const double d = static_cast<double>(__ldg(a.ref_logps + r)) - lp, e = exp(d);
    const double kl = e - d - 1.0;
    o.kl = w * kl;
    if (a.kl_coef != 0.0f) {
      o.loss += a.kl_coef * kl;
      slope += a.kl_coef * (1.0 - e);
    }
  }
  o.loss *= w;
  o.c = static_cast<float>(w * slope * a.t.inv_temp);
  return o;
}

template <typename T>
__global__ void __launch_bounds__(256) policy_row_kernel(PolicyArgs a) {
  __shared__ double smem[8];
  __shared__ int ismem[8];
  double scale = 1.0;
  if (a.reduction != 2) {
    const int n = block_sum(threadIdx.x < a.count_blocks ? a.counts[threadIdx.x] : 0, ismem);
    scale = n > 0 ? 1.0 / n : 0.0;
  }
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  PolicyTerm o{0.0, 0.0, 0.0, 0.0f};
  if (r < a.t.rows) {
    const int64_t t = a.t.targets[r];
    const int64_t s = a.seq.count > 0 ? a.seq.of(r) : 0;
    RowStat st{0.0f, 1.0f};
    double lp = 0.0;
    if (t != a.t.ignore_index) {
      lp = row_logp<T>(a.t, r, t, st);
      if (s >= 0) o = policy_term(a, r, s, lp, a.reduction == 1 ? scale * a.seq_w[s] : scale);
    }
    a.t.logps[r] = static_cast<float>(lp);
    if (a.t.row) a.t.row[r] = make_float4(st.m, 1.0f / st.s, o.c, 0.0f);
  }
  const double v[3] = {block_sum(o.loss, smem), block_sum(o.kl, smem), block_sum(o.clipped, smem)};
  if (threadIdx.x < 3) a.sums[blockIdx.x * 3 + threadIdx.x] = v[threadIdx.x];
  if (last_block(a.done, gridDim.x)) {
    for (int q = 0; q < 3; ++q) {
      double x = 0.0;
      for (int64_t b = threadIdx.x; b < gridDim.x; b += 256) x += __ldcg(a.sums + b * 3 + q);
      x = block_sum(x, smem);
      if (threadIdx.x == 0) a.out[q] = static_cast<float>(x);
    }
  }
}

// ---- preference loss -------------------------------------------------------------------------------
struct PreferenceArgs {
  TokenArgs t;
  SeqList seq;               // pairs: sequence i against sequence i + count / 2
  const float* ref_logps;
  int32_t kind, average;     // kind: 0 sigmoid, 1 hinge, 2 squared
  double beta, smoothing, margin;
  uint32_t* done;
  double* sums;              // [pairs]
  float *chosen, *rejected;  // [pairs]
  float* out;                // loss
};

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// loss and its slope over h = beta (D_chosen - D_rejected) - margin
__device__ __forceinline__ void preference_term(const PreferenceArgs& a, double h, double& loss, double& slope) {
  const double e = a.smoothing;
  if (a.kind == 0) {
    loss = (1.0 - e) * softplus(-h) + e * softplus(h);
    slope = e / (1.0 + exp(-h)) - (1.0 - e) / (1.0 + exp(h));
  } else if (a.kind == 1) {
    loss = isnan(h) ? h : fmax(1.0 - h, 0.0);
    slope = h < 1.0 ? -1.0 : (isnan(h) ? h : 0.0);
  } else {
    loss = (h - 0.5) * (h - 0.5);
    slope = 2.0 * (h - 0.5);
  }
}

__global__ void preference_zero_kernel(PreferenceArgs a) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (r == 0) *a.done = 0;
  if (r < a.t.rows) {
    a.t.logps[r] = 0.0f;
    if (a.t.row) a.t.row[r] = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
  }
}

// One block per pair.
template <typename T>
__global__ void __launch_bounds__(256) preference_pair_kernel(PreferenceArgs a) {
  __shared__ double smem[8];
  const int64_t pairs = a.seq.count / 2, i = blockIdx.x;
  double d[2], n[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t s = i + side * pairs;
    const int64_t lo = a.seq.begin(s, a.t.rows), hi = a.seq.begin(s + 1, a.t.rows);
    double x = 0.0, c = 0.0;
    for (int64_t r = lo + threadIdx.x; r < hi; r += 256) {
      const int64_t t = a.t.targets[r];
      if (t == a.t.ignore_index) continue;
      RowStat st;
      const double lp = row_logp<T>(a.t, r, t, st);
      a.t.logps[r] = static_cast<float>(lp);
      x += lp - (a.ref_logps ? static_cast<double>(__ldg(a.ref_logps + r)) : 0.0);
      c += 1.0;
      if (a.t.row) a.t.row[r] = make_float4(st.m, 1.0f / st.s, 0.0f, 0.0f);
    }
    d[side] = block_sum(x, smem);
    n[side] = block_sum(c, smem);
    if (a.average) d[side] = n[side] > 0.0 ? d[side] / n[side] : 0.0;
  }
  double loss, slope;
  preference_term(a, a.beta * (d[0] - d[1]) - a.margin, loss, slope);
  if (threadIdx.x == 0) {
    a.chosen[i] = static_cast<float>(a.beta * d[0]);
    a.rejected[i] = static_cast<float>(a.beta * d[1]);
    a.sums[i] = loss;
  }
  if (a.t.row) {
    for (int side = 0; side < 2; ++side) {
      const int64_t s = i + side * pairs;
      const int64_t lo = a.seq.begin(s, a.t.rows), hi = a.seq.begin(s + 1, a.t.rows);
      double c = slope * a.beta * a.t.inv_temp / static_cast<double>(pairs);
      if (a.average && n[side] > 0.0) c /= n[side];
      for (int64_t r = lo + threadIdx.x; r < hi; r += 256)
        if (a.t.targets[r] != a.t.ignore_index) a.t.row[r].z = static_cast<float>(side ? -c : c);
    }
  }
  if (last_block(a.done, gridDim.x)) {
    double x = 0.0;
    for (int64_t b = threadIdx.x; b < gridDim.x; b += 256) x += __ldcg(a.sums + b);
    x = block_sum(x, smem);
    if (threadIdx.x == 0) *a.out = static_cast<float>(x / static_cast<double>(pairs));
  }
}

// ---- gradient of the logits ------------------------------------------------------------------------
// One block per row; the coefficient is row[r].z, or slope[r] / T where slopes are given.  A row whose coefficient is zero (ignored, clipped without a KL term) is written as zeros and
// not read: what its logits hold, NaN and infinities included, does not reach the gradient.  `grad` may be the
// logits themselves: each element is read and written by one thread, the target's in front of the rest.
template <typename T>
__global__ void __launch_bounds__(256) logit_grad_kernel(const T* logits, RowMap map, int64_t cols, IntList targets,
                                                         float k, const float4* __restrict__ row,
                                                         const float* __restrict__ slope, float inv_temp,
                                                         int64_t ignore_index, T* grad, RowMap gmap) {
  const int64_t r = blockIdx.x;
  float4 st = row[r];
  if (slope) st.z = targets[r] == ignore_index ? 0.0f : slope[r] * inv_temp;
  const T* p = logits + map.at(r);
  T* g = grad + gmap.at(r);
  const float c = st.z, q = -st.z * st.y;
  const bool zero = c == 0.0f;
  const int64_t t = zero ? -1 : targets[r];
  float at_t = 0.0f;
  if (!zero && t >= 0 && t < cols) at_t = c + q * ex2((to_f32(p[t]) - st.x) * k);
  __syncthreads();
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  const int64_t head = same ? peel(g, cols) : cols;
  const int64_t nvec = (cols - head) / kVec16<T>;
  const int64_t tail = head + nvec * kVec16<T>;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  uint4* gv = reinterpret_cast<uint4*>(g + head);
  const int64_t tv = t >= head && t < tail ? (t - head) / kVec16<T> : -1;
  for (int64_t i = threadIdx.x; i < nvec; i += 256) {
    float v[kVec16<T>];
    if (zero) {
#pragma unroll
      for (int e = 0; e < kVec16<T>; ++e) v[e] = 0.0f;
    } else {
      unpack16<T>(pv[i], v);
#pragma unroll
      for (int e = 0; e < kVec16<T>; ++e) v[e] = q * ex2((v[e] - st.x) * k);
      if (i == tv) {
#pragma unroll
        for (int e = 0; e < kVec16<T>; ++e)
          if (head + i * kVec16<T> + e == t) v[e] = at_t;
      }
    }
    gv[i] = pack16<T>(v);
  }
  for (int64_t j = threadIdx.x; j < cols; j += 256) {
    if (j >= head && j < tail) {
      j += (tail - j - 1) / 256 * 256;
      continue;
    }
    const float v = zero ? 0.0f : (j == t ? at_t : q * ex2((to_f32(p[j]) - st.x) * k));
    g[j] = from_f32<T>(v);
  }
}

// x *= *factor over n elements; a factor of exactly 1 leaves the buffer untouched.
template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* x, int64_t n, const float* __restrict__ factor) {
  const float f = __ldg(factor);
  if (f == 1.0f) return;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += gridDim.x * 256ll)
    x[i] = from_f32<T>(to_f32(x[i]) * f);
}

// ---- launchers -------------------------------------------------------------------------------------
// Parts a row is cut into: 1 with rows enough for every SM, else as many as keep 4 blocks per SM busy with at
// least 4096 elements each.
int row_splits(int64_t rows, int64_t cols) {
  const int64_t want = (4 * 148 + rows - 1) / rows, most = (cols + 4095) / 4096;
  return static_cast<int>(want < most ? want : most);
}

template <typename T>
cudaError_t row_stats_t(const TokenArgs& a, RowStat* part, cudaStream_t stream) {
  row_stat_kernel<T><<<static_cast<unsigned>(a.rows * a.splits), kStatThreads, 0, stream>>>(
      static_cast<const T*>(a.logits), a.map, a.rows, a.cols, a.targets, a.ignore_index, a.k, a.splits, part);
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t logit_grad_t(const TokenArgs& a, const float* slope, void* grad, RowMap gmap, cudaStream_t stream) {
  logit_grad_kernel<T><<<static_cast<unsigned>(a.rows), 256, 0, stream>>>(
      static_cast<const T*>(a.logits), a.map, a.cols, a.targets, a.k, a.row, slope, static_cast<float>(a.inv_temp),
      a.ignore_index, static_cast<T*>(grad), gmap);
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t token_logps_t(const TokenArgs& a, RowStat* part, cudaStream_t stream) {
  cudaError_t e = row_stats_t<T>(a, part, stream);
  if (e != cudaSuccess) return e;
  token_logps_kernel<T><<<static_cast<unsigned>((a.rows + 255) / 256), 256, 0, stream>>>(a);
  count_launch();
  return cudaGetLastError();
}

template <typename T>
cudaError_t policy_loss_t(const PolicyArgs& a, RowStat* part, void* grad, RowMap gmap, cudaStream_t stream) {
  policy_count_kernel<<<a.count_blocks, 256, 0, stream>>>(a);
  count_launch();
  cudaError_t e = row_stats_t<T>(a.t, part, stream);
  if (e != cudaSuccess) return e;
  policy_row_kernel<T><<<static_cast<unsigned>((a.t.rows + 255) / 256), 256, 0, stream>>>(a);
  count_launch();
  e = cudaGetLastError();
  if (e != cudaSuccess || !grad) return e;
  return logit_grad_t<T>(a.t, nullptr, grad, gmap, stream);
}

template <typename T>
cudaError_t preference_loss_t(const PreferenceArgs& a, RowStat* part, void* grad, RowMap gmap, cudaStream_t stream) {
  preference_zero_kernel<<<static_cast<unsigned>((a.t.rows + 255) / 256), 256, 0, stream>>>(a);
  count_launch();
  cudaError_t e = row_stats_t<T>(a.t, part, stream);
  if (e != cudaSuccess) return e;
  preference_pair_kernel<T><<<static_cast<unsigned>(a.seq.count / 2), 256, 0, stream>>>(a);
  count_launch();
  e = cudaGetLastError();
  if (e != cudaSuccess || !grad) return e;
  return logit_grad_t<T>(a.t, nullptr, grad, gmap, stream);
}

template <typename T>
cudaError_t scale_by_t(void* x, int64_t n, const float* factor, cudaStream_t stream) {
  int64_t blocks = (n + 1023) / 1024;
  if (blocks > 148 * 8) blocks = 148 * 8;
  scale_by_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(static_cast<T*>(x), n, factor);
  count_launch();
  return cudaGetLastError();
}

}  // namespace mib
