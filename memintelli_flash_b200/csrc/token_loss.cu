// Token log-probabilities, the clipped policy loss and the paired preference loss over (rows, vocab) logits,
// with the gradient of the logits.  With x = logits / T, target t_r and
//   m_r = max_j logits[r, j],  s_r = sum_j exp(x[r, j] - m_r / T):
//   lp_r = x[r, t_r] - m_r / T - log s_r,     p[r, j] = exp(x[r, j] - m_r / T) / s_r
// and every loss here depends on the logits through lp alone, so
//   d loss / d logits[r, j] = c_r (1{j = t_r} - p[r, j]),   c_r = (d loss / d lp_r) / T.
//
// All are bound by memory: a few operations per 2- or 4-byte logit.  The policy loss's coefficient belongs to one row,
// so its row is loaded once, held in registers, and written as gradient; the preference loss's needs all rows of two
// sequences, so its gradient reads the logits a second time.
//
// The maximum starts at the lowest finite float, so a row of -inf, or of the type's lowest value, needs no special
// case: exp(-inf - m) = 0 and exp(lowest - lowest) = 1.  A row of -inf alone gives s = 0 and lp = NaN, as the
// formula does; a NaN or +inf logit makes its row's lp NaN.  Statistics are fp32; lp is formed in double from
// them (the difference lp - ref summed over a sequence would otherwise carry lp's fp32 rounding per token).
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

constexpr float kLowest = -3.402823466e38f;

struct RowStat {
  float m, s;
};
__device__ __forceinline__ RowStat merge(RowStat a, RowStat b, float k) {
  const float m = fmaxf(a.m, b.m);
  return RowStat{m, a.s * ex2((a.m - m) * k) + b.s * ex2((b.m - m) * k)};
}

// Elements in front of the first 16-byte boundary of a row at p (all of them when there is none).
template <typename T>
__device__ __forceinline__ int64_t peel(const T* p, int64_t cols) {
  const int64_t h = static_cast<int64_t>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T);
  return h < cols ? h : cols;
}

// A 16-byte load that leaves no line in L1 (each logit is read once per pass).  Not the read-only path: the gradient
// may overwrite the logits.
__device__ __forceinline__ uint4 load_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Two -inf of a 16-bit type, or one fp32 -inf.
template <typename T>
__device__ __forceinline__ uint32_t neg_inf_word() {
  return sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u);
}

template <typename T>
__device__ __forceinline__ float vec_max(const uint4& u, float m) {
  if constexpr (sizeof(T) == 4) {
    float v[4];
    unpack16<T>(u, v);
    return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), m);
  } else {
    using T2 = typename std::conditional<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>::type;
    const T2* w = reinterpret_cast<const T2*>(&u);
    const T2 x = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
    return fmaxf(fmaxf(to_f32(x.x), to_f32(x.y)), m);
  }
}

// sum of 2^((v - m) k) over a vector, as a tree.
template <typename T>
__device__ __forceinline__ float vec_sum(const uint4& u, float m, float k) {
  float v[kVec16<T>];
  unpack16<T>(u, v);
#pragma unroll
  for (int e = 0; e < kVec16<T>; ++e) v[e] = ex2((v[e] - m) * k);
#pragma unroll
  for (int w = kVec16<T> / 2; w > 0; w >>= 1)
#pragma unroll
    for (int e = 0; e < w; ++e) v[e] += v[e + w];
  return v[0];
}

// log s for s in (0, 2^127]: exponent and mantissa apart, so that the error is that of the log of a number near 1
// (3e-8) and not half an ulp of the result (5e-7 for a vocabulary's sum).  0 gives -inf, NaN and inf themselves.
__device__ __forceinline__ double log_sum(float s) {
  if (!(s >= 1.1754944e-38f && s < INFINITY)) return log(static_cast<double>(s));
  const int e = (__float_as_int(s) - 0x3f3504f3) >> 23;  // mantissa into [sqrt(1/2), sqrt(2))
  const float f = __int_as_float(__float_as_int(s) - (e << 23));
  return static_cast<double>(e) * 0.6931471805599453 + static_cast<double>(logf(f));
}

struct TokenArgs {
  const void* logits;
  RowMap map;
  int64_t rows, cols;
  IntList targets;
  int64_t ignore_index;
  float k;             // log2(e) / T
  double inv_temp;
  float* logps;        // [rows]
  float4* row;         // [rows] {m, 1 / s, c, -}, or null
};

__device__ __forceinline__ double row_logp(const TokenArgs& a, RowStat st, float target_logit, int64_t t) {
  if (t < 0 || t >= a.cols) return static_cast<double>(NAN);
  return (static_cast<double>(target_logit) - static_cast<double>(st.m)) * a.inv_temp - log_sum(st.s);
}

// Sequence s holds rows [cu[s], cu[s + 1]); both ends are held to [0, rows] whatever the list says.
struct SeqList {
  IntList cu;
  int64_t count;    // sequences; 0: no list, every row takes part
  int64_t uniform;  // > 0: no list, every sequence holds this many rows
  __device__ __forceinline__ int64_t begin(int64_t s, int64_t rows) const {
    const int64_t v = uniform > 0 ? s * uniform : cu[s];
    return v < 0 ? 0 : (v > rows ? rows : v);
  }
  __device__ __forceinline__ bool covers(int64_t r) const {
    if (count == 0) return true;
    if (uniform > 0) return r < count * uniform;
    return cu[0] <= r && r < cu[count];
  }
  // The sequence of a covered row, the last s with cu[s] <= r: a warp looks at 32 offsets at a time.
  __device__ __forceinline__ int64_t of(int64_t r) const {
    if (count == 0) return 0;
    if (uniform > 0) return r / uniform;
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, hi = count;  // cu[lo] <= r < cu[hi]
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + 31) / 32;
      const int64_t at = lo + lane * step;
      const uint32_t below = __ballot_sync(0xffffffffu, at < hi && (lane == 0 || cu[at] <= r));
      const int64_t top = lo + (31 - __clz(below)) * step;
      if (top + step < hi) hi = top + step;
      lo = top;
    }
    return lo;
  }
};

struct RowArgs {
  TokenArgs t;
  SeqList seq;
  const float *old_logps, *advantages, *ref_logps;
  // policy
  int32_t adv_per_seq, reduction;  // reduction: 0 token mean, 1 mean over sequences of their token means, 2 sum
  float lo, hi, kl_coef;           // ratio bounds
  int32_t count_blocks;
  int32_t* counts;                 // [count_blocks] tokens that take part (token mean) or non-empty sequences
  float* seq_w;                    // [sequences] 1 / tokens of the sequence (sequence mean)
  uint32_t* done;
  float4* terms;                   // [rows] weighted loss, KL, clipped
  float* out;                      // loss, KL, clip fraction
  void* grad;
  RowMap gmap;
  // preference
  double* d;                       // [rows] lp - ref
};

constexpr int kCountBlocks = 64;

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Tokens that take part: all (token mean), or per sequence with the number of non-empty ones (sequence mean).
__global__ void __launch_bounds__(256) policy_count_kernel(RowArgs a) {
  __shared__ int smem[8];
  pdl_release();
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

// What a row's warps need to know of it besides its logits.
struct RowScalars {
  float target_logit, old, adv, ref, w;
};

enum RowMode : int { kLogps = 0, kPolicy = 1, kPreference = 2 };

template <typename T, int MODE>
__device__ __forceinline__ RowScalars load_scalars(const RowArgs& a, int64_t r, int64_t t) {
  RowScalars o{0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (t >= 0 && t < a.t.cols) o.target_logit = to_f32(static_cast<const T*>(a.t.logits)[a.t.map.at(r) + t]);
  if constexpr (MODE == kPolicy) {
    const int64_t s = a.seq.of(r);
    o.old = a.old_logps[r];
    o.adv = a.advantages[a.adv_per_seq ? s : r];
    if (a.ref_logps) o.ref = a.ref_logps[r];
    o.w = 1.0f;
    pdl_wait();  // the counts are the kernel before's
    if (a.reduction != 2) {
      const int lane = threadIdx.x & 31;
      int n = lane < a.count_blocks ? __ldcg(a.counts + lane) : 0;
      if (lane + 32 < a.count_blocks) n += __ldcg(a.counts + lane + 32);
      n = __reduce_add_sync(0xffffffffu, n);
      o.w = n > 0 ? 1.0f / static_cast<float>(n) : 0.0f;
      if (a.reduction == 1) o.w *= __ldcg(a.seq_w + s);
    }
  }
  if constexpr (MODE == kPreference) o.ref = a.ref_logps ? a.ref_logps[r] : 0.0f;
  return o;
}

// One token's terms, weighted by w, and its coefficient d loss / d logit scale.  KL = e^d - d - 1, d = ref - lp (its
// estimate from one sample, >= 0), formed as expm1(d) - d: the plain sum cancels for the small d of a policy near its
// reference.
__device__ __forceinline__ float4 policy_term(const RowArgs& a, const RowScalars& v, double lp, float& coef) {
  const float ratio = expf(static_cast<float>(lp - static_cast<double>(v.old)));
  const float held = fminf(fmaxf(ratio, a.lo), a.hi);
  const float gain = ratio * v.adv, gain_held = held * v.adv;
  const bool clipped = gain_held < gain;
  float loss = -(clipped ? gain_held : gain), slope = clipped ? 0.0f : -gain, kl = 0.0f;
  if (a.ref_logps) {
    const float d = static_cast<float>(static_cast<double>(v.ref) - lp), e = expm1f(d);
    kl = e - d;
    if (a.kl_coef != 0.0f) {
      loss = fmaf(a.kl_coef, kl, loss);
      slope = fmaf(-a.kl_coef, e, slope);
    }
  }
  coef = v.w * slope * static_cast<float>(a.t.inv_temp);
  if (v.w == 0.0f) {
    coef = 0.0f;
    return make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  return make_float4(v.w * loss, v.w * kl, clipped ? v.w : 0.0f, 0.0f);
}

// ---- clusters: the blocks of a cluster share a row ---------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_store(RowStat* p, uint32_t rank, RowStat v) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(v.m), "f"(v.s) : "memory");
}

__device__ __forceinline__ RowStat warp_merge(RowStat t, float k) {
  float m = t.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = t.s * ex2((t.m - m) * k);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return RowStat{m, s};
}

constexpr int kMaxCluster = 8;

// One row per GROUP threads of a block (a warp: four rows per block), or per cluster of blocks of 512.  RESIDENT rows
// are held in registers, NV 16-byte vectors a thread, from their one load to the gradient's store; longer rows are
// read twice (the second time from L2, where a cluster's one row has stayed).
//   kLogps:      lp (and m, 1 / s for a later gradient)
//   kPolicy:     lp, the loss's terms, and, if asked for, the gradient
//   kPreference: lp, lp - ref, and m, 1 / s
template <typename T, int GROUP, int NV, bool RESIDENT, int MODE>
__global__ void __launch_bounds__(GROUP < 128 ? 128 : GROUP, GROUP == 512 ? 2 : 1) token_row_kernel(RowArgs a) {
  constexpr int kWarps = GROUP / 32, V = kVec16<T>;
  constexpr bool kBlock = GROUP > 32;
  __shared__ RowStat stat[kBlock ? kMaxCluster * kWarps : 1];
  __shared__ RowScalars shared_scalars;
  __shared__ bool last;
  const int tid = threadIdx.x % GROUP, lane = threadIdx.x & 31;
  const uint32_t nranks = kBlock ? cluster_size() : 1, rank = kBlock ? cluster_rank() : 0;
  const int64_t r = kBlock ? blockIdx.x / nranks : static_cast<int64_t>(blockIdx.x) * (128 / GROUP) + threadIdx.x / GROUP;
  const bool have = r < a.t.rows;
  if (kBlock && nranks > 1) cluster_arrive();
  if (MODE == kPreference) pdl_release();

  const int64_t t = have ? a.t.targets[r] : a.t.ignore_index;
  const bool live = t != a.t.ignore_index && (MODE == kLogps || a.seq.covers(r));
  const T* p = static_cast<const T*>(a.t.logits) + (have ? a.t.map.at(r) : 0);
  const int cols = static_cast<int>(a.t.cols), head = static_cast<int>(peel(p, a.t.cols));
  const int nvec = (cols - head) / V;
  const int per = (nvec + nranks - 1) / nranks, begin = per * rank;
  // this thread's vectors: pv[u * GROUP] for u * GROUP < left
  const int at = begin + tid, left = (begin + per < nvec ? begin + per : nvec) - at;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head) + at;
  // elements in front of the first and behind the last vector: at most one a thread, rank 0
  int edge_at = tid < head ? tid : nvec * V + tid;
  if (rank != 0 || edge_at >= cols) edge_at = -1;

  uint4 v[NV];
  float edge = -INFINITY, coef = 0.0f;
  RowStat st{kLowest, 0.0f};
  if (live) {
    const uint32_t none = neg_inf_word<T>();
    if (edge_at >= 0) edge = to_f32(p[edge_at]);
    if constexpr (RESIDENT) {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        v[u] = u * GROUP < left ? load_stream(pv + u * GROUP) : make_uint4(none, none, none, none);
      }
    }
    RowScalars sc;
    if (!kBlock || threadIdx.x < 32) {
      sc = load_scalars<T, MODE>(a, r, t);
      if (kBlock && lane == 0) shared_scalars = sc;
    }
    if constexpr (RESIDENT) {
      st.m = fmaxf(edge, kLowest);
#pragma unroll
      for (int u = 0; u < NV; ++u) st.m = vec_max<T>(v[u], st.m);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) st.m = fmaxf(st.m, __shfl_xor_sync(0xffffffffu, st.m, o));
      st.s = ex2((edge - st.m) * a.t.k);
#pragma unroll
      for (int u = 0; u < NV; ++u) st.s += vec_sum<T>(v[u], st.m, a.t.k);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    } else {
      for (int i = 0; i < left; i += NV * GROUP) {
        float m = st.m;
#pragma unroll
        for (int u = 0; u < NV; ++u)
          v[u] = i + u * GROUP < left ? load_stream(pv + i + u * GROUP) : make_uint4(none, none, none, none);
#pragma unroll
        for (int u = 0; u < NV; ++u) m = vec_max<T>(v[u], m);
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < NV; ++u) s += vec_sum<T>(v[u], m, a.t.k);
        st.s = fmaf(st.s, ex2((st.m - m) * a.t.k), s);
        st.m = m;
      }
      const float m = fmaxf(edge, st.m);
      st.s = st.s * ex2((st.m - m) * a.t.k) + ex2((edge - m) * a.t.k);
      st.m = m;
      st = warp_merge(st, a.t.k);
    }
    if constexpr (kBlock) {
      const int warp = threadIdx.x >> 5;
      if (nranks > 1) {
        cluster_wait();  // every block of the cluster runs: its shared memory may be written
        if (lane < static_cast<int>(nranks)) cluster_store(&stat[rank * kWarps + warp], lane, st);
        cluster_arrive();
        cluster_wait();
      } else {
        if (lane == 0) stat[warp] = st;
        __syncthreads();
      }
      sc = shared_scalars;
      const int n = static_cast<int>(nranks) * kWarps;
      st = lane < n ? stat[lane] : RowStat{kLowest, 0.0f};
      for (int i = lane + 32; i < n; i += 32) st = merge(st, stat[i], a.t.k);
      st = warp_merge(st, a.t.k);
    }
    const double lp = row_logp(a.t, st, sc.target_logit, t);
    float4 term = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (MODE == kPolicy) term = policy_term(a, sc, lp, coef);
    if (rank == 0 && tid == 0) {
      a.t.logps[r] = static_cast<float>(lp);
      if constexpr (MODE == kPolicy) a.terms[r] = term;
      if constexpr (MODE == kPreference) a.d[r] = lp - static_cast<double>(sc.ref);
      if (MODE != kPolicy && a.t.row) a.t.row[r] = make_float4(st.m, 1.0f / st.s, 0.0f, 0.0f);
    }
  } else {
    if (kBlock && nranks > 1) cluster_wait();
    if (MODE == kPolicy) pdl_wait();
    if (have && rank == 0 && tid == 0) {
      a.t.logps[r] = 0.0f;
      if constexpr (MODE == kPolicy) a.terms[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if constexpr (MODE == kPreference) a.d[r] = 0.0;
      if (MODE != kPolicy && a.t.row) a.t.row[r] = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
    }
  }
  if (MODE == kPreference && blockIdx.x == 0 && threadIdx.x == 0) *a.done = 0;

  if constexpr (MODE == kPolicy) {
    // the block (of rank 0) whose rows' terms are the last to arrive adds them all, below
    if (!kBlock) __syncthreads();
    if (threadIdx.x == 0) {
      last = false;
      if (rank == 0) {
        __threadfence();
        last = atomicAdd(a.done, 1u) == gridDim.x / nranks - 1;
      }
    }
    if (a.grad && have) {
      T* g = static_cast<T*>(a.grad) + a.gmap.at(r);
      const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
      const float q = -coef / st.s;
      const bool zero = coef == 0.0f;  // zeros whatever the logits hold, NaN and infinities included
      float at_t = 0.0f;
      int target_at = -1;  // the target among this thread's vectors, in elements from its first
      if (!zero && t >= 0 && t < cols) {
        const float x = kBlock ? shared_scalars.target_logit : to_f32(p[t]);
        at_t = fmaf(q, ex2((x - st.m) * a.t.k), coef);
        target_at = static_cast<int>(t) - head - at * V;
      }
      if (!kBlock) __syncwarp();  // in place: the target's logit is read before it is overwritten
      uint4* gv = reinterpret_cast<uint4*>(g + head) + at;
      auto put = [&](const uint4& raw, int i) {
        float x[V];
        if (zero) {
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = 0.0f;
        } else {
          unpack16<T>(raw, x);
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = q * ex2((x[e] - st.m) * a.t.k);
          if (static_cast<uint32_t>(target_at - i * V) < static_cast<uint32_t>(V)) {
#pragma unroll
            for (int e = 0; e < V; ++e)
              if (target_at - i * V == e) x[e] = at_t;
          }
        }
        if (same) {
          __stcs(gv + i, pack16<T>(x));
        } else {
          T* to = reinterpret_cast<T*>(gv) + static_cast<int64_t>(i) * V;
#pragma unroll
          for (int e = 0; e < V; ++e) to[e] = from_f32<T>(x[e]);
        }
      };
      if constexpr (RESIDENT) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
          if (u * GROUP < left) put(v[u], u * GROUP);
      } else {
        for (int i = 0; i < left; i += NV * GROUP) {
#pragma unroll
          for (int u = 0; u < NV; ++u)
            if (!zero && i + u * GROUP < left) v[u] = load_stream(pv + i + u * GROUP);
#pragma unroll
          for (int u = 0; u < NV; ++u)
            if (i + u * GROUP < left) put(v[u], i + u * GROUP);
        }
      }
      if (edge_at >= 0)
        g[edge_at] = from_f32<T>(zero ? 0.0f : (edge_at == t ? at_t : q * ex2((edge - st.m) * a.t.k)));
    }
    __syncthreads();
    if (last) {
      __shared__ double smem[kBlock ? kWarps : 4];
      __threadfence();
      double x = 0.0, y = 0.0, z = 0.0;
      for (int64_t i = threadIdx.x; i < a.t.rows; i += blockDim.x) {
        const float4 f = __ldcg(a.terms + i);
        x += f.x;
        y += f.y;
        z += f.z;
      }
      x = block_sum(x, smem);
      y = block_sum(y, smem);
      z = block_sum(z, smem);
      if (threadIdx.x == 0) {
        a.out[0] = static_cast<float>(x);
        a.out[1] = static_cast<float>(y);
        a.out[2] = static_cast<float>(z);
      }
    }
  }
}

// ---- preference loss -------------------------------------------------------------------------------
struct PreferenceArgs {
  TokenArgs t;
  SeqList seq;               // pairs: sequence i against sequence i + count / 2
  const double* d;           // [rows] lp - ref, 0 at rows that take no part
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
    if (isnan(h)) loss = h;
  } else if (a.kind == 1) {
    loss = isnan(h) ? h : fmax(1.0 - h, 0.0);
    slope = h < 1.0 ? -1.0 : (isnan(h) ? h : 0.0);
  } else {
    loss = (h - 0.5) * (h - 0.5);
    slope = 2.0 * (h - 0.5);
  }
}

// One block per pair: the sums of both sequences, the pair's loss, and the coefficient of their rows.
__global__ void __launch_bounds__(256) preference_pair_kernel(PreferenceArgs a) {
  __shared__ double smem[8];
  pdl_release();
  pdl_wait();
  const int64_t pairs = a.seq.count / 2, i = blockIdx.x;
  double d[2], n[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t s = i + side * pairs;
    const int64_t lo = a.seq.begin(s, a.t.rows), hi = a.seq.begin(s + 1, a.t.rows);
    double x = 0.0, c = 0.0;
    for (int64_t r = lo + threadIdx.x; r < hi; r += 256) {
      x += __ldcg(a.d + r);
      c += a.t.targets[r] != a.t.ignore_index ? 1.0 : 0.0;
    }
    d[side] = block_sum(x, smem);
    n[side] = a.average ? block_sum(c, smem) : 1.0;
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
      if (n[side] > 0.0) c /= n[side];
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

// ---- gradient of the logits from kept row statistics ---------------------------------------------------
struct GradArgs {
  TokenArgs t;
  const float* slope;  // [rows] d loss / d lp, or null: the coefficient is row[r].z
  void* grad;
  RowMap gmap;
  int32_t parts;       // blocks per row
};

// `parts` blocks per row, the last rows first: the pass before read them last, and what of them is still in L2 need
// not come from memory again.  A row whose coefficient is zero (ignored, or a flat loss) is written as zeros and not
// read: what its logits hold does not reach the gradient.  `grad` may be the logits themselves: then one block writes
// a row (parts is 1), after it has read the target's logit.
template <typename T>
__global__ void __launch_bounds__(256) logit_grad_kernel(GradArgs a) {
  constexpr int V = kVec16<T>, U = 4;
  pdl_wait();
  const int64_t r = a.t.rows - 1 - blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const float4 st = __ldcg(a.t.row + r);
  const int64_t t = a.t.targets[r];
  const float c = a.slope ? (t == a.t.ignore_index ? 0.0f : a.slope[r] * static_cast<float>(a.t.inv_temp)) : st.z;
  const T* p = static_cast<const T*>(a.t.logits) + a.t.map.at(r);
  T* g = static_cast<T*>(a.grad) + a.gmap.at(r);
  const float q = -c * st.y;
  const bool zero = c == 0.0f;
  float at_t = 0.0f;
  if (!zero && t >= 0 && t < a.t.cols) at_t = fmaf(q, ex2((to_f32(p[t]) - st.x) * a.t.k), c);
  if (p == g) __syncthreads();
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  const int64_t head = same ? peel(g, a.t.cols) : a.t.cols;
  const int64_t nvec = (a.t.cols - head) / V, tail = head + nvec * V;
  const int64_t per = (nvec + a.parts - 1) / a.parts;
  const int64_t end = per * (part + 1) < nvec ? per * (part + 1) : nvec;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  uint4* gv = reinterpret_cast<uint4*>(g + head);
  const int64_t tv = !zero && t >= head && t < tail ? (t - head) / V : -1;
  for (int64_t i0 = per * part + threadIdx.x; i0 < end; i0 += 256 * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!zero && i0 + u * 256 < end) raw[u] = load_stream(pv + i0 + u * 256);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * 256;
      if (i >= end) break;
      float v[V];
      if (zero) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = 0.0f;
      } else {
        unpack16<T>(raw[u], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = q * ex2((v[e] - st.x) * a.t.k);
        if (i == tv) {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (head + i * V + e == t) v[e] = at_t;
        }
      }
      __stcs(gv + i, pack16<T>(v));
    }
  }
  auto one = [&](int64_t j) {
    g[j] = from_f32<T>(zero ? 0.0f : (j == t ? at_t : q * ex2((to_f32(p[j]) - st.x) * a.t.k)));
  };
  if (same) {  // the few elements in front of and behind the vectors
    const int64_t j = static_cast<int64_t>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
    if (part == 0 && j < a.t.cols) one(j);
  } else {     // rows of the two off each other's alignment
    for (int64_t j = static_cast<int64_t>(part) * 256 + threadIdx.x; j < a.t.cols; j += 256ll * a.parts) one(j);
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
// A launch in clusters of `cluster` blocks; `early`: it may start before the kernel in front of it has ended, and
// waits (griddepcontrol.wait) where it needs that kernel's results.
template <typename Args>
cudaError_t launch_kernel(void (*fn)(Args), int64_t blocks, int threads, int cluster, bool early, const Args& args,
                          cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (early) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = static_cast<unsigned>(n);
  count_launch();
  return cudaLaunchKernelEx(&cfg, fn, args);
}

// The row kernel for a row of `vecs` 16-byte vectors: a warp up to 8 vectors a lane, a block of 128 up to 8 a thread,
// else blocks of 512 in the smallest cluster whose threads hold the row in 10 vectors each; longer rows
// run through a cluster of 8 twice.  With fewer rows than fill the SMs, a larger cluster shares a row.
template <typename T, int MODE>
cudaError_t launch_rows(const RowArgs& a, bool early, cudaStream_t stream) {
  const int64_t rows = a.t.rows, vecs = (a.t.cols + kVec16<T> - 1) / kVec16<T>;
  if (vecs <= 32 * 2) return launch_kernel(token_row_kernel<T, 32, 2, true, MODE>, (rows + 3) / 4, 128, 1, early, a, stream);
  if (vecs <= 32 * 8 && rows > 4 * 148)
    return launch_kernel(token_row_kernel<T, 32, 8, true, MODE>, (rows + 3) / 4, 128, 1, early, a, stream);
  if (vecs <= 128 * 3) return launch_kernel(token_row_kernel<T, 128, 3, true, MODE>, rows, 128, 1, early, a, stream);
  if (vecs <= 128 * 8 && rows > 2 * 148)
    return launch_kernel(token_row_kernel<T, 128, 8, true, MODE>, rows, 128, 1, early, a, stream);
  int cluster = 1;
  while (cluster < kMaxCluster && (vecs > 512 * 10 * cluster || (rows * cluster < 148 && vecs > 1024 * cluster))) cluster *= 2;
  const int64_t need = (vecs + 512 * cluster - 1) / (512 * cluster);
  const int64_t blocks = rows * cluster;
  if (need <= 3) return launch_kernel(token_row_kernel<T, 512, 3, true, MODE>, blocks, 512, cluster, early, a, stream);
  if (need <= 6) return launch_kernel(token_row_kernel<T, 512, 6, true, MODE>, blocks, 512, cluster, early, a, stream);
  if (need <= 8) return launch_kernel(token_row_kernel<T, 512, 8, true, MODE>, blocks, 512, cluster, early, a, stream);
  if (need <= 10) return launch_kernel(token_row_kernel<T, 512, 10, true, MODE>, blocks, 512, cluster, early, a, stream);
  return launch_kernel(token_row_kernel<T, 512, 4, false, MODE>, blocks, 512, cluster, early, a, stream);
}

template <typename T>
cudaError_t token_logps_t(const RowArgs& a, cudaStream_t stream) {
  return launch_rows<T, kLogps>(a, false, stream);
}

template <typename T>
cudaError_t policy_loss_t(const RowArgs& a, cudaStream_t stream) {
  const cudaError_t e = launch_kernel(policy_count_kernel, a.count_blocks, 256, 1, false, a, stream);
  return e != cudaSuccess ? e : launch_rows<T, kPolicy>(a, true, stream);
}

template <typename T>
cudaError_t logit_grad_t(GradArgs a, bool early, cudaStream_t stream) {
  const bool in_place = a.grad == a.t.logits;
  const int64_t want = (4 * 148 + a.t.rows - 1) / a.t.rows, most = (a.t.cols + 8191) / 8192;
  a.parts = static_cast<int32_t>(in_place ? 1 : (want < most ? want : most));
  return launch_kernel(logit_grad_kernel<T>, a.t.rows * a.parts, 256, 1, early, a, stream);
}

template <typename T>
cudaError_t preference_loss_t(const RowArgs& rows, const PreferenceArgs& a, const GradArgs& g, cudaStream_t stream) {
  cudaError_t e = launch_rows<T, kPreference>(rows, false, stream);
  if (e == cudaSuccess) e = launch_kernel(preference_pair_kernel, a.seq.count / 2, 256, 1, true, a, stream);
  return e != cudaSuccess || !g.grad ? e : logit_grad_t<T>(g, true, stream);
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
