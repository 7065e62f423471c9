// Token log-probabilities, the clipped policy loss and the paired preference loss over (rows, vocab) logits,
// with the gradient of the logits.  With x = logits / T, target t_r and
//   m_r = max_j logits[r, j],  s_r = sum_j exp(x[r, j] - m_r / T):
//   lp_r = x[r, t_r] - m_r / T - log s_r,     p[r, j] = exp(x[r, j] - m_r / T) / s_r
// and every loss here depends on the logits through lp alone, so
//   d loss / d logits[r, j] = c_r (1{j = t_r} - p[r, j]),   c_r = (d loss / d lp_r) / T.
//
// fp32 logits are bound by memory; 16-bit ones by the operations of a row's sum (an exponential per logit, 16 a clock and
// SM, and about six operations around it).  The policy loss's coefficient belongs to one row, so its row is read once and
// written as gradient from what is still on the chip; the preference loss's needs all rows of two sequences, so its
// gradient reads the logits a second time.
//
// The maximum starts at the lowest finite float, so a row of -inf, or of the type's lowest value, needs no special
// case: exp(-inf - m) = 0 and exp(lowest - lowest) = 1.  A row of -inf alone gives s = 0 and lp = NaN, as the
// formula does; a NaN or +inf logit makes its row's lp NaN.  A thread's sums are fp32, without a mean error (see Part);
// threads, warps and blocks are joined in double, and lp is formed in double (the difference lp - ref summed over a
// sequence would otherwise carry each token's last rounding).
#include "kernels.cuh"
#include "lm_common.cuh"

namespace mib {

constexpr float kLowest = -3.402823466e38f;

// log2(e) / T as hi + lo.  One fp32 number is up to 6e-8 off, which every exponential of a row has in the same direction:
// nothing next to a log-probability's own rounding, but summed over a sequence's tokens more than all their roundings.
// hi is rounded down and lo is above zero, so that -inf times either is -inf.
struct Scale {
  float hi, lo;
  double k;    // log2(e) / T
  float unit;  // of 2's logarithm: 1 / k
};

// exp((a - b) / T) for joining a row's sums, in double: an fp32 factor's rounding would be the same in every row whose
// differences are (16-bit logits).  2^x with x = n + f, |f| <= 1/2: the exponential's series at f log(2), within 1e-11.  Below
// 2^-1000 it is 2^-1000, for a NaN too (the sums of a part that holds one are NaN by themselves).  (The library's exp2 and
// log cost rows of 128 to 1500 fp32 logits 1 us of 10 to 20 more, by 16384 rows.)
constexpr double kLn2 = 0.6931471805599453;
__device__ __forceinline__ double exp_of(float a, float b, Scale k) {
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52: adding it leaves n in the low bits
  const double x = fmax((static_cast<double>(a) - static_cast<double>(b)) * k.k, -1000.0), t = x + kWhole;
  const double r = (x - (t - kWhole)) * kLn2;
  double p = 1.0 / 362880;
  p = fma(r, p, 1.0 / 40320);
  p = fma(r, p, 1.0 / 5040);
  p = fma(r, p, 1.0 / 720);
  p = fma(r, p, 1.0 / 120);
  p = fma(r, p, 1.0 / 24);
  p = fma(r, p, 1.0 / 6);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}
// log s of a row's sum: s = 2^e f with f in [sqrt(1/2), sqrt(2)), log f = 2 artanh z with z = (f - 1) / (f + 1), by its series
// (within 1e-12).  0 gives -inf, NaN and inf themselves.
__device__ __forceinline__ double log_of(double s) {
  if (!(s > 1e-300 && s < 1e300)) return s > 0.0 ? s : (s == 0.0 ? -static_cast<double>(INFINITY) : s);
  const int hi = __double2hiint(s), e = (hi - 0x3fe6a09e) >> 20;
  const double f = __hiloint2double(hi - (e << 20), __double2loint(s)), b = f + 1.0;
  double y = static_cast<double>(__frcp_rn(static_cast<float>(b)));
  y *= fma(-b, y, 2.0);
  const double z = (f - 1.0) * y, w = z * z;
  double p = 1.0 / 13;
  p = fma(w, p, 1.0 / 11);
  p = fma(w, p, 1.0 / 9);
  p = fma(w, p, 1.0 / 7);
  p = fma(w, p, 1.0 / 5);
  p = fma(w, p, 1.0 / 3);
  return fma(static_cast<double>(e), kLn2, fma(z * w, 2.0 * p, 2.0 * z));
}
// exp(d / T) by the hardware, within 2e-7: the gradient's elements, whose errors stay their own, and the sums' terms (see
// Part).
__device__ __forceinline__ float exp_hw(float d, Scale k) { return ex2(fmaf(d, k.hi, d * k.lo)); }

// Maximum and sum of exponentials of a part of a row.
struct __align__(16) RowStat {
  double s;
  float m;
};
__device__ __forceinline__ RowStat merge(RowStat a, RowStat b, Scale k) {
  const float m = fmaxf(a.m, b.m);
  return RowStat{a.s * exp_of(a.m, m, k) + b.s * exp_of(b.m, m, k), m};
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

// The maximum of a vector's elements and m.
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

// How a thread adds up exponentials without a mean error.  The hardware's ex2 is low on average: by 4.95e-8 to 5.1e-8 over
// any octave of arguments below -1, by 2.2e-8 from -1 to 0 (measured on a B200, 2^26 arguments an octave), and by up to 2e-7
// either way at one argument.  A sequence's tokens would add the mean up, and where logits repeat (16-bit ones on a grid,
// flat rows) the error of the same few arguments too.  So each thread refers its terms to its maximum (or more) plus an
// offset of its own and the row's, between 1 and 2 in units of 2's logarithm and spread evenly over the threads: whatever
// the logits are, the arguments of a row and of all rows cover an octave below -1, the mean error is the octave's, and
// 1 + 5.0e-8 takes it out.  The largest term is taken out too and counts as 1 exactly: a row that one logit carries has no
// error at all.  (A polynomial in place of ex2 takes 150 us on 2048 x 151936 bf16 where this takes 107, and still rounds
// repeated logits alike.)
//
// The sums keep what their additions round away: the many small terms beside a large one would each be lost, always
// downwards (1e-8 of the row where logits spread over 30, and twice that at 32003 columns; 97 us).  (Adding 16-bit logits'
// terms in twos plainly before takes 104 us, and loses 2.5e-9 of such a row.)  What is left is within 2e-9 on average over
// the spreads, temperatures, types and vocabularies tried.
constexpr double kEx2Low = 5.0e-8;
constexpr int kSums = 4, kLosts = 2;  // pairs
constexpr float kSlack = 8.0f;        // a reference leaves room for a maximum 2^8 times as large
struct Part {
  float m, limit, ref;  // the maximum so far; the largest logit that `ref` has room for
  uint32_t place;       // the thread's, in steps near the golden section: any run of threads covers the octave evenly
  float2 sum[kSums], lost[kLosts];
  __device__ __forceinline__ Part(int tid) {
    place = static_cast<uint32_t>(tid) * 5184445u;
    restart();
  }
  __device__ __forceinline__ void restart() {
    m = limit = ref = kLowest;
#pragma unroll
    for (int i = 0; i < kSums; ++i) sum[i] = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < kLosts; ++i) lost[i] = make_float2(0.0f, 0.0f);
  }
  // For logits up to `top`.
  __device__ __forceinline__ void refer(float top, Scale k) {
    limit = top;
    const uint32_t w = (place + (__float_as_uint(top) * 0x9e3779b1u >> 9)) & 0x7fffffu;
    ref = top + fmaf(static_cast<float>(w), 0x1p-23f, 1.0f) * k.unit;
  }
  // The same with logits added before, and room for more.
  __device__ __forceinline__ void raise(float top, Scale k) {
    const float old = ref;
    refer(top + kSlack * k.unit, k);
    float2 any = sum[0];
#pragma unroll
    for (int i = 1; i < kSums; ++i) any = add2(any, sum[i]);
    if (any.x + any.y == 0.0f) return;  // nothing yet
    const float f = static_cast<float>(exp_of(old, ref, k));
#pragma unroll
    for (int i = 0; i < kSums; ++i) sum[i] = mul2(sum[i], make_float2(f, f));
#pragma unroll
    for (int i = 0; i < kLosts; ++i) lost[i] = mul2(lost[i], make_float2(f, f));
  }
  // N vectors' elements, none above `limit`; FRESH: the first ones
  template <typename T, bool FRESH, int N>
  __device__ __forceinline__ void add(const uint4 (&u)[N], Scale k) {
    constexpr int P = kVec16<T> / 2;
    const float2 minus = make_float2(-ref, -ref), hi = make_float2(k.hi, k.hi), lo = make_float2(k.lo, k.lo);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v[kVec16<T>];
      unpack16<T>(u[i], v);
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 d = add2(make_float2(v[2 * j], v[2 * j + 1]), minus), y = fma2(d, hi, mul2(d, lo));
        const float2 e = make_float2(ex2(y.x), ex2(y.y));
        float2 &s = sum[(i * P + j) % kSums], &l = lost[j % kLosts];
        if (FRESH && i * P + j < kSums) {
          s = e;
          continue;
        }
        const float2 next = add2(s, e);
        l = add2(l, sub2(e, sub2(next, s)));
        s = next;
      }
    }
  }
  // The sum relative to m.  `own`: one of the terms, if there are any, is that of m itself.
  __device__ __forceinline__ double total(bool own, Scale k) const {
    // additions in fp32 that keep their errors (each the exact rest of a sum of two), then one conversion of sum and rest
    float2 s2 = sum[0], l = lost[0];
#pragma unroll
    for (int i = 1; i < kSums; ++i) {
      const float2 next = add2(s2, sum[i]), b = sub2(next, s2);
      l = add2(l, add2(sub2(s2, sub2(next, b)), sub2(sum[i], b)));
      s2 = next;
    }
#pragma unroll
    for (int i = 1; i < kLosts; ++i) l = add2(l, lost[i]);
    const float h = s2.x + s2.y, b = h - s2.x, rest = (s2.x - (h - b)) + (s2.y - b) + (l.x + l.y);
    const double s = static_cast<double>(h) + static_cast<double>(rest);
    const double factor = exp_of(ref, m, k) * (1.0 + kEx2Low);
    return own && s != 0.0 ? 1.0 + (s - static_cast<double>(exp_hw(m - ref, k))) * factor : s * factor;
  }
};

// One element as a part of its own (an absent one is -inf): NaN and +inf have no sum.
__device__ __forceinline__ RowStat one_stat(float v) {
  return RowStat{v == -INFINITY ? 0.0 : 1.0 + static_cast<double>(v - v), fmaxf(v, kLowest)};
}

// N vectors of logits to q times their exponentials, and with SCALED times f, in the logits' type.
template <typename T, bool SCALED, int N>
__device__ __forceinline__ void vecs_grad(uint4 (&u)[N], float m, Scale k, float q, float f = 1.0f) {
  const float2 minus = make_float2(-m, -m), hi = make_float2(k.hi, k.hi), lo = make_float2(k.lo, k.lo);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float v[kVec16<T>];
    unpack16<T>(u[i], v);
#pragma unroll
    for (int e = 0; e < kVec16<T>; e += 2) {
      const float2 d = add2(make_float2(v[e], v[e + 1]), minus), y = fma2(d, hi, mul2(d, lo));
      float2 g = mul2(make_float2(q, q), make_float2(ex2(y.x), ex2(y.y)));
      if (SCALED) g = mul2(g, make_float2(f, f));
      v[e] = g.x;
      v[e + 1] = g.y;
    }
    u[i] = pack16<T>(v);
  }
}

struct TokenArgs {
  const void* logits;
  RowMap map;
  int64_t rows, cols;
  IntList targets;
  int64_t ignore_index;
  Scale k;             // log2(e) / T
  double inv_temp;     // 1 / T
  float* logps;        // [rows]
  float4* row;         // [rows] {m, s, c, -} for a gradient later, or null
};

__device__ __forceinline__ double row_logp(const TokenArgs& a, RowStat st, float target_logit, int64_t t) {
  if (t < 0 || t >= a.cols) return static_cast<double>(NAN);
  return (static_cast<double>(target_logit) - static_cast<double>(st.m)) * a.inv_temp - log_of(st.s);
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

enum RowMode : int { kStats = 0, kPolicy = 1 };

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
  if (MODE == kStats && a.ref_logps) o.ref = a.ref_logps[r];
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
__device__ __forceinline__ void cluster_store(RowStat* p, uint32_t rank, RowStat v) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(v.s) : "memory");
  asm volatile("st.shared::cluster.f32 [%0+8], %1;" ::"r"(to), "f"(v.m) : "memory");
}

__device__ __forceinline__ RowStat warp_sum(double s, float m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return RowStat{s, m};
}
__device__ __forceinline__ RowStat warp_merge(RowStat t, Scale k) {
  float m = t.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return warp_sum(t.s * exp_of(t.m, m, k), m);
}

// The loss and its statistics from the rows' terms, by the block that arrived last.
template <int WARPS>
__device__ __forceinline__ void add_terms(const RowArgs& a) {
  __shared__ double smem[WARPS];
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

// A vector's elements one by one, to a place off its alignment.
template <typename T>
__device__ __forceinline__ void store_elements(const uint4& v, uint4* to) {
  if (!to) return;
  const T* x = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int e = 0; e < kVec16<T>; ++e) reinterpret_cast<T*>(to)[e] = x[e];
}

constexpr int kMaxCluster = 8;

// One row per GROUP threads of a block (a warp: four rows per block), or per cluster of blocks of 512.  RESIDENT rows
// are held in registers, NV 16-byte vectors a thread, from their one load to the gradient's store; longer rows are
// read twice (the second time from L2, where a cluster's one row has stayed).
//   kStats:   lp and, where asked for, m and 1 / s for a later gradient, and lp - ref
//   kPolicy:  lp, the loss's terms, and, where asked for, the gradient
// (A warp that reads its row twice has many loads to wait for: 8 blocks an SM, 64 registers, make the policy loss on
// 16384 x 1500 fp32 60 us, 67 without.)
template <typename T, int GROUP, int NV, bool RESIDENT, int MODE>
__global__ void __launch_bounds__(GROUP < 128 ? 128 : GROUP, GROUP == 512 ? 2 : (GROUP == 32 && !RESIDENT ? 8 : 1))
    token_row_kernel(RowArgs a) {
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
  if (MODE == kStats) pdl_release();

  const int64_t t = have ? a.t.targets[r] : a.t.ignore_index;
  const bool live = t != a.t.ignore_index && a.seq.covers(r);
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
  RowStat st{0.0, kLowest};
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
    Part part(tid);
    if constexpr (RESIDENT) {
      float top = kLowest;
#pragma unroll
      for (int u = 0; u < NV; ++u) top = vec_max<T>(v[u], top);
      float m = fmaxf(edge, top);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      part.m = m;
      part.refer(m, a.t.k);
      part.add<T, true>(v, a.t.k);
      double s = part.total(top == m, a.t.k);
      if (edge_at >= 0) s += one_stat(edge).s * exp_of(edge, m, a.t.k);
      st = warp_sum(s, m);
    } else {
      for (int i = 0; i < left; i += NV * GROUP) {
        float top = part.m;
#pragma unroll
        for (int u = 0; u < NV; ++u)
          v[u] = i + u * GROUP < left ? load_stream(pv + i + u * GROUP) : make_uint4(none, none, none, none);
#pragma unroll
        for (int u = 0; u < NV; ++u) top = vec_max<T>(v[u], top);
        if (top > part.limit) part.raise(top, a.t.k);
        part.m = top;
        part.add<T, false>(v, a.t.k);
      }
      st = RowStat{part.total(true, a.t.k), part.m};
      if (edge_at >= 0) st = merge(st, one_stat(edge), a.t.k);
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
      st = lane < n ? stat[lane] : RowStat{0.0, kLowest};
      for (int i = lane + 32; i < n; i += 32) st = merge(st, stat[i], a.t.k);
      st = warp_merge(st, a.t.k);
    }
    const double lp = row_logp(a.t, st, sc.target_logit, t);
    float4 term = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (MODE == kPolicy) term = policy_term(a, sc, lp, coef);
    if (rank == 0 && tid == 0) {
      a.t.logps[r] = static_cast<float>(lp);
      if constexpr (MODE == kPolicy) a.terms[r] = term;
      if (MODE == kStats && a.d) a.d[r] = lp - static_cast<double>(sc.ref);
      if (a.t.row) a.t.row[r] = make_float4(st.m, static_cast<float>(st.s), coef, 0.0f);
    }
  } else {
    if (kBlock && nranks > 1) cluster_wait();
    if (MODE == kPolicy) pdl_wait();
    if (have && rank == 0 && tid == 0) {
      a.t.logps[r] = 0.0f;
      if constexpr (MODE == kPolicy) a.terms[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (MODE == kStats && a.d) a.d[r] = 0.0;
      if (a.t.row) a.t.row[r] = make_float4(0.0f, 1.0f, 0.0f, 0.0f);
    }
  }
  if (MODE == kStats && a.done && blockIdx.x == 0 && threadIdx.x == 0) *a.done = 0;

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
      const float q = -coef / static_cast<float>(st.s);
      const bool zero = coef == 0.0f;  // zeros whatever the logits hold, NaN and infinities included
      const bool hit = t >= 0 && t < cols;
      float target_logit = 0.0f;
      if (hit) target_logit = kBlock ? shared_scalars.target_logit : to_f32(p[t]);
      if (!kBlock) __syncwarp();  // in place: the target's logit is read before it is overwritten
      uint4* gv = reinterpret_cast<uint4*>(g + head) + at;
      auto store = [&](int i0) {
        if (zero) {
#pragma unroll
          for (int u = 0; u < NV; ++u) v[u] = make_uint4(0, 0, 0, 0);
        } else {
          vecs_grad<T, false>(v, st.m, a.t.k, q);
        }
        if (same) {
#pragma unroll
          for (int u = 0; u < NV; ++u)
            if (i0 + u * GROUP < left) __stcs(gv + i0 + u * GROUP, v[u]);
        } else {
#pragma unroll
          for (int u = 0; u < NV; ++u) store_elements<T>(v[u], i0 + u * GROUP < left ? gv + i0 + u * GROUP : nullptr);
        }
      };
      if constexpr (RESIDENT) {
        store(0);
      } else {
        for (int i = 0; i < left; i += NV * GROUP) {
#pragma unroll
          for (int u = 0; u < NV; ++u)
            if (!zero && i + u * GROUP < left) v[u] = load_stream(pv + i + u * GROUP);
          store(i);
        }
      }
      if (edge_at >= 0) g[edge_at] = from_f32<T>(zero ? 0.0f : q * exp_hw(edge - st.m, a.t.k));
      if (hit && !zero) {  // the target's element again, by the thread that wrote it
        const int j = static_cast<int>(t), i = (j - head) / V;
        if (j == edge_at || (j >= head && i < nvec && i >= begin && i < begin + per && (i - begin) % GROUP == tid))
          g[j] = from_f32<T>(fmaf(q, exp_hw(target_logit - st.m, a.t.k), coef));
      }
    }
    __syncthreads();
    if (last) add_terms<kBlock ? kWarps : 4>(a);
  }
}

// ---- long rows: a ring of shared memory between the copies and the arithmetic ---------------------------
// One block per SM (or a few smaller ones); the grid has a block per row, and a running block takes over rows whose
// blocks have not started (clusterlaunchcontrol), so that rows that take no part cost nobody a turn.  Three roles that
// meet at mbarriers only:
//   copies      one thread fetches the next row's number and copies the row, chunk by chunk, into a ring of SLOTS slots;
//   arithmetic  CT threads: running maximum and sum of their part of every chunk, then the gradient;
//   scalars     one warp fetches what the row needs besides its logits while its statistics are made, merges the
//               warps' parts, and forms the row's log-probability, loss terms and coefficient once for all.
// A policy row with a gradient is walked twice: its last KEEP chunks stay in the ring for the second walk, the ones in
// front of them are given back after the statistics and copied again (from L2: the row passed moments before), while
// the kept ones turn into gradient.  Copies of the next row start as slots fall free.
//
// On one B200, 1536 of 2048 rows taking part: log-probabilities of 151936 fp32 logits 135 us, 6.9 TB/s (bound by memory),
// bf16 107 us, 4.4 TB/s (the sums' operations: 65% of the issue slots, 55% of the multiply and of the special-function
// pipes' cycles); the policy loss with gradient on fp32 406 us, 5.4 TB/s of the bytes it cannot do without, on bf16 229 us,
// 4.8 TB/s.  The second copies of fp32 rows miss L2 for about a third (148 rows of 608 KB are on their way; without the
// eviction hints 457 us).  Sharing a row between the blocks of a cluster needs no second copy and measured 385 us on fp32,
// but 490 us on 4096 rows of bf16 where this took 416, a row's exchange costing 2 us, so it is not used.
constexpr int kRowSlots = 4;  // rows between the copies and the other two

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}
// L2 eviction policies: lines that will be copied again, and lines that will not.
__device__ __forceinline__ uint64_t l2_keep() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t l2_drop() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Asks for the number of a block of this grid that has not started; the answer (16 bytes) arrives at `bar`.
__device__ __forceinline__ void next_row_ask(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// The block's number, or -1 when none is left (then nothing more may be asked).
__device__ __forceinline__ int64_t next_row_read(const uint4* answer) {
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\tld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return got ? static_cast<int64_t>(x) : -1;
}

template <int SLOTS>
struct RingPos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++slot == SLOTS) {
      slot = 0;
      phase ^= 1;
    }
  }
};

template <int CT, int VECS, int SLOTS>
constexpr size_t ring_bytes() {
  return static_cast<size_t>(SLOTS) * CT * VECS * 16;
}

template <typename T, int CT, int VECS, int SLOTS, int KEEP, int MODE>
__global__ void __launch_bounds__(CT + 64, CT < 512 ? 512 / CT : 1) token_ring_kernel(RowArgs a) {
  constexpr int V = kVec16<T>, kWarps = CT / 32, kChunk = CT * VECS;
  constexpr int kErr = 0x70;
  extern __shared__ __align__(128) uint4 ring[];
  __shared__ uint64_t full[SLOTS], empty[SLOTS], row_full[kRowSlots], row_empty[kRowSlots];
  __shared__ uint64_t stat_full[2], stat_empty[2], coef_full, asked;
  __shared__ __align__(16) uint4 answer;
  __shared__ RowStat stat[2][kWarps];
  __shared__ float4 row_coef;  // m, coefficient, -coefficient / s, target's logit
  __shared__ int64_t row_number[kRowSlots], row_target[kRowSlots];
  __shared__ volatile int abort_flag;
  __shared__ bool last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cols = static_cast<int>(a.t.cols);
  const bool want_grad = MODE == kPolicy && a.grad;
  if (MODE == kStats) pdl_release();
  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], kWarps);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      mbar_init(&row_full[i], 1);
      mbar_init(&row_empty[i], kWarps + 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&stat_full[i], kWarps);
      mbar_init(&stat_empty[i], 1);
    }
    mbar_init(&coef_full, 1);
    mbar_init(&asked, 1);
    abort_flag = 0;
    last = false;
    fence_mbar_init();
  }
  __syncthreads();

  if (warp == kWarps) {  // ---- rows and copies
    if (lane == 0) {
      const uint64_t keep_policy = l2_keep(), drop_policy = l2_drop();
      RingPos<SLOTS> pos;
      int64_t issued = 0, r = blockIdx.x;
      bool ok = true;
      for (int64_t k = 0; ok; ++k) {
        const int b = static_cast<int>(k % kRowSlots);
        int64_t t = a.t.ignore_index;
        if (r >= 0) {
          t = a.t.targets[r];
          if (!a.seq.covers(r)) t = a.t.ignore_index;
        }
        if (k >= kRowSlots) ok = mbar_wait(&row_empty[b], static_cast<uint32_t>(k / kRowSlots - 1) & 1, &abort_flag, kErr);
        if (!ok) break;
        row_number[b] = r;
        row_target[b] = t;
        mbar_arrive(&row_full[b]);
        if (r < 0) break;
        mbar_arrive_expect_tx(&asked, 16);
        next_row_ask(&answer, &asked);
        if (t != a.t.ignore_index) {
          const T* p = static_cast<const T*>(a.t.logits) + a.t.map.at(r);
          const int head = static_cast<int>(peel(p, cols)), nvec = (cols - head) / V;
          const int n = (nvec + kChunk - 1) / kChunk, again = want_grad && n > KEEP ? n - KEEP : 0;
          const uint4* pv = reinterpret_cast<const uint4*>(p + head);
          for (int l = 0; l < n + again; ++l) {
            const int c = l < n ? l : l - n;
            if (issued >= SLOTS && !mbar_wait(&empty[pos.slot], pos.phase ^ 1, &abort_flag, kErr + 1)) {
              ok = false;
              break;
            }
            const int vecs = nvec - c * kChunk < kChunk ? nvec - c * kChunk : kChunk;
            mbar_arrive_expect_tx(&full[pos.slot], vecs * 16);
            bulk_load(ring + pos.slot * kChunk, pv + static_cast<int64_t>(c) * kChunk, vecs * 16, &full[pos.slot],
                      l < again ? keep_policy : drop_policy);
            pos.next();
            ++issued;
          }
        }
        if (ok) ok = mbar_wait(&asked, static_cast<uint32_t>(k) & 1, &abort_flag, kErr + 2);
        if (!ok) mbar_wait_drain(&asked, static_cast<uint32_t>(k) & 1, kErr + 2);
        if (ok) {
          r = next_row_read(&answer);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the answer is read before the next overwrites it
        }
      }
      if (!ok) {  // a wait ran out: let the copies in flight land before the block ends
        const int64_t first = issued > SLOTS ? issued - SLOTS : 0;
        for (int64_t q = first; q < issued; ++q)
          mbar_wait_drain(&full[q % SLOTS], static_cast<uint32_t>(q / SLOTS) & 1, kErr + 3);
      }
    }
    __syncwarp();
  } else if (warp == kWarps + 1) {  // ---- scalars
    if (MODE == kPolicy) pdl_wait();
    int64_t live = 0;  // rows with statistics so far
    uint32_t counted = 0;
    for (int64_t k = 0;; ++k) {
      const int b = static_cast<int>(k % kRowSlots);
      const bool here = mbar_wait(&row_full[b], static_cast<uint32_t>(k / kRowSlots) & 1, &abort_flag, kErr + 4);
      if (!__all_sync(0xffffffffu, here)) break;
      const int64_t r = row_number[b], t = row_target[b];
      __syncwarp();
      if (lane == 0) mbar_arrive(&row_empty[b]);
      if (r < 0) break;
      double lp = 0.0, d = 0.0;
      float coef = 0.0f;
      float4 term = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      RowStat st{1.0, 0.0f};
      if (t != a.t.ignore_index) {
        const RowScalars sc = load_scalars<T, MODE>(a, r, t);
        const int h = static_cast<int>(live & 1);
        const bool made = mbar_wait(&stat_full[h], static_cast<uint32_t>(live >> 1) & 1, &abort_flag, kErr + 5);
        if (!__all_sync(0xffffffffu, made)) break;
        st = warp_merge(lane < kWarps ? stat[h][lane] : RowStat{0.0, kLowest}, a.t.k);
        lp = row_logp(a.t, st, sc.target_logit, t);
        if constexpr (MODE == kPolicy) term = policy_term(a, sc, lp, coef);
        d = lp - static_cast<double>(sc.ref);
        __syncwarp();
        if (lane == 0) {
          if (want_grad) {
            row_coef = make_float4(st.m, coef, coef == 0.0f ? 0.0f : -coef / static_cast<float>(st.s), sc.target_logit);
            mbar_arrive(&coef_full);
          }
          mbar_arrive(&stat_empty[h]);
        }
        ++live;
      }
      if (lane == 0) {
        // for the next kernel; by the row, as the block of that number need not run itself
        if (MODE == kStats && a.done && r == 0) *a.done = 0;
        a.t.logps[r] = static_cast<float>(lp);
        if constexpr (MODE == kPolicy) {
          a.terms[r] = term;
          ++counted;
        } else {
          if (a.d) a.d[r] = d;
        }
        if (a.t.row) a.t.row[r] = make_float4(st.m, static_cast<float>(st.s), coef, 0.0f);
      }
    }
    if (MODE == kPolicy && lane == 0) {
      __threadfence();
      last = atomicAdd(a.done, counted) + counted == a.t.rows;
    }
  } else {  // ---- arithmetic
    const int tid = threadIdx.x;
    const uint32_t none = neg_inf_word<T>();
    const Scale k2 = a.t.k;
    Part part(tid);
    RingPos<SLOTS> pos;
    int64_t live = 0;
    bool ok = true;
    for (int64_t k = 0; ok; ++k) {
      const int b = static_cast<int>(k % kRowSlots);
      ok = __all_sync(0xffffffffu,
                      mbar_wait(&row_full[b], static_cast<uint32_t>(k / kRowSlots) & 1, &abort_flag, kErr + 6));
      if (!ok) break;
      const int64_t r = row_number[b], t = row_target[b];
      __syncwarp();
      if (lane == 0) mbar_arrive(&row_empty[b]);
      if (r < 0) break;
      const T* p = static_cast<const T*>(a.t.logits) + a.t.map.at(r);
      const int head = static_cast<int>(peel(p, cols)), nvec = (cols - head) / V;
      const int n = (nvec + kChunk - 1) / kChunk;
      const int keep = !want_grad ? 0 : (n < KEEP ? n : KEEP);
      // elements in front of the first and behind the last vector: at most one a thread
      int edge_at = tid < head ? tid : nvec * V + tid;
      if (edge_at >= cols) edge_at = -1;
      if (t == a.t.ignore_index) {  // zeros, whatever the logits hold
        if (want_grad) {
          T* g = static_cast<T*>(a.grad) + a.gmap.at(r);
          const int ghead = static_cast<int>(peel(g, cols)), gvec = (cols - ghead) / V;
          uint4* gv = reinterpret_cast<uint4*>(g + ghead);
          for (int i = tid; i < gvec; i += CT) __stcs(gv + i, make_uint4(0, 0, 0, 0));
          const int j = tid < ghead ? tid : gvec * V + tid;
          if (j < cols) g[j] = from_f32<T>(0.0f);
        }
        continue;
      }
      const float edge = edge_at >= 0 ? to_f32(p[edge_at]) : -INFINITY;
      part.restart();
      for (int c = 0; c < n && ok; ++c) {
        ok = __all_sync(0xffffffffu, mbar_wait(&full[pos.slot], pos.phase, &abort_flag, kErr + 7));
        const uint4* base = ring + pos.slot * kChunk + tid;
        uint4 v[VECS];
        if (c < n - 1) {
#pragma unroll
          for (int u = 0; u < VECS; ++u) v[u] = base[u * CT];
        } else {
          const int left = nvec - c * kChunk - tid;
#pragma unroll
          for (int u = 0; u < VECS; ++u) v[u] = u * CT < left ? base[u * CT] : make_uint4(none, none, none, none);
        }
        if (c < n - keep) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[pos.slot]);
        }
        float top = part.m;
#pragma unroll
        for (int u = 0; u < VECS; ++u) top = vec_max<T>(v[u], top);
        if (top > part.limit) part.raise(top, k2);
        part.m = top;
        part.add<T, false>(v, k2);
        pos.next();
      }
      RowStat st{part.total(true, k2), part.m};
      if (edge_at >= 0) st = merge(st, one_stat(edge), k2);
      st = warp_merge(st, k2);
      const int h = static_cast<int>(live & 1);
      if (live >= 2)
        ok = ok && __all_sync(0xffffffffu, mbar_wait(&stat_empty[h], static_cast<uint32_t>((live >> 1) - 1) & 1,
                                                     &abort_flag, kErr + 8));
      if (!ok) break;
      if (lane == 0) {
        stat[h][warp] = st;
        mbar_arrive(&stat_full[h]);
      }
      ++live;
      if (!want_grad) continue;

      ok = __all_sync(0xffffffffu, mbar_wait(&coef_full, static_cast<uint32_t>(live - 1) & 1, &abort_flag, kErr + 9));
      if (!ok) break;
      const float4 f = row_coef;
      const float coef = f.y, q = f.z;
      T* g = static_cast<T*>(a.grad) + a.gmap.at(r);
      uint4* gv = reinterpret_cast<uint4*>(g + head) + tid;
      const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
      // the kept chunks n - keep .. n - 1, then 0 .. n - keep - 1 as they arrive again
      RingPos<SLOTS> at = pos;
      at.slot = pos.slot >= keep ? pos.slot - keep : pos.slot - keep + SLOTS;
      for (int l = 0; l < n && ok; ++l) {
        const int c = l < keep ? n - keep + l : l - keep;
        if (l == keep) at = pos;
        if (l >= keep) ok = __all_sync(0xffffffffu, mbar_wait(&full[at.slot], at.phase, &abort_flag, kErr + 10));
        const uint4* base = ring + at.slot * kChunk + tid;
        const int left = nvec - c * kChunk - tid;
        uint4 v[VECS];
        if (c < n - 1) {
#pragma unroll
          for (int u = 0; u < VECS; ++u) v[u] = base[u * CT];
        } else {
#pragma unroll
          for (int u = 0; u < VECS; ++u)
            if (u * CT < left) v[u] = base[u * CT];
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[at.slot]);
        at.next();
        uint4* to = gv + static_cast<int64_t>(c) * kChunk;
        vecs_grad<T, false>(v, f.x, k2, q);
        if (same) {
#pragma unroll
          for (int u = 0; u < VECS; ++u)
            if (u * CT < left) __stcs(to + u * CT, v[u]);
        } else {  // the gradient's rows are off the logits' alignment
#pragma unroll
          for (int u = 0; u < VECS; ++u) store_elements<T>(v[u], u * CT < left ? to + u * CT : nullptr);
        }
      }
      if (n > keep) pos = at;
      if (edge_at >= 0) g[edge_at] = from_f32<T>(q * exp_hw(edge - f.x, k2));
      // the target's element again, by the thread that wrote it
      if (t >= 0 && t < cols) {
        const int j = static_cast<int>(t), i = (j - head) / V;
        if (j == edge_at || (j >= head && i < nvec && i % CT == tid))
          g[j] = from_f32<T>(fmaf(q, exp_hw(f.w - f.x, k2), coef));
      }
    }
  }
  if constexpr (MODE == kPolicy) {
    __syncthreads();
    if (last) add_terms<kWarps + 2>(a);
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

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.0f) + log1pf(expf(-fabsf(x))); }

// loss and its slope over h = beta (D_chosen - D_rejected) - margin.  The functions of h are fp32: their relative error
// of 1e-7 is the pair's alone, while the double ones cost microseconds of latency.
__device__ __forceinline__ void preference_term(const PreferenceArgs& a, double h, double& loss, double& slope) {
  const float e = static_cast<float>(a.smoothing), x = static_cast<float>(h);
  if (a.kind == 0) {
    loss = isnan(x) ? h : static_cast<double>((1.0f - e) * softplus(-x) + e * softplus(x));
    slope = static_cast<double>(e / (1.0f + expf(-x)) - (1.0f - e) / (1.0f + expf(x)));
  } else if (a.kind == 1) {
    loss = isnan(h) ? h : fmax(1.0 - h, 0.0);
    slope = h < 1.0 ? -1.0 : (isnan(h) ? h : 0.0);
  } else {
    loss = (h - 0.5) * (h - 0.5);
    slope = 2.0 * (h - 0.5);
  }
}

// One block per pair, one half of it per sequence: the sums of both, the pair's loss, and the coefficient of their rows
// (of all of them: rows that take no part are the gradient's to leave out).
__global__ void __launch_bounds__(512) preference_pair_kernel(PreferenceArgs a) {
  __shared__ double part[2][8], counted[2][8], smem[16];
  pdl_release();
  const int64_t pairs = a.seq.count / 2, i = blockIdx.x;
  const int side = threadIdx.x >> 8, lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 7, tid = threadIdx.x & 255;
  const int64_t s = i + side * pairs;
  const int64_t lo = a.seq.begin(s, a.t.rows), hi = a.seq.begin(s + 1, a.t.rows);
  double c = 0.0, x = 0.0;
  if (a.average)
    for (int64_t r = lo + tid; r < hi; r += 256) c += a.t.targets[r] != a.t.ignore_index ? 1.0 : 0.0;
  pdl_wait();
  for (int64_t r = lo + tid; r < hi; r += 256) x += __ldcg(a.d + r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if (lane == 0) {
    part[side][warp] = x;
    counted[side][warp] = c;
  }
  __syncthreads();
  double d[2] = {0.0, 0.0}, n[2] = {0.0, 0.0};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    for (int w = 0; w < 8; ++w) {
      d[q] += part[q][w];
      n[q] += counted[q][w];
    }
    if (a.average) d[q] = n[q] > 0.0 ? d[q] / n[q] : 0.0;
  }
  double loss, slope;
  preference_term(a, a.beta * (d[0] - d[1]) - a.margin, loss, slope);
  double k = slope * a.beta * a.t.inv_temp / static_cast<double>(pairs);
  if (a.average && n[side] > 0.0) k /= n[side];
  for (int64_t r = lo + tid; r < hi; r += 256) a.t.row[r].z = static_cast<float>(side ? -k : k);
  if (threadIdx.x == 0) {
    a.chosen[i] = static_cast<float>(a.beta * d[0]);
    a.rejected[i] = static_cast<float>(a.beta * d[1]);
    a.sums[i] = loss;
  }
  if (last_block(a.done, gridDim.x)) {
    double t = 0.0;
    for (int64_t b = threadIdx.x; b < gridDim.x; b += 512) t += __ldcg(a.sums + b);
    t = block_sum(t, smem);
    if (threadIdx.x == 0) *a.out = static_cast<float>(t / static_cast<double>(pairs));
  }
}

// ---- gradient of the logits from kept row statistics ---------------------------------------------------
struct GradArgs {
  TokenArgs t;
  const float* slope;   // [rows] d loss / d lp, or null: the coefficient is row[r].z
  const float* factor;  // one number that multiplies the gradient before it is rounded, or null
  void* grad;
  RowMap gmap;
  int32_t parts;       // blocks per row
};

// Bound by memory: 2048 x 151936 bf16 (a quarter of the rows zero) 175 us, 6.2 TB/s.
//
// `parts` blocks per row, the last rows first: the pass before read them last, and what of them is still in L2 need
// not come from memory again.  A row whose coefficient is zero (ignored, or a flat loss) is written as zeros and not
// read: what its logits hold does not reach the gradient.  The factor multiplies each element last, so that a factor of 1
// leaves the bits that the policy kernels write.  `grad` may be the logits themselves: then one block writes
// a row (parts is 1), after it has read the target's logit.
template <typename T>
__global__ void __launch_bounds__(256) logit_grad_kernel(GradArgs a) {
  constexpr int V = kVec16<T>, U = 4;
  const int64_t r = a.t.rows - 1 - blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const int64_t t = a.t.targets[r];
  pdl_wait();
  const float4 st = __ldcg(a.t.row + r);
  const bool in = t >= 0 && t < a.t.cols;
  float c = t == a.t.ignore_index ? 0.0f : (a.slope ? a.slope[r] * static_cast<float>(a.t.inv_temp) : st.z);
  if (!in && c != 0.0f) c = NAN;  // as the row's log-probability
  const T* p = static_cast<const T*>(a.t.logits) + a.t.map.at(r);
  T* g = static_cast<T*>(a.grad) + a.gmap.at(r);
  const float q = -c / st.y, f = a.factor ? __ldg(a.factor) : 1.0f;
  const bool zero = c == 0.0f;
  float at_t = 0.0f;
  if (!zero && in) at_t = fmaf(q, exp_hw(to_f32(p[t]) - st.x, a.t.k), c) * f;
  if (p == g) __syncthreads();
  const bool same = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  const int64_t head = same ? peel(g, a.t.cols) : a.t.cols;
  const int64_t nvec = (a.t.cols - head) / V, tail = head + nvec * V;
  const int64_t per = (nvec + a.parts - 1) / a.parts;
  const int64_t end = per * (part + 1) < nvec ? per * (part + 1) : nvec;
  const uint4* pv = reinterpret_cast<const uint4*>(p + head);
  uint4* gv = reinterpret_cast<uint4*>(g + head);
  const int64_t tv = t >= head && t < tail ? (t - head) / V : -1;
  for (int64_t i0 = per * part + threadIdx.x; i0 < end; i0 += 256 * U) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!zero && i0 + u * 256 < end) raw[u] = load_stream(pv + i0 + u * 256);
    if (zero) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = make_uint4(0, 0, 0, 0);
    } else {
      vecs_grad<T, true>(raw, st.x, a.t.k, q, f);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * 256 < end) __stcs(gv + i0 + u * 256, raw[u]);
  }
  auto one = [&](int64_t j) {
    g[j] = from_f32<T>(zero ? 0.0f : (j == t ? at_t : q * exp_hw(to_f32(p[j]) - st.x, a.t.k) * f));
  };
  // the target's element again, by the thread that wrote it
  if (!zero && tv >= per * part && tv < end && (tv - per * part) % 256 == threadIdx.x) g[t] = from_f32<T>(at_t);
  if (same) {  // the few elements in front of and behind the vectors
    const int64_t j = static_cast<int64_t>(threadIdx.x) < head ? threadIdx.x : tail + (threadIdx.x - head);
    if (part == 0 && j < a.t.cols) one(j);
  } else {     // rows of the two off each other's alignment
    for (int64_t j = static_cast<int64_t>(part) * 256 + threadIdx.x; j < a.t.cols; j += 256ll * a.parts) one(j);
  }
}

// ---- launchers -------------------------------------------------------------------------------------
template <typename T, int CT, int VECS, int SLOTS, int KEEP, int MODE>
cudaError_t launch_ring(const RowArgs& a, bool early, cudaStream_t stream) {
  auto fn = token_ring_kernel<T, CT, VECS, SLOTS, KEEP, MODE>;
  constexpr size_t kSmem = ring_bytes<CT, VECS, SLOTS>();
  // the shared-memory cap is a function attribute of each device
  static std::atomic<uint64_t> configured[2] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 0 || device >= 128) return cudaErrorInvalidDevice;
  const uint64_t bit = uint64_t(1) << (device & 63);
  if (!(configured[device >> 6].load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmem));
    if (e != cudaSuccess) return e;
    configured[device >> 6].fetch_or(bit, std::memory_order_release);
  }
  return launch_kernel(fn, a.t.rows, CT + 64, 1, early, a, stream, kSmem);
}

// The kernel for `rows` rows of `vecs` 16-byte vectors (16384 rows on one B200 where nothing else is said; "with gradient":
// the policy loss):
//   up to 256 vectors   a warp per row, in registers (1000 fp32: 13 us, with gradient 54; a block of 128 per row 37, 108)
//   up to 1024          a warp per row that reads it twice (2500 fp32: 33 us; the ring 66); with gradient up to 800, as
//                       the third reading then leaves the caches (3000 fp32: 108 us, the ring 134; 4000: 144, the ring 135;
//                       5000 bf16: 102, the ring 171)
//   longer              the ring: blocks of 128, 4 an SM, up to 150 KB a row (8192 rows of 64 KB: 118 us; blocks of 256 129);
//                       of 256, 2 an SM, up to 400 KB (2048 rows of 304 KB, a quarter ignored: 106 us, with gradient 229;
//                       blocks of 128 114, 274; of 512 107, 228); of 512 beyond (608 KB: 135 us, 411; of 256 140, 483)
// With too few rows for one each to fill the SMs, a row goes to a block or a cluster of up to 8 blocks of 512 that
// hold it in registers (10 vectors a thread, of which the policy kernel spills 400 bytes; longer rows are read twice).
template <typename T, int MODE>
cudaError_t launch_rows(const RowArgs& a, bool early, cudaStream_t stream) {
  const int64_t rows = a.t.rows, vecs = (a.t.cols + kVec16<T> - 1) / kVec16<T>;
  const int64_t fours = (rows + 3) / 4;
  if (vecs <= 64) return launch_kernel(token_row_kernel<T, 32, 2, true, MODE>, fours, 128, 1, early, a, stream);
  if (rows >= 192) {
    if (vecs <= 256) return launch_kernel(token_row_kernel<T, 32, 8, true, MODE>, fours, 128, 1, early, a, stream);
    if (vecs <= (MODE == kPolicy ? 800 : 1024) && rows >= 8 * 148)
      return launch_kernel(token_row_kernel<T, 32, 4, false, MODE>, fours, 128, 1, early, a, stream);
    if (vecs <= 9600) return launch_ring<T, 128, 4, 6, 4, MODE>(a, early, stream);
    if (vecs <= 25600) return launch_ring<T, 256, 4, 6, 4, MODE>(a, early, stream);
    return launch_ring<T, 512, 4, 6, 4, MODE>(a, early, stream);
  }
  if (vecs <= 128 * 3) return launch_kernel(token_row_kernel<T, 128, 3, true, MODE>, rows, 128, 1, early, a, stream);
  int cluster = 1;
  while (cluster < kMaxCluster && (vecs > 512 * 10 * cluster || (rows * cluster < 148 && vecs > 1024 * cluster))) cluster *= 2;
  const int64_t need = (vecs + 512 * cluster - 1) / (512 * cluster), blocks = rows * cluster;
  if (need <= 3) return launch_kernel(token_row_kernel<T, 512, 3, true, MODE>, blocks, 512, cluster, early, a, stream);
  if (need <= 10) return launch_kernel(token_row_kernel<T, 512, 10, true, MODE>, blocks, 512, cluster, early, a, stream);
  return launch_kernel(token_row_kernel<T, 512, 4, false, MODE>, blocks, 512, cluster, early, a, stream);
}

template <typename T>
cudaError_t token_logps_t(const RowArgs& a, cudaStream_t stream) {
  return launch_rows<T, kStats>(a, false, stream);
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
  cudaError_t e = launch_rows<T, kStats>(rows, false, stream);
  if (e == cudaSuccess) e = launch_kernel(preference_pair_kernel, a.seq.count / 2, 512, 1, true, a, stream);
  return e != cudaSuccess || !g.grad ? e : logit_grad_t<T>(g, true, stream);
}

}  // namespace mib
