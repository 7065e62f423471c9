// C ABI of the language-model tuning operators (declared in include/memintelli_b200.h): argument checks, workspace
// layout and launches.
#include <algorithm>
#include <cmath>
#include <new>
#include <string>
#include <vector>

#include "kernels.cuh"

namespace {

int fail(int code, const char* msg) { return mib::record_error(code, msg); }
int fail(int code, const std::string& msg) { return mib::record_error(code, msg.c_str()); }
int cuda_fail(cudaError_t e, const char* what) {
  return fail(MIB_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

bool known_dtype(int32_t d) { return d == MIB_F32 || d == MIB_BF16 || d == MIB_F16; }
size_t dtype_size(int32_t d) { return d == MIB_F32 ? 4 : 2; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t index_size(int32_t is64) { return is64 ? 8 : 4; }

// Calls fn with a value of the element type.
template <typename F>
cudaError_t with_dtype(int32_t d, F fn) {
  if (d == MIB_F32) return fn(float());
  if (d == MIB_BF16) return fn(__nv_bfloat16());
  return fn(__half());
}

constexpr int64_t kMaxRows = int64_t(1) << 31;

mib::RowMap row_map(const mib_out_layout& l) { return mib::RowMap{l.rows_per_group, l.group_stride, l.row_stride}; }

int check_grad(const mib_token_rows* t, const void* grad) {
  return aligned(grad, dtype_size(t->dtype)) ? MIB_OK : fail(MIB_ERR_PARAM, "misaligned gradient");
}

int check_rows_layout(const mib_out_layout* l, int64_t rows, int64_t cols, const char* what) {
  if (!l) return fail(MIB_ERR_PARAM, std::string(what) + " layout is NULL");
  if (l->rows_per_group < 1 || l->col_stride != 1) 
    return fail(MIB_ERR_SHAPE, std::string(what) + " needs unit column stride and rows in groups");
  if (rows > 1 && l->rows_per_group > 1 && l->row_stride < cols)
    return fail(MIB_ERR_SHAPE, std::string(what) + " rows overlap");
  return MIB_OK;
}

int check_token_rows(const mib_token_rows* t) {
  if (!t || !t->logits || !t->targets) return fail(MIB_ERR_PARAM, "NULL logits or targets");
  if (!known_dtype(t->dtype)) return fail(MIB_ERR_UNSUPPORTED, "logits must be fp32, bf16 or fp16");
  if (t->rows < 1 || t->cols < 1) return fail(MIB_ERR_SHAPE, "logits must be non-empty");
  if (t->rows >= kMaxRows / 1024 || t->cols >= kMaxRows)
    return fail(MIB_ERR_SHAPE, "too many rows (2^21 or more) or columns (2^31 or more)");
  if (!(t->temperature >= 1e-30) || !(t->temperature < 1e30))  // its inverse, in fp32 too
    return fail(MIB_ERR_PARAM, "temperature must be positive, from 1e-30 to 1e30");
  if (!aligned(t->logits, dtype_size(t->dtype)) || !aligned(t->targets, index_size(t->targets_i64)) ||
      !aligned(t->cu_seqlens, index_size(t->cu_i64)))
    return fail(MIB_ERR_PARAM, "misaligned logits, targets or row offsets");
  return check_rows_layout(&t->layout, t->rows, t->cols, "logits");
}

int check_sequences(const mib_token_rows* t) {
  if (t->sequences < 0 || t->sequences >= kMaxRows / 2) return fail(MIB_ERR_SHAPE, "invalid number of sequences");
  if (t->sequences > 0 && !t->cu_seqlens && t->rows_per_sequence < 1)
    return fail(MIB_ERR_PARAM, "sequences need their row offsets or a common length");
  return MIB_OK;
}

// Workspace of a loss: row coefficients and terms, per-pair sums, counters.
struct TokenSpace {
  int64_t row, terms, counts, seq_w, sums, done, bytes;
};
TokenSpace token_space(int64_t rows, int64_t sequences) {
  TokenSpace s;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  s.row = take(rows * static_cast<int64_t>(sizeof(float4)));
  s.terms = take(rows * static_cast<int64_t>(sizeof(float4)));
  s.counts = take(mib::kCountBlocks * 4);
  s.seq_w = take(sequences * 4);
  s.sums = take(sequences * 8);
  s.done = take(4);
  s.bytes = at;
  return s;
}

mib::TokenArgs token_args(const mib_token_rows* t, float* logps, void* row) {
  mib::TokenArgs a{};
  a.logits = t->logits;
  a.map = row_map(t->layout);
  a.rows = t->rows;
  a.cols = t->cols;
  a.targets = mib::IntList{t->targets, t->targets_i64};
  a.ignore_index = t->ignore_index;
  a.k.k = 1.4426950408889634 / t->temperature;
  a.k.hi = static_cast<float>(a.k.k);
  if (static_cast<double>(a.k.hi) >= a.k.k) a.k.hi = std::nextafter(a.k.hi, 0.0f);
  a.k.lo = static_cast<float>(a.k.k - static_cast<double>(a.k.hi));
  a.k.unit = static_cast<float>(1.0 / a.k.k);
  a.inv_temp = 1.0 / t->temperature;
  a.logps = logps;
  a.row = static_cast<float4*>(row);
  return a;
}

mib::SeqList seq_list(const mib_token_rows* t) {
  return mib::SeqList{mib::IntList{t->cu_seqlens, t->cu_i64}, t->sequences, t->cu_seqlens ? 0 : t->rows_per_sequence};
}

// Refuses tensors of which one that is written shares memory with another that is read or written (a pair in[i], out[i]
// may be the same tensor): the blocks that scale them run in no order.
int check_apart(const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
                const int32_t* out_dtype, int32_t count) {
  struct Span {
    uintptr_t first, end;
    bool written;
  };
  std::vector<Span> spans;
  try {
    spans.reserve(2 * static_cast<size_t>(count));
  } catch (const std::bad_alloc&) {
    return fail(MIB_ERR_PARAM, "out of host memory");
  }
  for (int32_t i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    auto add = [&](const void* p, int32_t dtype, bool written) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(p);
      spans.push_back(Span{at, at + static_cast<uintptr_t>(numel[i]) * dtype_size(dtype), written});
    };
    add(out[i], out_dtype[i], true);
    if (in[i] != out[i] || in_dtype[i] != out_dtype[i]) add(in[i], in_dtype[i], false);
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.first < b.first; });
  uintptr_t any = 0, written = 0;  // ends of the spans so far
  for (const Span& s : spans) {
    if (s.first < (s.written ? any : written)) return fail(MIB_ERR_PARAM, "tensors to clip overlap in memory");
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return MIB_OK;
}

int check_space(void* ws, int64_t have, int64_t need) {
  if (!ws || have < need) return fail(MIB_ERR_PARAM, "workspace is missing or too small");
  if (reinterpret_cast<uintptr_t>(ws) % 256) return fail(MIB_ERR_PARAM, "workspace must be 256-byte aligned");
  return MIB_OK;
}

}  // namespace

extern "C" {

int mib_embedding_lookup(const void* ids, int32_t ids_i64, int64_t n, const void* table, int32_t dtype, int64_t vocab,
                         int64_t hidden, int64_t ld_table, float scale, void* out, cudaStream_t stream) {
  if (!ids || !table || !out) return fail(MIB_ERR_PARAM, "NULL buffer");
  if (!known_dtype(dtype)) return fail(MIB_ERR_UNSUPPORTED, "the table must be fp32, bf16 or fp16");
  if (n < 1 || vocab < 1 || hidden < 1 || ld_table < hidden) return fail(MIB_ERR_SHAPE, "invalid embedding shape");
  if (n >= kMaxRows || hidden > (1 << 24)) return fail(MIB_ERR_SHAPE, "too many tokens or columns");
  if (!aligned(ids, index_size(ids_i64)) || !aligned(table, dtype_size(dtype)) || !aligned(out, dtype_size(dtype)))
    return fail(MIB_ERR_PARAM, "misaligned buffer");
  cudaError_t e = with_dtype(dtype, [&](auto v) {
    return mib::lookup_t<decltype(v)>(mib::IntList{ids, ids_i64}, n, table, vocab, hidden, ld_table, scale, out, stream);
  });
  if (e != cudaSuccess) return cuda_fail(e, "embedding_lookup launch");
  return MIB_OK;
}

int mib_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t hidden, int64_t* bytes_out) {
  if (!bytes_out) return fail(MIB_ERR_PARAM, "NULL argument");
  if (n < 1 || vocab < 1 || hidden < 1) return fail(MIB_ERR_SHAPE, "invalid embedding shape");
  *bytes_out = align256(static_cast<int64_t>(mib::embed_plan(n, vocab, hidden).bytes));
  return MIB_OK;
}

int mib_embedding_grad(const void* ids, int32_t ids_i64, int64_t n, const void* grad, int32_t grad_dtype,
                       int64_t ld_grad, int64_t vocab, int64_t hidden, float scale, int64_t padding_idx, void* out,
                       int32_t out_dtype, int64_t ld_out, int32_t accumulate, void* workspace, int64_t workspace_bytes,
                       cudaStream_t stream) {
  if (!ids || !grad || !out) return fail(MIB_ERR_PARAM, "NULL buffer");
  if (!known_dtype(grad_dtype) || (out_dtype != grad_dtype && out_dtype != MIB_F32))
    return fail(MIB_ERR_UNSUPPORTED, "gradients are fp32, bf16 or fp16; the table's gradient has that type or fp32");
  if (n < 1 || vocab < 1 || hidden < 1 || ld_grad < hidden || ld_out < hidden)
    return fail(MIB_ERR_SHAPE, "invalid embedding shape");
  if (n >= kMaxRows || vocab >= kMaxRows || hidden > (1 << 23)) return fail(MIB_ERR_SHAPE, "too many tokens, rows or columns");
  if (!aligned(ids, index_size(ids_i64)) || !aligned(grad, dtype_size(grad_dtype)) || !aligned(out, dtype_size(out_dtype)))
    return fail(MIB_ERR_PARAM, "misaligned buffer");
  if (int r = check_space(workspace, workspace_bytes, static_cast<int64_t>(mib::embed_plan(n, vocab, hidden).bytes))) return r;
  mib::EmbedGradArgs a{};
  a.n = n;
  a.vocab = vocab;
  a.hidden = hidden;
  a.ld_grad = ld_grad;
  a.ld_out = ld_out;
  a.scale = scale;
  a.accumulate = accumulate;
  a.grad = grad;
  a.out = out;
  mib::SortArgs s{};
  s.ids = mib::IntList{ids, ids_i64};
  s.n = n;
  s.vocab = vocab;
  s.padding = padding_idx;
  cudaError_t e = with_dtype(grad_dtype, [&](auto v) {
    using G = decltype(v);
    return out_dtype == MIB_F32 ? mib::embed_grad_t<G, float>(a, s, workspace, stream)
                                : mib::embed_grad_t<G, G>(a, s, workspace, stream);
  });
  if (e != cudaSuccess) return cuda_fail(e, "embedding_grad launch");
  return MIB_OK;
}

int mib_token_loss_workspace(int64_t rows, int64_t cols, int64_t sequences, int64_t* bytes_out) {
  if (!bytes_out) return fail(MIB_ERR_PARAM, "NULL argument");
  if (rows < 1 || cols < 1 || sequences < 0) return fail(MIB_ERR_SHAPE, "invalid logit block");
  *bytes_out = token_space(rows, sequences).bytes;
  return MIB_OK;
}

int mib_token_logps(const mib_token_rows* t, float* logps, void* stats, cudaStream_t stream) {
  if (int r = check_token_rows(t)) return r;
  if (!logps || reinterpret_cast<uintptr_t>(stats) % 16) return fail(MIB_ERR_PARAM, "NULL or misaligned buffer");
  mib::RowArgs a{};
  a.t = token_args(t, logps, stats);
  cudaError_t e = with_dtype(t->dtype, [&](auto v) { return mib::token_logps_t<decltype(v)>(a, stream); });
  if (e != cudaSuccess) return cuda_fail(e, "token_logps launch");
  return MIB_OK;
}

int mib_token_logps_grad(const mib_token_rows* t, const void* stats, const float* grad_logps, void* grad,
                         const mib_out_layout* grad_layout, cudaStream_t stream) {
  if (int r = check_token_rows(t)) return r;
  if (!stats || !grad_logps || !grad || reinterpret_cast<uintptr_t>(stats) % 16)
    return fail(MIB_ERR_PARAM, "NULL or misaligned buffer");
  if (int r = check_rows_layout(grad_layout, t->rows, t->cols, "gradient")) return r;
  if (int r = check_grad(t, grad)) return r;
  mib::GradArgs g{};
  g.t = token_args(t, nullptr, const_cast<void*>(stats));
  g.slope = grad_logps;
  g.grad = grad;
  g.gmap = row_map(*grad_layout);
  cudaError_t e = with_dtype(t->dtype, [&](auto v) { return mib::logit_grad_t<decltype(v)>(g, false, stream); });
  if (e != cudaSuccess) return cuda_fail(e, "token_logps_grad launch");
  return MIB_OK;
}

int mib_policy_loss(const mib_token_rows* t, const mib_policy_spec* spec, const float* old_logps,
                    const float* advantages, const float* ref_logps, float* loss_kl_clip, float* logps, void* grad,
                    const mib_out_layout* grad_layout, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  if (int r = check_token_rows(t)) return r;
  if (int r = check_sequences(t)) return r;
  if (!spec || !old_logps || !advantages || !loss_kl_clip || !logps) return fail(MIB_ERR_PARAM, "NULL buffer");
  if (!(spec->clip_low >= 0.0) || !(spec->clip_low <= 1.0) || !(spec->clip_high >= 0.0))
    return fail(MIB_ERR_PARAM, "clip bounds must be non-negative, the lower one at most 1");
  if (!(spec->kl_coef >= 0.0)) return fail(MIB_ERR_PARAM, "kl_coef must be non-negative");
  if (spec->kl_coef > 0.0 && !ref_logps) return fail(MIB_ERR_PARAM, "the KL term needs reference log-probabilities");
  if (spec->reduction < 0 || spec->reduction > 2) return fail(MIB_ERR_PARAM, "unknown reduction");
  if ((spec->reduction == 1 || spec->adv_per_sequence) && t->sequences < 1)
    return fail(MIB_ERR_PARAM, "a sequence mean or advantages per sequence need the sequences");
  if (grad) {
    if (int r = check_rows_layout(grad_layout, t->rows, t->cols, "gradient")) return r;
    if (int r = check_grad(t, grad)) return r;
  }
  const TokenSpace s = token_space(t->rows, t->sequences);
  if (int r = check_space(workspace, workspace_bytes, s.bytes)) return r;
  char* ws = static_cast<char*>(workspace);
  mib::RowArgs a{};
  a.t = token_args(t, logps, grad ? nullptr : ws + s.row);
  a.seq = seq_list(t);
  a.old_logps = old_logps;
  a.advantages = advantages;
  a.ref_logps = ref_logps;
  a.adv_per_seq = spec->adv_per_sequence;
  a.reduction = spec->reduction;
  a.lo = static_cast<float>(1.0 - spec->clip_low);
  a.hi = static_cast<float>(1.0 + spec->clip_high);
  a.kl_coef = static_cast<float>(spec->kl_coef);
  const int64_t want = spec->reduction == 1 ? (t->sequences + 7) / 8 : (spec->reduction == 0 ? (t->rows + 255) / 256 : 1);
  a.count_blocks = static_cast<int32_t>(want < mib::kCountBlocks ? want : mib::kCountBlocks);
  a.counts = reinterpret_cast<int32_t*>(ws + s.counts);
  a.seq_w = reinterpret_cast<float*>(ws + s.seq_w);
  a.done = reinterpret_cast<uint32_t*>(ws + s.done);
  a.terms = reinterpret_cast<float4*>(ws + s.terms);
  a.out = loss_kl_clip;
  a.grad = grad;
  if (grad) a.gmap = row_map(*grad_layout);
  cudaError_t e = with_dtype(t->dtype, [&](auto v) { return mib::policy_loss_t<decltype(v)>(a, stream); });
  if (e != cudaSuccess) return cuda_fail(e, "policy_loss launch");
  return MIB_OK;
}

int mib_preference_loss(const mib_token_rows* t, const mib_preference_spec* spec, const float* ref_logps, float* loss,
                        float* chosen_rewards, float* rejected_rewards, float* logps, void* grad,
                        const mib_out_layout* grad_layout, void* workspace, int64_t workspace_bytes,
                        cudaStream_t stream) {
  if (int r = check_token_rows(t)) return r;
  if (int r = check_sequences(t)) return r;
  if (!spec || !loss || !chosen_rewards || !rejected_rewards || !logps) return fail(MIB_ERR_PARAM, "NULL buffer");
  if (t->sequences < 2 || t->sequences % 2) return fail(MIB_ERR_SHAPE, "preference pairs need an even number of sequences");
  if (spec->kind < 0 || spec->kind > 2) return fail(MIB_ERR_PARAM, "unknown preference loss");
  if (!(spec->label_smoothing >= 0.0) || !(spec->label_smoothing <= 0.5) || (spec->kind != 0 && spec->label_smoothing != 0.0))
    return fail(MIB_ERR_PARAM, "label smoothing must be in [0, 0.5], and 0 except for the sigmoid loss");
  if (!(spec->beta > 0.0) || !(spec->beta < 1e30) || !(std::fabs(spec->margin) < 1e30))
    return fail(MIB_ERR_PARAM, "beta must be positive and the margin finite");
  if (grad) {
    if (int r = check_rows_layout(grad_layout, t->rows, t->cols, "gradient")) return r;
    if (int r = check_grad(t, grad)) return r;
  }
  const TokenSpace s = token_space(t->rows, t->sequences);
  if (int r = check_space(workspace, workspace_bytes, s.bytes)) return r;
  char* ws = static_cast<char*>(workspace);
  mib::RowArgs rows{};
  rows.t = token_args(t, logps, ws + s.row);
  rows.seq = seq_list(t);
  rows.ref_logps = ref_logps;
  rows.done = reinterpret_cast<uint32_t*>(ws + s.done);
  rows.d = reinterpret_cast<double*>(ws + s.terms);
  mib::PreferenceArgs a{};
  a.t = rows.t;
  a.seq = rows.seq;
  a.d = rows.d;
  a.kind = spec->kind;
  a.average = spec->average;
  a.beta = spec->beta;
  a.smoothing = spec->label_smoothing;
  a.margin = spec->margin;
  a.done = rows.done;
  a.sums = reinterpret_cast<double*>(ws + s.sums);
  a.chosen = chosen_rewards;
  a.rejected = rejected_rewards;
  a.out = loss;
  mib::GradArgs g{};
  g.t = rows.t;
  g.grad = grad;
  if (grad) g.gmap = row_map(*grad_layout);
  cudaError_t e = with_dtype(t->dtype, [&](auto v) { return mib::preference_loss_t<decltype(v)>(rows, a, g, stream); });
  if (e != cudaSuccess) return cuda_fail(e, "preference_loss launch");
  return MIB_OK;
}

int mib_loss_grad(const mib_token_rows* t, const void* workspace, int64_t workspace_bytes, const float* factor, void* grad,
                  const mib_out_layout* grad_layout, cudaStream_t stream) {
  if (int r = check_token_rows(t)) return r;
  if (int r = check_sequences(t)) return r;
  if (!grad) return fail(MIB_ERR_PARAM, "NULL buffer");
  if (int r = check_rows_layout(grad_layout, t->rows, t->cols, "gradient")) return r;
  if (int r = check_grad(t, grad)) return r;
  if (!aligned(factor, 4)) return fail(MIB_ERR_PARAM, "misaligned factor");
  const TokenSpace s = token_space(t->rows, t->sequences);
  if (int r = check_space(const_cast<void*>(workspace), workspace_bytes, s.bytes)) return r;
  mib::GradArgs g{};
  g.t = token_args(t, nullptr, static_cast<char*>(const_cast<void*>(workspace)) + s.row);
  g.factor = factor;
  g.grad = grad;
  g.gmap = row_map(*grad_layout);
  cudaError_t e = with_dtype(t->dtype, [&](auto v) { return mib::logit_grad_t<decltype(v)>(g, false, stream); });
  if (e != cudaSuccess) return cuda_fail(e, "loss_grad launch");
  return MIB_OK;
}

int mib_clip_grad_norm_workspace(int32_t count, int64_t* bytes_out) {
  if (!bytes_out) return fail(MIB_ERR_PARAM, "NULL argument");
  if (count < 0) return fail(MIB_ERR_SHAPE, "negative tensor count");
  const int64_t launches = (static_cast<int64_t>(count) + mib::kClipTensors - 1) / mib::kClipTensors;
  *bytes_out = align256((launches + 1) * mib::kClipBlocks * 8);
  return MIB_OK;
}

int mib_clip_grad_norm(const void* const* in, void* const* out, const int64_t* numel, const int32_t* in_dtype,
                       const int32_t* out_dtype, int32_t count, int32_t norm_type, float max_norm, float eps,
                       float* norm, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  if (!norm || count < 0 || (count > 0 && (!in || !numel || !in_dtype || (out && !out_dtype))))
    return fail(MIB_ERR_PARAM, "NULL buffer");
  if (norm_type < 0 || norm_type > 2) return fail(MIB_ERR_UNSUPPORTED, "norm_type must be 1, 2 or infinity");
  if (out && (!(max_norm >= 0.0f) || !(eps >= 0.0f))) return fail(MIB_ERR_PARAM, "max_norm must be non-negative");
  bool in_place = out != nullptr;
  for (int32_t i = 0; i < count; ++i) {
    if (numel[i] < 0 || numel[i] > (int64_t(1) << 42)) return fail(MIB_ERR_SHAPE, "invalid tensor size");
    if (!known_dtype(in_dtype[i]) || (out && !known_dtype(out_dtype[i])))
      return fail(MIB_ERR_UNSUPPORTED, "gradients must be fp32, bf16 or fp16");
    if (numel[i] > 0 && (!in[i] || (out && !out[i]))) return fail(MIB_ERR_PARAM, "NULL tensor");
    if (!aligned(in[i], dtype_size(in_dtype[i])) || (out && !aligned(out[i], dtype_size(out_dtype[i]))))
      return fail(MIB_ERR_PARAM, "misaligned tensor");
    if (out && (out[i] != in[i] || out_dtype[i] != in_dtype[i])) in_place = false;
  }
  if (out)
    if (int r = check_apart(in, out, numel, in_dtype, out_dtype, count)) return r;
  int64_t need = 0;
  if (int r = mib_clip_grad_norm_workspace(count, &need)) return r;
  if (int r = check_space(workspace, workspace_bytes, need)) return r;
  mib::ClipState s{};
  s.part = static_cast<double*>(workspace);
  s.max_norm = max_norm;
  s.eps = eps;
  s.norm = norm;
  // calls f with the norm's kind as a compile-time constant
  auto by_norm = [&](auto f) {
    if (norm_type == 2) return f(std::integral_constant<int, 2>());
    if (norm_type == 1) return f(std::integral_constant<int, 1>());
    return f(std::integral_constant<int, 0>());
  };
  const cudaError_t ok = cudaSuccess;
  cudaError_t e = ok;
  int launches = 0;
  int r = mib::clip_tables(in, out, numel, in_dtype, out_dtype, count, [&](const mib::ClipTable& t) {
    s.part_first = s.part_total;
    s.part_total += static_cast<int32_t>(mib::clip_grid(t));
    if (static_cast<int64_t>(s.part_total) * 8 > need) return fail(MIB_ERR_SHAPE, "tensor list too large");
    e = by_norm([&](auto p) { return mib::clip_norm_p<decltype(p)::value>(t, s, stream); });
    ++launches;
    return e == ok ? MIB_OK : cuda_fail(e, "clip_grad_norm launch");
  });
  if (r) return r;
  if (!out || launches == 0) {
    e = by_norm([&](auto p) { return mib::clip_finish_p<decltype(p)::value>(s, stream); });
    return e == ok ? MIB_OK : cuda_fail(e, "clip_grad_norm launch");
  }
  // the scaling may start early only behind the one launch that it waits for
  bool early = launches == 1;
  return mib::clip_tables(in, out, numel, in_dtype, out_dtype, count, [&](const mib::ClipTable& t) {
    e = by_norm([&](auto p) { return mib::clip_scale_p<decltype(p)::value>(t, s, in_place, early, stream); });
    early = false;
    return e == ok ? MIB_OK : cuda_fail(e, "clip_grad_norm launch");
  });
}

}  // extern "C"
