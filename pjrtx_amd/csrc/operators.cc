// Lowering and dispatch of the operator custom calls:
//
//   pjrtx.paged_attention(q [B, Hq, D], k_pages, v_pages [P, Hkv, S, D],
//       page_table s32 [B, M], lengths s32 [B]) -> [B, Hq, D]
//       {scale = 1/sqrt(D), window = 0}
//   pjrtx.paged_append(k_pages, v_pages [P, Hkv, S, D], k_new, v_new
//       [N, Hkv, D], slots s32|s64 [N]) -> (k_pages, v_pages)
//   pjrtx.add_rms_norm(x [..., D], [residual [..., D],] gain [D]) ->
//       (y | y s8, scales f32 [...] [, sum]) {eps = 1e-5}
//   pjrtx.add_rms_norm_grad(dy, [dsum,] sum [..., D], gain [D]) ->
//       (dx, dgain) {eps = 1e-5}
//   pjrtx.token_logprobs(logits [N, V], tokens s32|s64 [N]) -> (logprobs,
//       entropy, lse f32 [N] [, top_logprobs f32, top_tokens s32 [N, K]])
//   pjrtx.token_logprobs_grad(logits, tokens, lse, entropy, d_logprobs,
//       d_entropy f32 [N]) -> d_logits
//
// The configuration is the call's backend_config dictionary, as
// jax.ffi.ffi_call prints its attributes. What the operands and results
// already say (8-bit rows, top_k) is not repeated in it.
#include "operators.h"

#include <cmath>
#include <cstdlib>
#include <set>

#include "kernels/operators.h"

namespace pjrtx {

namespace {

// Workgroups a launch may have: 256 threads each within 2^32.
constexpr int64_t kMaxGroups = (int64_t(1) << 24) - 1;
constexpr int64_t kMaxIndex = (int64_t(1) << 31) - 1;

bool is_operator_float(DType t) { return t == DType::kF32 || t == DType::kF16 || t == DType::kBF16; }
bool is_index(DType t) { return t == DType::kS32 || t == DType::kS64; }

class CallArgs {
 public:
  CallArgs(const Program& prog, const Op& op) : prog_(prog), op_(op) {}
  const TensorType& in(size_t i) const { return prog_.type(op_.operands.at(i)); }
  const TensorType& out(size_t i) const { return prog_.type(op_.results.at(i)); }
  size_t ins() const { return op_.operands.size(); }
  size_t outs() const { return op_.results.size(); }
  void need(bool ok, const std::string& what) const {
    PJRTX_CHECK(ok, Code::kInvalidArgument, op_.target + ": " + what);
  }
  void within(bool ok, const std::string& what) const {
    PJRTX_CHECK(ok, Code::kUnimplemented, op_.target + ": " + what);
  }
  void known_keys(const std::set<std::string>& keys) const {
    for (const auto& [k, v] : op_.config) need(keys.count(k) > 0, "unknown attribute '" + k + "'");
  }
  double number(const char* key, double dflt) const {
    auto it = op_.config.find(key);
    if (it == op_.config.end()) return dflt;
    char* end = nullptr;
    const double v = std::strtod(it->second.c_str(), &end);
    // MLIR writes infinities and NaNs as hexadecimal bits.
    const bool bits = it->second.find_first_of("xX") < it->second.find(':');
    need(end != it->second.c_str() && at_type(end) && !bits && std::isfinite(static_cast<float>(v)),
         std::string(key) + " must be a finite number");
    return v;
  }
  int64_t integer(const char* key, int64_t dflt) const {
    auto it = op_.config.find(key);
    if (it == op_.config.end()) return dflt;
    char* end = nullptr;
    const long long v = std::strtoll(it->second.c_str(), &end, 10);
    need(end != it->second.c_str() && at_type(end), std::string(key) + " must be an integer");
    return v;
  }

 private:
  // What follows a literal: nothing, or ": type".
  static bool at_type(const char* end) {
    while (*end == ' ') ++end;
    return *end == '\0' || *end == ':';
  }
  const Program& prog_;
  const Op& op_;
};

void check_pages(const CallArgs& c, const TensorType& k, const TensorType& v) {
  c.need(k.rank() == 4 && k.dims == v.dims && k.dtype == v.dtype,
         "k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] of one shape and type");
  c.need(is_operator_float(k.dtype), "pages must be f32, f16 or bf16");
  for (int64_t d : k.dims) c.need(d > 0, "pages must not be empty");
  c.within(k.dims[0] * k.dims[1] <= kMaxIndex && k.dims[0] * k.dims[1] * k.dims[2] <= kMaxIndex,
           "more than 2^31 - 1 rows of a head in the pages");
}

void lower_paged_attention(const CallArgs& c, Op* op) {
  c.need(c.ins() == 5 && c.outs() == 1, "takes q, k_pages, v_pages, page_table and lengths, and has one result");
  c.known_keys({"scale", "window"});
  const TensorType &q = c.in(0), &k = c.in(1), &table = c.in(3), &lengths = c.in(4);
  check_pages(c, k, c.in(2));
  c.need(q.rank() == 3 && q.dtype == k.dtype && q.dims[2] == k.dims[3],
         "q must be [batch, heads, head_dim] of the pages' type and head dim");
  c.need(q.dims[1] > 0 && q.dims[1] % k.dims[1] == 0, "q's heads must be a multiple of the pages'");
  c.need(table.rank() == 2 && table.dtype == DType::kS32 && table.dims[0] == q.dims[0] && table.dims[1] > 0,
         "page_table must be s32 [batch, pages of a sequence]");
  c.need(lengths.rank() == 1 && lengths.dtype == DType::kS32 && lengths.dims[0] == q.dims[0],
         "lengths must be s32 [batch]");
  c.need(c.out(0) == q, "the result must have q's shape and type");
  const double scale = c.number("scale", 1.0 / std::sqrt(static_cast<double>(q.dims[2])));
  // the kernels take scores in powers of two
  c.need(std::isfinite(static_cast<float>(scale) * 1.44269504f), "scale times log2(e) must be a finite number");
  const int64_t window = c.integer("window", 0);
  c.need(window >= 0, "window must not be negative");
  c.within(q.dims[2] <= 512, "head dim above 512");
  // keys are counted in 32 bits, up to a tile past the last
  c.within(table.dims[1] <= kMaxIndex && table.dims[1] * k.dims[2] <= kMaxIndex - 64,
           "a page table of more than 2^31 - 65 keys");
  c.within(q.dims[0] <= kMaxGroups && q.dims[1] <= kMaxGroups && q.dims[0] * q.dims[1] <= kMaxGroups, "too many query heads");
  // tiles of 32 keys of every head are counted in 32 bits
  c.within(q.dims[0] * q.dims[1] * ((table.dims[1] * k.dims[2] + 31) / 32 + 1) <= kMaxIndex,
           "too many keys in the page table");
  op->kind = OpKind::kPagedAttention;
  op->oper.scale = scale;
  op->oper.window = window;
}

void lower_paged_append(const CallArgs& c, Op* op) {
  c.need(c.ins() == 5 && c.outs() == 2, "takes k_pages, v_pages, k_new, v_new and slots, and has two results");
  c.known_keys({});
  const TensorType &k = c.in(0), &kn = c.in(2), &slots = c.in(4);
  check_pages(c, k, c.in(1));
  c.need(kn.rank() == 3 && kn == c.in(3) && kn.dtype == k.dtype && kn.dims[1] == k.dims[1] && kn.dims[2] == k.dims[3],
         "k_new and v_new must be [rows, kv_heads, head_dim] of the pages' type, heads and head dim");
  c.need(slots.rank() == 1 && is_index(slots.dtype) && slots.dims[0] == kn.dims[0], "slots must be s32 or s64 [rows]");
  c.need(c.out(0) == k && c.out(1) == k, "the results must have the pages' shape and type");
  c.within(kn.dims[0] <= kMaxGroups, "too many rows");
  c.within(kn.dims[1] <= (int64_t(1) << 24) && kn.dims[2] <= (int64_t(1) << 24) &&
               kn.dims[1] * kn.dims[2] <= (int64_t(1) << 24),
           "rows of more than 2^24 elements");
  c.within(k.dims[0] * k.dims[2] <= kMaxIndex, "more than 2^31 - 1 slots");
  op->kind = OpKind::kPagedAppend;
}

// Leading dims of x as rows.
Dims rows_of(const TensorType& x) { return Dims(x.dims.begin(), x.dims.end() - 1); }

void check_rows(const CallArgs& c, const TensorType& x, const TensorType& gain) {
  c.need(is_operator_float(x.dtype), "the rows must be f32, f16 or bf16");
  c.need(x.rank() >= 1 && x.dims.back() > 0, "the rows must be [..., dim] with a dim of at least 1");
  c.need(gain.rank() == 1 && gain.dims[0] == x.dims.back() && gain.dtype == x.dtype,
         "gain must be [dim] of the rows' type");
  c.within(num_elements(rows_of(x)) < (int64_t(1) << 22), "2^22 rows or more");
  c.within(x.dims.back() <= (int64_t(1) << 28), "rows of more than 2^28 elements");
}

double epsilon(const CallArgs& c) {
  const double eps = c.number("eps", 1e-5);
  c.need(eps >= 0, "eps must not be negative");
  return eps;
}

void lower_add_rms_norm(const CallArgs& c, Op* op) {
  c.need(c.ins() == 2 || c.ins() == 3, "takes x, a residual or none, and gain");
  c.known_keys({"eps"});
  const TensorType& x = c.in(0);
  check_rows(c, x, c.in(c.ins() - 1));
  const bool residual = c.ins() == 3;
  if (residual) c.need(c.in(1) == x, "the residual must have x's shape and type");
  c.need(c.outs() >= 1, "has no result");
  const bool quantize = c.out(0).dtype == DType::kS8;
  const size_t want = (quantize ? 2u : 1u) + (residual ? 1u : 0u);
  c.need(c.outs() == want, quantize ? "an s8 result is followed by its scales, and with a residual by the sum"
                                    : "has the norm as result, and with a residual the sum");
  c.need(c.out(0).dims == x.dims && (quantize || c.out(0) == x), "the norm must have x's shape, and its type or s8");
  if (quantize) {
    const TensorType scales{DType::kF32, rows_of(x)};
    c.need(c.out(1) == scales, "the scales must be f32, one a row");
  }
  if (residual) c.need(c.out(want - 1) == x, "the sum must have x's shape and type");
  op->kind = OpKind::kAddRmsNorm;
  op->oper.eps = epsilon(c);
}

void lower_add_rms_norm_grad(const CallArgs& c, Op* op) {
  c.need((c.ins() == 3 || c.ins() == 4) && c.outs() == 2,
         "takes dy, dsum or none, the sum and gain, and has two results");
  c.known_keys({"eps"});
  const TensorType& dy = c.in(0);
  check_rows(c, dy, c.in(c.ins() - 1));
  for (size_t i = 1; i + 1 < c.ins(); ++i) c.need(c.in(i) == dy, "dy, dsum and the sum must have one shape and type");
  c.need(c.out(0) == dy, "dx must have dy's shape and type");
  c.need(c.out(1) == c.in(c.ins() - 1), "dgain must have gain's shape and type");
  c.within((dy.dims.back() + 15) / 16 <= kMaxGroups, "rows too long");
  op->kind = OpKind::kAddRmsNormGrad;
  op->oper.eps = epsilon(c);
}

void check_logits(const CallArgs& c) {
  const TensorType &x = c.in(0), &tokens = c.in(1);
  c.need(x.rank() == 2 && is_operator_float(x.dtype) && x.dims[1] > 0,
         "logits must be f32, f16 or bf16 [rows, vocabulary]");
  c.need(tokens.rank() == 1 && is_index(tokens.dtype) && tokens.dims[0] == x.dims[0],
         "tokens must be s32 or s64 [rows]");
  c.within(x.dims[1] <= kMaxIndex, "a vocabulary of more than 2^31 - 1");
  c.within(x.dims[0] <= kMaxGroups && x.dims[0] * ((x.dims[1] + 8191) / 8192) <= kMaxGroups, "too many logits");
}

void lower_token_logprobs(const CallArgs& c, Op* op) {
  c.need(c.ins() == 2 && (c.outs() == 3 || c.outs() == 5),
         "takes logits and tokens, and has logprobs, entropy and lse, or these with top_logprobs and top_tokens");
  c.known_keys({});
  check_logits(c);
  const TensorType& x = c.in(0);
  const TensorType row{DType::kF32, {x.dims[0]}};
  for (size_t i = 0; i < 3; ++i) c.need(c.out(i) == row, "logprobs, entropy and lse must be f32 [rows]");
  if (c.outs() == 5) {
    const TensorType &v = c.out(3), &t = c.out(4);
    c.need(v.rank() == 2 && v.dtype == DType::kF32 && v.dims[0] == x.dims[0] && t.dtype == DType::kS32 &&
               t.dims == v.dims,
           "top_logprobs must be f32 [rows, k] and top_tokens s32 [rows, k]");
    c.need(v.dims[1] >= 1 && v.dims[1] <= x.dims[1], "k must be from 1 to the vocabulary's size");
    c.within(v.dims[1] <= kLogprobsMaxTopK, strformat("k above %d", kLogprobsMaxTopK));
    op->oper.top_k = v.dims[1];
  }
  op->kind = OpKind::kTokenLogprobs;
}

void lower_token_logprobs_grad(const CallArgs& c, Op* op) {
  c.need(c.ins() == 6 && c.outs() == 1,
         "takes logits, tokens, lse, entropy, d_logprobs and d_entropy, and has one result");
  c.known_keys({});
  check_logits(c);
  const TensorType row{DType::kF32, {c.in(0).dims[0]}};
  for (size_t i = 2; i < 6; ++i) c.need(c.in(i) == row, "lse, entropy and the gradients must be f32 [rows]");
  c.need(c.out(0) == c.in(0), "the result must have the logits' shape and type");
  op->kind = OpKind::kTokenLogprobsGrad;
}

}  // namespace

bool lower_operator_call(const Program& prog, Op* op) {
  using Lower = void (*)(const CallArgs&, Op*);
  static const std::map<std::string, Lower> targets = {
      {"pjrtx.paged_attention", lower_paged_attention},
      {"pjrtx.paged_append", lower_paged_append},
      {"pjrtx.add_rms_norm", lower_add_rms_norm},
      {"pjrtx.add_rms_norm_grad", lower_add_rms_norm_grad},
      {"pjrtx.token_logprobs", lower_token_logprobs},
      {"pjrtx.token_logprobs_grad", lower_token_logprobs_grad},
  };
  auto it = targets.find(op->target);
  if (it == targets.end()) return false;
  const CallArgs c(prog, *op);
  c.need(op->config.count("backend_config") == 0, "backend_config must be a dictionary");
  // The checks multiply dims in 64 bits.
  for (const std::vector<int>* values : {&op->operands, &op->results})
    for (int v : *values) {
      int64_t n = 8;
      for (int64_t d : prog.type(v).dims)
        c.within(!__builtin_mul_overflow(n, std::max<int64_t>(d, 1), &n), "a tensor of 2^60 elements or more");
    }
  it->second(c, op);
  op->name = op->target;
  return true;
}

LibKind operator_lib_kind(OpKind k) {
  switch (k) {
    case OpKind::kPagedAttention: return LibKind::kPagedAttention;
    case OpKind::kPagedAppend: return LibKind::kPagedAppend;
    case OpKind::kAddRmsNorm: return LibKind::kAddRmsNorm;
    case OpKind::kAddRmsNormGrad: return LibKind::kAddRmsNormGrad;
    case OpKind::kTokenLogprobs: return LibKind::kTokenLogprobs;
    case OpKind::kTokenLogprobsGrad: return LibKind::kTokenLogprobsGrad;
    default: return LibKind::kCopy;
  }
}

double operator_bytes(const Program& prog, const Step& step) {
  const Op& op = prog.ops.at(step.lib_op);
  double bytes = 0;
  for (size_t i = 0; i < op.operands.size(); ++i) {
    const bool pages = (op.kind == OpKind::kPagedAttention && (i == 1 || i == 2)) ||
                       (op.kind == OpKind::kPagedAppend && i < 2);
    if (!pages) bytes += static_cast<double>(prog.type(op.operands[i]).bytes());
  }
  if (op.kind == OpKind::kPagedAppend) {
    bytes += static_cast<double>(prog.type(op.operands[2]).bytes() + prog.type(op.operands[3]).bytes());
    for (int k = 0; k < 2; ++k)
      if (!(step.in_place_operands & (1u << k))) bytes += 2.0 * static_cast<double>(prog.type(op.operands[k]).bytes());
    return bytes;
  }
  for (int v : op.results) bytes += static_cast<double>(prog.type(v).bytes());
  if (op.kind == OpKind::kPagedAttention) {
    const TensorType& k = prog.type(op.operands[1]);
    const double named = static_cast<double>(prog.type(op.operands[3]).elements()) / static_cast<double>(k.dims[0]);
    bytes += 2.0 * std::min(named, 1.0) * static_cast<double>(k.bytes());
  }
  return bytes;
}

void run_operator(Device* dev, const Program& prog, const Step& step, std::vector<MemRef>& vals) {
  const Op& op = prog.ops.at(step.lib_op);
  auto type = [&](size_t i) -> const TensorType& { return prog.type(op.operands[i]); };
  auto in = [&](size_t i) -> const void* { return vals[op.operands[i]] ? vals[op.operands[i]]->ptr : nullptr; };
  auto out = [&](size_t i) -> void* { return vals[op.results[i]] ? vals[op.results[i]]->ptr : nullptr; };
  auto scratch = [&](size_t bytes) { return bytes ? dev->allocate(bytes) : MemRef(); };
  auto at = [](const MemRef& m) -> void* { return m ? m->ptr : nullptr; };
  const DType t = type(0).dtype;
  switch (op.kind) {
    case OpKind::kPagedAttention: {
      PagedParams p;
      const Dims &q = type(0).dims, &k = type(1).dims;
      p.B = q[0];
      p.Hq = static_cast<int>(q[1]);
      p.D = static_cast<int>(q[2]);
      p.P = k[0];
      p.Hkv = static_cast<int>(k[1]);
      p.S = k[2];
      p.M = type(3).dims[1];
      p.window = op.oper.window;
      p.scale = static_cast<float>(op.oper.scale);
      MemRef m = scratch(paged_attention_scratch_bytes(p, t));
      launch_paged_attention(dev->stream(), p, t, in(0), in(1), in(2), static_cast<const int32_t*>(in(3)),
                             static_cast<const int32_t*>(in(4)), out(0), at(m));
      return;
    }
    case OpKind::kPagedAppend: {
      AppendParams p;
      const Dims& k = type(0).dims;
      p.N = type(2).dims[0];
      p.P = k[0];
      p.Hkv = k[1];
      p.S = k[2];
      p.D = k[3];
      p.slot_bytes = static_cast<int>(dtype_size(type(4).dtype));
      for (size_t i = 0; i < 2; ++i)
        if (!(step.in_place_operands & (1u << i)) && type(i).bytes())
          hip_check(hipMemcpyAsync(out(i), in(i), type(i).bytes(), hipMemcpyDeviceToDevice, dev->stream()),
                    "hipMemcpyAsync(pages)");
      launch_paged_append(dev->stream(), p, static_cast<int>(dtype_size(t)), out(0), out(1), in(2), in(3), in(4));
      return;
    }
    case OpKind::kAddRmsNorm: {
      NormParams p;
      p.D = type(0).dims.back();
      p.rows = type(0).elements() / p.D;
      p.eps = static_cast<float>(op.oper.eps);
      const bool residual = op.operands.size() == 3, quantize = prog.type(op.results[0]).dtype == DType::kS8;
      launch_add_rms_norm(dev->stream(), p, t, in(0), residual ? in(1) : nullptr, in(op.operands.size() - 1),
                          quantize ? nullptr : out(0), quantize ? static_cast<int8_t*>(out(0)) : nullptr,
                          quantize ? static_cast<float*>(out(1)) : nullptr,
                          residual ? out(op.results.size() - 1) : nullptr);
      return;
    }
    case OpKind::kAddRmsNormGrad: {
      NormParams p;
      p.D = type(0).dims.back();
      p.rows = type(0).elements() / p.D;
      p.eps = static_cast<float>(op.oper.eps);
      const size_t n = op.operands.size();
      MemRef m = scratch(add_rms_norm_grad_scratch_bytes(p, t));
      launch_add_rms_norm_grad(dev->stream(), p, t, in(0), n == 4 ? in(1) : nullptr, in(n - 2), in(n - 1), out(0),
                               out(1), at(m));
      return;
    }
    case OpKind::kTokenLogprobs:
    case OpKind::kTokenLogprobsGrad: {
      LogprobsParams p;
      p.rows = type(0).dims[0];
      p.V = type(0).dims[1];
      p.top_k = static_cast<int>(op.oper.top_k);
      p.token_bytes = static_cast<int>(dtype_size(type(1).dtype));
      if (op.kind == OpKind::kTokenLogprobs) {
        MemRef m = scratch(token_logprobs_scratch_bytes(p, t));
        launch_token_logprobs(dev->stream(), p, t, in(0), in(1), static_cast<float*>(out(0)),
                              static_cast<float*>(out(1)), static_cast<float*>(out(2)),
                              p.top_k ? static_cast<float*>(out(3)) : nullptr,
                              p.top_k ? static_cast<int32_t*>(out(4)) : nullptr, at(m));
      } else {
        auto f = [&](size_t i) { return static_cast<const float*>(in(i)); };
        launch_token_logprobs_grad(dev->stream(), p, t, in(0), in(1), f(2), f(3), f(4), f(5), out(0));
      }
      return;
    }
    default:
      fail(Code::kInternal, "not an operator: " + op.name);
  }
}

}  // namespace pjrtx
