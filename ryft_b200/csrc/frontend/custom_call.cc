// Reads and checks the operators of custom_call.h.
#include "custom_call.h"

#include <cmath>
#include <set>

namespace b2x {
namespace {

struct Reader {
  const Op& op;
  std::set<std::string> seen;

  [[noreturn]] void fail(int code, const std::string& msg) const {
    throw CompileError(code, "stablehlo.custom_call @" + op.call_target + " (line " + std::to_string(op.line) + "): " + msg);
  }
  void need(bool ok, const std::string& msg) const { if (!ok) fail(kInvalidArgument, msg); }
  void limit(bool ok, const std::string& msg) const { if (!ok) fail(kUnimplemented, msg); }

  const CallAttr* find(const char* name) {
    seen.insert(name);
    auto it = op.call_attrs.find(name);
    return it == op.call_attrs.end() ? nullptr : &it->second;
  }
  bool flag(const char* name) {
    const CallAttr* a = find(name);
    if (!a) return false;
    need(a->kind == CallAttr::BOOL, std::string(name) + " must be true or false");
    return a->b;
  }
  int64_t integer(const char* name, int64_t otherwise) {
    const CallAttr* a = find(name);
    if (!a) return otherwise;
    need(a->kind == CallAttr::INT, std::string(name) + " must be an integer");
    return a->i;
  }
  double number(const char* name, double otherwise) {
    const CallAttr* a = find(name);
    if (!a) return otherwise;
    need(a->kind == CallAttr::FLOAT || a->kind == CallAttr::INT, std::string(name) + " must be a number");
    const double v = a->kind == CallAttr::FLOAT ? a->f : (double)a->i;
    need(std::isfinite(v), std::string(name) + " must be finite");
    return v;
  }
  std::string word(const char* name, const char* otherwise) {
    const CallAttr* a = find(name);
    if (!a) return otherwise;
    need(a->kind == CallAttr::STRING, std::string(name) + " must be a string");
    return a->s;
  }
  std::vector<std::string> words(const char* name) {
    const CallAttr* a = find(name);
    std::vector<std::string> r;
    if (!a) return r;
    need(a->kind == CallAttr::ARRAY, std::string(name) + " must be an array of strings");
    for (auto& e : a->items) { need(e.kind == CallAttr::STRING, std::string(name) + " must be an array of strings"); r.push_back(e.s); }
    return r;
  }
  void done() const {
    for (auto& kv : op.call_attrs) need(seen.count(kv.first) != 0, "unknown attribute '" + kv.first + "'");
  }
  bool layout() {
    const std::string l = word("layout", "bhsd");
    need(l == "bhsd" || l == "bshd", "layout must be \"bhsd\" or \"bshd\"");
    return l == "bshd";
  }
  const TensorType& in(size_t i) const { return op.operands[i]->type; }
  const TensorType& out(size_t i) const { return op.results[i]->type; }
  void same(const TensorType& a, const TensorType& b, const std::string& what) const { need(a == b, what + " has type " + a.str() + " where " + b.str() + " is needed"); }
};

TensorType heads_type(DType t, bool bshd, int64_t B, int64_t H, int64_t S, int64_t D) {
  TensorType r;
  r.dtype = t;
  r.dims = bshd ? std::vector<int64_t>{B, S, H, D} : std::vector<int64_t>{B, H, S, D};
  return r;
}
TensorType type_of(DType t, std::vector<int64_t> dims) {
  TensorType r;
  r.dtype = t;
  r.dims = std::move(dims);
  return r;
}

RotarySpec describe_rotary(Reader& r, bool gradient) {
  const Op& op = r.op;
  RotarySpec s;
  s.gradient = gradient;
  s.bshd = r.layout();
  s.interleaved = r.flag("interleaved");
  s.norm = op.call_attrs.count("epsilon") != 0;
  s.epsilon = r.number("epsilon", 0.0);
  r.need(s.epsilon >= 0.0, "epsilon must not be negative");
  s.base = r.number("base", 10000.0);
  r.need(s.base >= 1.0, "base must be at least 1");
  s.factor = r.number("factor", 1.0);
  r.need(s.factor > 0.0, "factor must be positive");
  s.bands = op.call_attrs.count("bands") != 0;
  if (const CallAttr* a = r.find("bands")) {
    r.need(a->kind == CallAttr::ARRAY && a->items.size() == 3, "bands must be [low, high, original context]");
    double v[3];
    for (int i = 0; i < 3; i++) {
      const CallAttr& e = a->items[i];
      r.need(e.kind == CallAttr::FLOAT || e.kind == CallAttr::INT, "bands must hold numbers");
      v[i] = e.kind == CallAttr::FLOAT ? e.f : (double)e.i;
    }
    s.low = v[0]; s.high = v[1]; s.original = v[2];
    r.need(s.low > 0.0 && s.high > s.low && s.original > 0.0 && std::isfinite(s.high) && std::isfinite(s.original), "bands need 0 < low < high and an original context above 0");
  }
  // how many tensors: every tensor has one result, and one more (its weight's gradient) in a gradient with norms
  const int per = gradient && s.norm ? 2 : 1;
  r.need(!op.results.empty() && op.results.size() % per == 0, "the results do not match the operands");
  s.n = (int)op.results.size() / per;
  r.limit(s.n <= 2, "one or two tensors are rotated in a call");
  size_t want = (size_t)s.n;
  if (s.norm) want += (gradient ? 2 : 1) * (size_t)s.n;
  r.need(op.operands.size() == want || op.operands.size() == want + 1, "expects " + std::to_string(want) + " operands, and the positions where they are given");
  size_t at = 0;
  if (gradient) for (int i = 0; i < s.n; i++) s.dy[i] = (int)at++;
  if (!gradient || s.norm) for (int i = 0; i < s.n; i++) s.x[i] = (int)at++;
  if (s.norm) for (int i = 0; i < s.n; i++) s.w[i] = (int)at++;
  if (at < op.operands.size()) s.positions = (int)at;

  const TensorType& first = r.in(0);
  r.need(first.rank() == 4, "the tensors must have four dimensions");
  s.dtype = first.dtype;
  r.limit(s.dtype == DType::BF16 || s.dtype == DType::F16 || s.dtype == DType::F32, "element types are bf16, f16 and f32");
  s.B = first.dims[0];
  s.S = first.dims[s.bshd ? 1 : 2];
  s.D = first.dims[3];
  s.R = r.integer("rotary_dims", s.D);
  r.need(s.R >= 0 && s.R <= s.D && s.R % 2 == 0, "rotary_dims must be even and at most the head's width");
  r.limit(s.D <= 256, "heads are at most 256 wide");
  for (int i = 0; i < s.n; i++) {
    const TensorType& t = r.in(i);
    r.need(t.rank() == 4, "the tensors must have four dimensions");
    s.heads[i] = t.dims[s.bshd ? 2 : 1];
    const TensorType full = heads_type(s.dtype, s.bshd, s.B, s.heads[i], s.S, s.D);
    r.same(t, full, "operand " + std::to_string(i));
    if (gradient && s.norm) r.same(r.in(s.x[i]), full, "operand " + std::to_string(s.x[i]));
    r.same(r.out(i), full, "result " + std::to_string(i));
    if (s.norm) {
      const TensorType& w = r.in(s.w[i]);
      if (i == 0) s.weight_dtype = w.dtype;
      r.need(w.dtype == DType::F32 || w.dtype == s.dtype, "weights are f32 or of the tensors' element type");
      r.same(w, type_of(s.weight_dtype, {s.D}), "operand " + std::to_string(s.w[i]));
      if (gradient) r.same(r.out(s.n + i), type_of(DType::F32, {s.D}), "result " + std::to_string(s.n + i));
    }
  }
  if (s.positions >= 0) r.same(r.in(s.positions), type_of(DType::S32, {s.B, s.S}), "the positions");
  r.limit(s.B < (1ll << 31) && s.S < (1ll << 31) && s.B * s.S < (1ll << 31) && s.heads[0] < (1 << 20) && s.heads[1] < (1 << 20), "too many tokens or heads");
  return s;
}

AttentionSpec describe_attention(Reader& r, bool gradient) {
  const Op& op = r.op;
  AttentionSpec s;
  s.gradient = gradient;
  s.bshd = r.layout();
  s.causal = r.flag("causal");
  s.queries_at_end = r.flag("queries_at_end");
  s.query_offset = r.integer("query_offset", 0);
  s.softcap = r.number("softcap", 0.0);
  r.need(s.softcap == 0.0 || (s.softcap >= 1e-6 && s.softcap <= 1e6), "softcap must be 0 (none) or lie in [1e-6, 1e6]");
  const std::vector<std::string> extra = r.words("inputs");
  const size_t fixed = gradient ? 6 : 3;
  r.need(op.operands.size() == fixed + extra.size(), "expects " + std::to_string(fixed) + " operands and those that `inputs` names");
  for (size_t i = 0; i < extra.size(); i++) {
    int* slot = extra[i] == "slopes" ? &s.slopes : extra[i] == "documents" ? &s.documents : extra[i] == "prefix" ? &s.prefix : extra[i] == "lengths" ? &s.lengths : nullptr;
    r.need(slot != nullptr, "unknown input '" + extra[i] + "'");
    r.need(*slot < 0, "input '" + extra[i] + "' is named twice");
    *slot = (int)(fixed + i);
  }
  const TensorType& q = r.in(0);
  const TensorType& k = r.in(1);
  r.need(q.rank() == 4 && k.rank() == 4, "the tensors must have four dimensions");
  const int ht = s.bshd ? 2 : 1, st = s.bshd ? 1 : 2;
  s.dtype = q.dtype;
  s.B = q.dims[0]; s.Hq = q.dims[ht]; s.Sq = q.dims[st]; s.D = q.dims[3];
  s.Hk = k.dims[ht]; s.Sk = k.dims[st];
  r.limit(s.dtype == DType::BF16 || s.dtype == DType::F16, "element types are bf16 and f16");
  r.limit(s.D > 0 && s.D % 8 == 0 && s.D <= 128, "the head's width must be a multiple of 8 and at most 128");
  r.need(s.Hk > 0 ? s.Hq % s.Hk == 0 : s.Hq == 0, "the query heads must be a multiple of the key heads");
  const TensorType qt = heads_type(s.dtype, s.bshd, s.B, s.Hq, s.Sq, s.D), kt = heads_type(s.dtype, s.bshd, s.B, s.Hk, s.Sk, s.D);
  const TensorType sums = type_of(DType::F32, {s.B, s.Hq, s.Sq});
  r.same(k, kt, "the keys");
  r.same(r.in(2), kt, "the values");
  if (gradient) {
    r.same(r.in(3), qt, "the result of the attention");
    r.same(r.in(4), sums, "the log sums");
    r.same(r.in(5), qt, "the result's gradient");
    r.need(op.results.size() == 3, "has three results");
    r.same(r.out(0), qt, "the queries' gradient");
    r.same(r.out(1), kt, "the keys' gradient");
    r.same(r.out(2), kt, "the values' gradient");
  } else {
    r.need(op.results.size() == 1 || op.results.size() == 2, "has one result, and the log sums where they are asked for");
    s.log_sum = op.results.size() == 2;
    r.same(r.out(0), qt, "the result");
    if (s.log_sum) r.same(r.out(1), sums, "the log sums");
  }
  s.scale = r.number("scale", s.D > 0 ? 1.0 / std::sqrt((double)s.D) : 1.0);
  r.need(std::fabs(s.scale) <= 1e6, "scale must lie in [-1e6, 1e6]");
  if (s.slopes >= 0) r.same(r.in(s.slopes), type_of(DType::F32, {s.Hq}), "the slopes");
  if (s.documents >= 0) r.same(r.in(s.documents), type_of(DType::S32, {s.B, s.Sk}), "the documents");
  if (s.prefix >= 0) r.same(r.in(s.prefix), type_of(DType::S32, {s.B}), "the prefix");
  if (s.lengths >= 0) r.same(r.in(s.lengths), type_of(DType::S32, {s.B}), "the lengths");
  r.need(s.prefix < 0 || s.causal, "a prefix means something under a causal mask only");
  r.need(!s.queries_at_end || s.lengths >= 0, "queries_at_end needs the lengths");
  r.need(!s.queries_at_end || s.query_offset == 0, "query_offset and queries_at_end exclude one another");
  r.need(s.query_offset >= 0 && s.query_offset < (1ll << 30), "query_offset must lie in [0, 2^30)");
  if (s.documents >= 0 && !s.queries_at_end) r.need(s.query_offset + s.Sq <= s.Sk, "with documents every query must have its place among the keys");
  r.limit(s.Sq < (1ll << 30) && s.Sk < (1ll << 30) && s.B < (1 << 16) && s.Hq < (1 << 16), "too many tokens, heads or sequences");
  return s;
}

}  // namespace

std::vector<uint64_t> RotarySpec::turns() const {
  std::vector<uint64_t> t;
  const long double two_pi = 2.0L * acosl(-1.0L);
  for (int64_t i = 0; i < R / 2; i++) {
    long double f = powl((long double)base, -2.0L * (long double)i / (long double)R);
    if (bands) {
      // share of the frequency that stays: 1 for wavelengths below original / high, 0 above original / low
      long double keep = ((long double)original * f / two_pi - (long double)low) / ((long double)high - (long double)low);
      keep = keep < 0.0L ? 0.0L : keep > 1.0L ? 1.0L : keep;
      f = (1.0L - keep) * f / (long double)factor + keep * f;
    } else {
      f /= (long double)factor;
    }
    long double turn = f / two_pi;
    turn -= floorl(turn);
    const long double scaled = turn * 18446744073709551616.0L;
    t.push_back(scaled >= 18446744073709551615.0L ? 0 : (uint64_t)(scaled + 0.5L));
  }
  return t;
}

CallSpec describe_call(const Op& op) {
  Reader r{op, {}};
  CallSpec c;
  if (op.call_target == "b2x.rotary" || op.call_target == "b2x.rotary_gradient") {
    c.kind = CallKind::ROTARY;
    c.rotary = describe_rotary(r, op.call_target == "b2x.rotary_gradient");
  } else if (op.call_target == "b2x.attention" || op.call_target == "b2x.attention_gradient") {
    c.kind = CallKind::ATTENTION;
    c.attention = describe_attention(r, op.call_target == "b2x.attention_gradient");
  } else {
    r.fail(kUnimplemented, "this executor provides no such target");
  }
  r.done();
  return c;
}

}  // namespace b2x
