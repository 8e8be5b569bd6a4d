// A plan's CALL step as the arguments of its kernel entry point; `bind` turns a buffer reference into a device pointer.
#pragma once
#include "../../../include/b2x_kernels.h"
#include "plan.h"

namespace b2x {

// For questions about sizes before there is memory: operands that are there are not NULL, as at a launch.
inline void* bind_nowhere(const BufRef& b) { return b.valid() ? (void*)16 : nullptr; }

inline B2xHeadStrides head_strides(const Step::CallTensor& t) { return B2xHeadStrides{t.batch, t.head, t.token}; }

template <typename Bind>
B2xRotaryArgs rotary_args(const Step& s, const Bind& bind) {
  const RotarySpec& r = s.call->rotary;
  B2xRotaryArgs a{};
  a.elem = (uint8_t)r.dtype; a.weight_elem = (uint8_t)r.weight_dtype;
  a.n = (uint8_t)r.n; a.norm = r.norm; a.interleaved = r.interleaved;
  a.B = r.B; a.S = r.S; a.D = r.D; a.R = r.R;
  a.epsilon = (float)r.epsilon;
  for (int i = 0; i < r.n; i++) {
    a.heads[i] = r.heads[i];
    if (r.x[i] >= 0) { a.x[i] = bind(s.call_in[r.x[i]].buf); a.xs[i] = head_strides(s.call_in[r.x[i]]); }
    if (r.dy[i] >= 0) { a.dy[i] = bind(s.call_in[r.dy[i]].buf); a.dys[i] = head_strides(s.call_in[r.dy[i]]); }
    if (r.w[i] >= 0) a.weight[i] = bind(s.call_in[r.w[i]].buf);
    a.y[i] = bind(s.call_out[i].buf); a.ys[i] = head_strides(s.call_out[i]);
    if (r.gradient && r.norm) a.dweight[i] = (float*)bind(s.call_out[r.n + i].buf);
  }
  if (r.positions >= 0) a.positions = (const int32_t*)bind(s.call_in[r.positions].buf);
  a.turns = (const uint64_t*)bind(s.call_table);
  if (s.scratch.valid()) a.scratch = bind(s.scratch);
  return a;
}

template <typename Bind>
B2xHeadAttentionArgs head_attention_args(const Step& s, const Bind& bind) {
  const AttentionSpec& t = s.call->attention;
  B2xHeadAttentionArgs a{};
  auto in = [&](int i) { return bind(s.call_in[i].buf); };
  a.elem = (uint8_t)t.dtype; a.causal = t.causal; a.queries_at_end = t.queries_at_end;
  a.B = t.B; a.Hq = t.Hq; a.Hk = t.Hk; a.Sq = t.Sq; a.Sk = t.Sk; a.D = t.D;
  a.scale = (float)t.scale; a.softcap = (float)t.softcap; a.query_offset = t.query_offset;
  a.q = in(0); a.k = in(1); a.v = in(2);
  a.qs = head_strides(s.call_in[0]); a.ks = head_strides(s.call_in[1]); a.vs = head_strides(s.call_in[2]);
  if (t.slopes >= 0) a.slopes = (const float*)in(t.slopes);
  if (t.documents >= 0) a.documents = (const int32_t*)in(t.documents);
  if (t.prefix >= 0) a.prefix = (const int32_t*)in(t.prefix);
  if (t.lengths >= 0) a.lengths = (const int32_t*)in(t.lengths);
  if (t.gradient) {
    a.o = in(3); a.os = head_strides(s.call_in[3]);
    a.lse = (float*)in(4);
    a.dout = in(5); a.dos = head_strides(s.call_in[5]);
    a.dq = bind(s.call_out[0].buf); a.dk = bind(s.call_out[1].buf); a.dv = bind(s.call_out[2].buf);
    a.dqs = head_strides(s.call_out[0]); a.dks = head_strides(s.call_out[1]); a.dvs = head_strides(s.call_out[2]);
  } else {
    a.o = bind(s.call_out[0].buf); a.os = head_strides(s.call_out[0]);
    if (t.log_sum) a.lse = (float*)bind(s.call_out[1].buf);
  }
  if (s.scratch.valid()) a.scratch = bind(s.scratch);
  return a;
}

}  // namespace b2x
