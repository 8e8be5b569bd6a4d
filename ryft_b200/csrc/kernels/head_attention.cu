// Attention with grouped heads, capped scores, a bias by distance and document, prefix and length masks, and its gradient.
//
// Forward: one pass over the keys with the running maximum m and sum l of a softmax, o = sum exp(s - m) v / l, log sum m + ln l.
// Gradient: P = exp(s - lse), dP = dO V^T, delta = sum(dO * O), dS = P (dP - delta) (1 - tanh^2) scale; dQ = dS K, dK = dS^T Q,
// dV = P^T dO, the last two over all query heads that share the key head.  Sums, statistics and scores in f32.
//
// The entry points; the kernels are in head_attention_tc.cu (forward), head_attention_token.cu (few queries) and
// head_attention_gradient.cu.
#include <cmath>

#include "head_attention_tc.cuh"

namespace b2x {
namespace {

// Rows that 16-byte accesses can reach; where there are none, no memory is asked for.
bool ha_rows(const void* p, const B2xHeadStrides& s, int64_t B, int64_t H, int64_t S) {
  if (B == 0 || H == 0 || S == 0) return true;
  return p && ((uintptr_t)p & 15) == 0 && (B <= 1 || s.batch % 8 == 0) && (H <= 1 || s.head % 8 == 0) && (S <= 1 || s.token % 8 == 0);
}
bool ha_words(const void* p) { return ((uintptr_t)p & 3) == 0; }   // 32-bit values, or none
bool ha_sizes(const B2xHeadAttentionArgs* a) {
  constexpr int64_t most = 1ll << 31;
  return a->B >= 0 && a->B < most && a->Hq >= 0 && a->Hq < most && a->Hk >= 0 && a->Hk < most && a->B * a->Hq < most && a->B * a->Hk < most && a->Sq >= 0 &&
         a->Sq < (1ll << 30) && a->Sk >= 0 && a->Sk < (1ll << 30) && a->D > 0 && a->D % 8 == 0 && a->D <= 128 && (a->Hk > 0 ? a->Hq % a->Hk == 0 : a->Hq == 0);
}
bool ha_valid(const B2xHeadAttentionArgs* a) {
  return ha_sizes(a) && (a->elem == EL_BF16 || a->elem == EL_F16) && ha_rows(a->q, a->qs, a->B, a->Hq, a->Sq) && ha_rows(a->k, a->ks, a->B, a->Hk, a->Sk) &&
         ha_rows(a->v, a->vs, a->B, a->Hk, a->Sk) && ha_rows(a->o, a->os, a->B, a->Hq, a->Sq) && ha_words(a->lse) && ha_words(a->slopes) && ha_words(a->documents) &&
         ha_words(a->prefix) && ha_words(a->lengths) && (a->softcap == 0.f || (a->softcap >= 1e-6f && a->softcap <= 1e6f)) && std::fabs(a->scale) <= 1e6f &&
         a->query_offset >= 0 && a->query_offset < (1ll << 30) && (!a->queries_at_end || a->lengths);
}

HeadAttn ha_params(const B2xHeadAttentionArgs* a) {
  HeadAttn p{};
  p.q = (const char*)a->q; p.k = (const char*)a->k; p.v = (const char*)a->v;
  p.qs = a->qs; p.ks = a->ks; p.vs = a->vs; p.os = a->os; p.dos = a->dos; p.dqs = a->dqs; p.dks = a->dks; p.dvs = a->dvs;
  p.slopes = a->slopes; p.documents = a->documents; p.prefix = a->prefix; p.lengths = a->lengths;
  p.o = (char*)a->o; p.lse = a->lse; p.dout = (const char*)a->dout;
  p.dq = (char*)a->dq; p.dk = (char*)a->dk; p.dv = (char*)a->dv;
  p.B = (int32_t)a->B; p.Hq = (int32_t)a->Hq; p.Hk = (int32_t)a->Hk; p.group = a->Hk > 0 ? (int32_t)(a->Hq / a->Hk) : 1;
  p.Sq = (int32_t)a->Sq; p.Sk = (int32_t)a->Sk; p.D = (int32_t)a->D;
  p.offset = (int32_t)a->query_offset;
  p.scale = a->scale; p.softcap = a->softcap;
  p.causal = a->causal; p.at_end = a->queries_at_end;
  return p;
}

}  // namespace
}  // namespace b2x

extern "C" int64_t b2x_head_attention_scratch_bytes(const B2xHeadAttentionArgs* a, int gradient) {
  const int64_t ranges = a->documents ? a->B * ((a->Sk + b2x::HA_BLOCK - 1) / b2x::HA_BLOCK) * 8 : 0;
  if (gradient) return b2x::ha_gradient_scratch(a, ranges);
  const b2x::HeadAttn p = b2x::ha_params(a);
  return b2x::ha_token_takes(p) ? b2x::ha_token_scratch(p) : b2x::ha_forward_scratch(p, ranges);
}

extern "C" int b2x_head_attention_launches(const B2xHeadAttentionArgs* a, int gradient) {
  const int q = a->B * a->Hq * a->Sq > 0, k = a->B * a->Hk * a->Sk > 0, ranges = k && a->documents;
  if (gradient) return ranges + b2x::ha_gradient_launches(a);
  const b2x::HeadAttn p = b2x::ha_params(a);
  return !q ? 0 : b2x::ha_token_takes(p) ? b2x::ha_token_launches(p) : b2x::ha_forward_launches(p) + ranges;
}

extern "C" int b2x_launch_head_attention(const B2xHeadAttentionArgs* a, int32_t* status, b2x_stream_t stream) {
  using namespace b2x;
  if (!ha_valid(a) || (b2x_head_attention_scratch_bytes(a, 0) > 0 && !a->scratch) || ((uintptr_t)a->scratch & 15) != 0) return (int)cudaErrorInvalidValue;
  const HeadAttn p = ha_params(a);
  if (ha_token_takes(p)) return ha_launch_token(p, a->elem, a->scratch, (cudaStream_t)stream);
  return ha_launch_forward(p, a->elem, (int2*)a->scratch, status, (cudaStream_t)stream);
}

extern "C" int b2x_launch_head_attention_gradient(const B2xHeadAttentionArgs* a, int32_t* status, b2x_stream_t stream) {
  using namespace b2x;
  if (!ha_valid(a) || (!a->lse && a->B * a->Hq * a->Sq > 0) || (b2x_head_attention_scratch_bytes(a, 1) > 0 && !a->scratch) || ((uintptr_t)a->scratch & 15) != 0) return (int)cudaErrorInvalidValue;
  if (!ha_rows(a->dout, a->dos, a->B, a->Hq, a->Sq) || !ha_rows(a->dq, a->dqs, a->B, a->Hq, a->Sq) || !ha_rows(a->dk, a->dks, a->B, a->Hk, a->Sk) ||
      !ha_rows(a->dv, a->dvs, a->B, a->Hk, a->Sk)) return (int)cudaErrorInvalidValue;
  return ha_launch_gradient(ha_params(a), a->elem, a->scratch, status, (cudaStream_t)stream);
}
