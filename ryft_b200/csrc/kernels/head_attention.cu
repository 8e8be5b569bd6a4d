// Attention with grouped heads, capped scores, a bias by distance and document, prefix and length masks, and its gradient.
//
// Forward: one pass over the keys with the running maximum m and sum l of a softmax, o = sum exp(s - m) v / l, log sum m + ln l.
// Gradient: P = exp(s - lse), dP = dO V^T, delta = sum(dO * O), dS = P (dP - delta) (1 - tanh^2) scale; dQ = dS K, dK = dS^T Q,
// dV = P^T dO, the last two over all query heads that share the key head.  Sums, statistics and scores in f32.
//
// The forward pass is in head_attention_tc.cu.  Gradient: one warp per query (dQ) or per key (dK, dV); lanes share the head's width.
#include <cmath>

#include "head_attention_tc.cuh"

namespace b2x {
namespace {

template <int EL> __device__ __forceinline__ float ha_get(const char* p, int64_t i) {
  const uint16_t h = (uint16_t)ld_global((const uint16_t*)p + i);
  if constexpr (EL == EL_BF16) return __uint_as_float((uint32_t)h << 16);
  else return __half2float(__ushort_as_half(h));
}
template <int EL> __device__ __forceinline__ void ha_put(char* p, int64_t i, float v) {
  if constexpr (EL == EL_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16(v);
  else ((__half*)p)[i] = __float2half(v);
}
__device__ __forceinline__ int64_t ha_at(const B2xHeadStrides& s, int b, int h, int t) { return (int64_t)b * s.batch + (int64_t)h * s.head + (int64_t)t * s.token; }

template <int EL> struct Row {
  float v[4];
  __device__ __forceinline__ void load(const char* p, int64_t at, int D) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = lane + 32 * i < D ? ha_get<EL>(p, at + lane + 32 * i) : 0.f;
  }
  __device__ __forceinline__ float dot(const Row& o) const {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) s = fmaf(v[i], o.v[i], s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    return s;
  }
};
template <int EL> __device__ __forceinline__ void ha_store(char* p, int64_t at, int D, const float (&v)[4], float f) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; i++) if (lane + 32 * i < D) ha_put<EL>(p, at + lane + 32 * i, v[i] * f);
}

// the score, and with it the derivative of the cap
__device__ __forceinline__ float ha_score(const HeadAttn& p, float dot, float slope, int pos, int key, float* bend) {
  float s = dot * p.scale;
  *bend = 1.f;
  if (p.softcap > 0.f) { const float t = tanhf(s / p.softcap); s = p.softcap * t; *bend = 1.f - t * t; }
  return s - slope * fabsf((float)(pos - key));
}
__device__ __forceinline__ bool ha_document(const HeadAttn& p, int b, int pos, int* doc) {
  *doc = 0;
  if (!p.documents) return true;
  if (pos < 0 || pos >= p.Sk) return false;
  *doc = (int)ld_global((const uint32_t*)p.documents + (int64_t)b * p.Sk + pos);
  return true;
}

template <int EL>
__global__ void __launch_bounds__(128) k_head_attention_dq_simple(const __grid_constant__ HeadAttn p) {
  pdl_trigger();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (int64_t)p.B * p.Hq * p.Sq) return;
  const int i = (int)(id % p.Sq), h = (int)(id / p.Sq % p.Hq), b = (int)(id / p.Sq / p.Hq), u = h / p.group;
  const HeadSequence s = head_sequence(p, b);
  const int pos = s.first + i;
  int doc;
  const int end = ha_document(p, b, pos, &doc) ? head_limit(p, s, pos) : 0;
  const float slope = p.slopes ? ld_global(p.slopes + h) : 0.f;
  Row<EL> q, k, v, d, o;
  q.load(p.q, ha_at(p.qs, b, h, i), p.D);
  d.load(p.dout, ha_at(p.dos, b, h, i), p.D);
  o.load(p.o, ha_at(p.os, b, h, i), p.D);
  const float delta = d.dot(o), lse = ld_global(p.lse + id);
  if ((threadIdx.x & 31) == 0) p.delta[id] = delta;
  float g[4] = {0.f, 0.f, 0.f, 0.f}, bend;
  for (int j = 0; j < end; j++) {
    if (p.documents && (int)ld_global((const uint32_t*)p.documents + (int64_t)b * p.Sk + j) != doc) continue;
    k.load(p.k, ha_at(p.ks, b, u, j), p.D);
    v.load(p.v, ha_at(p.vs, b, u, j), p.D);
    const float w = expf(ha_score(p, q.dot(k), slope, pos, j, &bend) - lse);
    const float ds = w * (d.dot(v) - delta) * bend * p.scale;
#pragma unroll
    for (int c = 0; c < 4; c++) g[c] = fmaf(ds, k.v[c], g[c]);
  }
  ha_store<EL>(p.dq, ha_at(p.dqs, b, h, i), p.D, g, 1.f);
}

template <int EL>
__global__ void __launch_bounds__(128) k_head_attention_dkv_simple(const __grid_constant__ HeadAttn p) {
  pdl_trigger();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (int64_t)p.B * p.Hk * p.Sk) return;
  const int j = (int)(id % p.Sk), u = (int)(id / p.Sk % p.Hk), b = (int)(id / p.Sk / p.Hk);
  const HeadSequence s = head_sequence(p, b);
  const int mine = p.documents ? (int)ld_global((const uint32_t*)p.documents + (int64_t)b * p.Sk + j) : 0;
  Row<EL> q, k, v, d;
  k.load(p.k, ha_at(p.ks, b, u, j), p.D);
  v.load(p.v, ha_at(p.vs, b, u, j), p.D);
  float gk[4] = {0.f, 0.f, 0.f, 0.f}, gv[4] = {0.f, 0.f, 0.f, 0.f}, bend;
  for (int h = u * p.group; h < (u + 1) * p.group; h++) {
    const float slope = p.slopes ? ld_global(p.slopes + h) : 0.f;
    for (int i = 0; i < p.Sq; i++) {
      const int pos = s.first + i;
      int doc;
      if (!ha_document(p, b, pos, &doc) || doc != mine || j >= head_limit(p, s, pos)) continue;
      const int64_t row = ((int64_t)b * p.Hq + h) * p.Sq + i;
      q.load(p.q, ha_at(p.qs, b, h, i), p.D);
      d.load(p.dout, ha_at(p.dos, b, h, i), p.D);
      const float w = expf(ha_score(p, q.dot(k), slope, pos, j, &bend) - ld_global(p.lse + row));
      const float ds = w * (d.dot(v) - ld_global(p.delta + row)) * bend * p.scale;
#pragma unroll
      for (int c = 0; c < 4; c++) { gk[c] = fmaf(ds, q.v[c], gk[c]); gv[c] = fmaf(w, d.v[c], gv[c]); }
    }
  }
  ha_store<EL>(p.dk, ha_at(p.dks, b, u, j), p.D, gk, 1.f);
  ha_store<EL>(p.dv, ha_at(p.dvs, b, u, j), p.D, gv, 1.f);
}

// rows that 16-byte accesses can reach
bool ha_rows(const void* p, const B2xHeadStrides& s, int64_t B, int64_t H, int64_t S) {
  return ((uintptr_t)p & 15) == 0 && (B <= 1 || s.batch % 8 == 0) && (H <= 1 || s.head % 8 == 0) && (S <= 1 || s.token % 8 == 0);
}
bool ha_valid(const B2xHeadAttentionArgs* a) {
  return ha_rows(a->q, a->qs, a->B, a->Hq, a->Sq) && ha_rows(a->k, a->ks, a->B, a->Hk, a->Sk) && ha_rows(a->v, a->vs, a->B, a->Hk, a->Sk) &&
         ha_rows(a->o, a->os, a->B, a->Hq, a->Sq) && (!a->lse || a->B * a->Hq * a->Sq < (1ll << 40)) && (a->elem == EL_BF16 || a->elem == EL_F16) && a->D > 0 && a->D % 8 == 0 && a->D <= 128 && a->Hk >= 0 && (a->Hk > 0 ? a->Hq % a->Hk == 0 : a->Hq == 0) &&
         a->Sq < (1ll << 30) && a->Sk < (1ll << 30) && a->query_offset >= 0 && a->query_offset < (1ll << 30) && (!a->queries_at_end || a->lengths);
}

HeadAttn ha_params(const B2xHeadAttentionArgs* a) {
  HeadAttn p{};
  p.q = (const char*)a->q; p.k = (const char*)a->k; p.v = (const char*)a->v;
  p.qs = a->qs; p.ks = a->ks; p.vs = a->vs; p.os = a->os; p.dos = a->dos; p.dqs = a->dqs; p.dks = a->dks; p.dvs = a->dvs;
  p.slopes = a->slopes; p.documents = a->documents; p.prefix = a->prefix; p.lengths = a->lengths;
  p.o = (char*)a->o; p.lse = a->lse; p.dout = (const char*)a->dout;
  p.dq = (char*)a->dq; p.dk = (char*)a->dk; p.dv = (char*)a->dv;
  p.delta = (float*)a->scratch;
  p.B = (int32_t)a->B; p.Hq = (int32_t)a->Hq; p.Hk = (int32_t)a->Hk; p.group = a->Hk > 0 ? (int32_t)(a->Hq / a->Hk) : 1;
  p.Sq = (int32_t)a->Sq; p.Sk = (int32_t)a->Sk; p.D = (int32_t)a->D;
  p.offset = (int32_t)a->query_offset;
  p.scale = a->scale; p.softcap = a->softcap;
  p.causal = a->causal; p.at_end = a->queries_at_end;
  return p;
}

int ha_launch(void (*bf16)(HeadAttn), void (*f16)(HeadAttn), int elem, const HeadAttn& p, int64_t rows, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if ((rows + 3) / 4 > 0x7fffffff) return (int)cudaErrorInvalidValue;
  const cudaError_t e = launch_overlapped(elem == EL_BF16 ? bf16 : f16, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, stream, p);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace b2x

extern "C" int64_t b2x_head_attention_scratch_bytes(const B2xHeadAttentionArgs* a, int gradient) {
  const int64_t ranges = a->documents ? a->B * ((a->Sk + b2x::HA_BLOCK - 1) / b2x::HA_BLOCK) * 8 : 0;
  return gradient ? a->B * a->Hq * a->Sq * 4 : ranges;
}

extern "C" int b2x_head_attention_launches(const B2xHeadAttentionArgs* a, int gradient) {
  const int q = a->B * a->Hq * a->Sq > 0, k = a->B * a->Hk * a->Sk > 0;
  return gradient ? q + k : q + (q && k && a->documents ? 1 : 0);
}

extern "C" int b2x_launch_head_attention(const B2xHeadAttentionArgs* a, int32_t* status, b2x_stream_t stream) {
  using namespace b2x;
  if (!ha_valid(a) || (b2x_head_attention_scratch_bytes(a, 0) > 0 && !a->scratch)) return (int)cudaErrorInvalidValue;
  return ha_launch_forward(ha_params(a), a->elem, (int2*)a->scratch, status, (cudaStream_t)stream);
}

extern "C" int b2x_launch_head_attention_gradient(const B2xHeadAttentionArgs* a, int32_t* status, b2x_stream_t stream) {
  using namespace b2x;
  (void)status;
  if (!ha_valid(a) || !a->lse || (b2x_head_attention_scratch_bytes(a, 1) > 0 && !a->scratch)) return (int)cudaErrorInvalidValue;
  const HeadAttn p = ha_params(a);
  const int rc = ha_launch(k_head_attention_dq_simple<EL_BF16>, k_head_attention_dq_simple<EL_F16>, a->elem, p, a->B * a->Hq * a->Sq, (cudaStream_t)stream);
  if (rc) return rc;
  return ha_launch(k_head_attention_dkv_simple<EL_BF16>, k_head_attention_dkv_simple<EL_F16>, a->elem, p, a->B * a->Hk * a->Sk, (cudaStream_t)stream);
}
