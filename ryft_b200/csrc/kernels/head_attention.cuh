// What the kernels of head_attention share: the problem as kernels see it, and which keys a query sees.
#pragma once
#include "../../../include/b2x_kernels.h"
#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2x {

struct HeadAttn {
  const char* q; const char* k; const char* v;
  B2xHeadStrides qs, ks, vs, os, dos, dqs, dks, dvs;
  const float* slopes;
  const int32_t* documents;
  const int32_t* prefix;
  const int32_t* lengths;
  char* o;
  float* lse;
  const char* dout;
  char* dq; char* dk; char* dv;
  int32_t B, Hq, Hk, group, Sq, Sk, D;
  int32_t offset;              // position of the first query, without queries_at_end
  float scale, softcap;
  uint8_t causal, at_end;
};

// Per sequence: how many keys there are, the first query's position, and the keys that every query sees.
struct HeadSequence {
  int length, first, prefix;
};
__device__ __forceinline__ HeadSequence head_sequence(const HeadAttn& p, int b) {
  HeadSequence s;
  s.length = p.Sk;
  if (p.lengths) s.length = min(max((int)ld_global((const uint32_t*)p.lengths + b), 0), p.Sk);
  s.first = p.at_end ? s.length - p.Sq : p.offset;
  s.prefix = p.prefix ? (int)ld_global((const uint32_t*)p.prefix + b) : 0;
  return s;
}
// A query at `pos` sees no key from here on (documents apart).
__device__ __forceinline__ int head_limit(const HeadAttn& p, const HeadSequence& s, int pos) {
  return p.causal ? min(s.length, max(pos + 1, s.prefix)) : s.length;
}

}  // namespace b2x
