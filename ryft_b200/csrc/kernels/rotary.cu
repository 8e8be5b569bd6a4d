// Rotary positions of queries and keys, with the norm of each head in the same pass, and the gradient of both.
//
//   n = x * r * w,  r = rsqrt(mean(x^2) + epsilon)          (or n = x)
//   (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin)      for every pair (a, b) of the first R elements of a head
// and back:  dn is dy turned the other way;  g = dn * w;  dx = r (g - x r^2 mean(g x));  dw = sum over tokens and heads of dn x r.
//
// Bound by HBM: every element is read once and written once (the gradient reads x and dy).  A head lies across L lanes of a warp
// (the smallest power of two that holds it with two 16-byte pieces per lane: 8 lanes for 128 elements of 16 bits), a pair's two
// elements always in one lane, so the only exchange is the norm's sum over L lanes.  A warp keeps one token, so that the 2R
// cosines and sines are computed once, a few per lane, shared through shared memory and then held in registers for all the
// heads that it walks.  8192 tokens of 40 heads of 128 bf16 elements, with norms: 37 us, 4.5 TB/s (54 % of the issue slots: the norm's
// and the turn's arithmetic in f32; without norms 33.5 us, 5.0 TB/s); the gradient of 16384 such tokens 115 us, 4.4 TB/s.  Each layout
// of pairs is a kernel of its own: with both in one, 38 and 118 us.  The gradient's instance for 16-byte pieces of bf16 spills 6
// registers, that of f16 13, at the 128 that two CTAs per SM leave.
//
// Angles: a position times a frequency in f32 is off by whole turns far into a context.  Frequencies are therefore turns per
// position as fractions of 2^64, computed in extended precision where the program is compiled; the product with the position
// wraps exactly, and its upper 32 bits are the angle to 2^-32 of a turn at any position.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../../include/b2x_kernels.h"
#include "attention_math.cuh"
#include "common.cuh"

namespace b2x {
namespace {

constexpr int kRotaryWarps = 8;
constexpr int kRotaryRows = 4;       // heads of a lane in flight: 128 bytes of loads per thread at 128 elements of 16 bits

struct RotaryParams {
  const char* x[2];
  const char* dy[2];
  char* y[2];
  B2xHeadStrides xs[2], dys[2], ys[2];
  const char* weight[2];
  const int32_t* positions;
  const uint64_t* turns;
  float* partial;              // gradient with norms: [tensor][CTA][D]
  int32_t tokens, S, D, R;
  int32_t heads[2];            // a token's heads are cut into jobs of `job_heads`: of both tensors together, in a gradient of each
  int32_t job_heads, lanes, units;
  int32_t pair_units;          // half layout: units whose two pieces are partners
  float epsilon, inv_d, sine;  // sine: 1, or -1 to turn back
  uint8_t norm, weight_f32, weight_wide;   // wide: weights start on 16 bytes
};

template <int EL> __device__ __forceinline__ float rot_get(const uint32_t* w, int i) {
  if constexpr (EL == EL_F32) return __uint_as_float(w[i]);
  else {
    const uint32_t h = (i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
    if constexpr (EL == EL_BF16) return __uint_as_float(h << 16);
    else return __half2float(__ushort_as_half((unsigned short)h));
  }
}
template <int EL> __device__ __forceinline__ uint32_t rot_pack(float a, float b) {   // two 16-bit elements
  if constexpr (EL == EL_BF16) { __nv_bfloat162 t = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&t); }
  else { __half2 t = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t*>(&t); }
}

// V elements as they lie in memory, and as floats
template <int EL, int V> struct RotRaw {
  static constexpr int BYTES = V * (EL == EL_F32 ? 4 : 2);
  uint32_t w[(BYTES + 3) / 4];
  // zeros where there is nothing, without a branch
  __device__ __forceinline__ void load(const char* p, bool on) {
    const int q = on;
    if constexpr (BYTES == 16)
      asm volatile("{\n .reg .pred q;\n setp.ne.s32 q, %5, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n mov.b32 %2, 0;\n mov.b32 %3, 0;\n @q ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
                   : "=&r"(w[0]), "=&r"(w[1]), "=&r"(w[2]), "=&r"(w[3]) : "l"(__cvta_generic_to_global(p)), "r"(q));
    else if constexpr (BYTES == 8)
      asm volatile("{\n .reg .pred q;\n setp.ne.s32 q, %3, 0;\n mov.b32 %0, 0;\n mov.b32 %1, 0;\n @q ld.global.v2.u32 {%0, %1}, [%2];\n}"
                   : "=&r"(w[0]), "=&r"(w[1]) : "l"(__cvta_generic_to_global(p)), "r"(q));
    else if constexpr (BYTES == 4)
      asm volatile("{\n .reg .pred q;\n setp.ne.s32 q, %2, 0;\n mov.b32 %0, 0;\n @q ld.global.u32 %0, [%1];\n}" : "=&r"(w[0]) : "l"(__cvta_generic_to_global(p)), "r"(q));
    else w[0] = on ? ld_global((const uint16_t*)p) : 0u;
  }
};
template <int EL, int V> __device__ __forceinline__ void rot_store(char* p, const float (&v)[V]) {
  if constexpr (EL == EL_F32) {
    if constexpr (V == 4) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
    else *(float*)p = v[0];
  } else if constexpr (V == 8) {
    *(uint4*)p = make_uint4(rot_pack<EL>(v[0], v[1]), rot_pack<EL>(v[2], v[3]), rot_pack<EL>(v[4], v[5]), rot_pack<EL>(v[6], v[7]));
  } else if constexpr (V == 4) {
    *(uint2*)p = make_uint2(rot_pack<EL>(v[0], v[1]), rot_pack<EL>(v[2], v[3]));
  } else {
    *(uint16_t*)p = (uint16_t)(rot_pack<EL>(v[0], 0.f) & 0xffffu);
  }
}

// Two adjacent elements of V at a time where there are two: the kernels are bound by the instructions that they issue as much as by HBM.
__device__ __forceinline__ uint64_t rot_two(const float* v) { return pack2(__float_as_uint(v[0]), __float_as_uint(v[1])); }
__device__ __forceinline__ void rot_put(float* v, uint64_t x) {
  uint32_t a, b;
  unpack2(x, a, b);
  v[0] = __uint_as_float(a); v[1] = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t rot_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t rot_neg2(uint64_t a) { return a ^ 0x8000000080000000ull; }
// o = a * b, o = a * f, o = a * b + c
template <int V> __device__ __forceinline__ void rot_mul(float (&o)[V], const float (&a)[V], const float (&b)[V]) {
  if constexpr (V == 1) o[0] = a[0] * b[0];
  else {
#pragma unroll
    for (int j = 0; j < V; j += 2) rot_put(o + j, rot_mul2(rot_two(a + j), rot_two(b + j)));
  }
}
template <int V> __device__ __forceinline__ void rot_scale(float (&o)[V], const float (&a)[V], float f) {
  if constexpr (V == 1) o[0] = a[0] * f;
  else {
    const uint64_t f2 = splat2(f);
#pragma unroll
    for (int j = 0; j < V; j += 2) rot_put(o + j, rot_mul2(rot_two(a + j), f2));
  }
}
template <int V> __device__ __forceinline__ void rot_fma(float (&o)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
  if constexpr (V == 1) o[0] = fmaf(a[0], b[0], c[0]);
  else {
#pragma unroll
    for (int j = 0; j < V; j += 2) rot_put(o + j, fma2(rot_two(a + j), rot_two(b + j), rot_two(c + j)));
  }
}
template <int V> __device__ __forceinline__ void rot_fma(float (&o)[V], const float (&a)[V], float f, const float (&c)[V]) {
  if constexpr (V == 1) o[0] = fmaf(a[0], f, c[0]);
  else {
    const uint64_t f2 = splat2(f);
#pragma unroll
    for (int j = 0; j < V; j += 2) rot_put(o + j, fma2(rot_two(a + j), f2, rot_two(c + j)));
  }
}

// PAIRS: interleaved.  NU units per lane; a unit is two pieces of V elements that start at e[u][0] and e[u][1] (-1: none)
template <int EL, int V, int NU, bool PAIRS> struct RotLane {
  static constexpr int ES = EL == EL_F32 ? 4 : 2;
  using Raw = RotRaw<EL, V>;
  int e[NU][2];
  int turns[NU];                   // pairs of the unit that turn: the first so many, the others pass
  float cs[NU][V], sn[NU][V];      // of pair j: half layout (a_j, b_j); interleaved pairs of piece 0, then of piece 1
  float w[NU][2][V];
  float ca[NU][V], sa[NU][V], cb[NU][V], sb[NU][V];

  __device__ __forceinline__ void pieces(const RotaryParams& p, int lane) {
#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int unit = lane + u * p.lanes;
      int a = -1, b = -1, t = 0;
      if (unit < p.units) {
        if constexpr (PAIRS) { a = 2 * unit * V; b = a + V; t = min(max(p.R / 2 - unit * V, 0), V); }
        else if (unit < p.pair_units) { a = unit * V; b = a + p.R / 2; t = V; }
        else { a = p.R + 2 * (unit - p.pair_units) * V; b = a + V; }
        if (b >= p.D) b = -1;
      }
      e[u][0] = a; e[u][1] = b; turns[u] = t;
    }
  }
  // cosines and sines of the warp's token
  __device__ __forceinline__ void angles(const RotaryParams& p, int token, float2* table) {
    const int lane = threadIdx.x & 31;
    const int64_t pos = p.positions ? (int64_t)(int32_t)ld_global((const uint32_t*)p.positions + token) : (int64_t)(token % p.S);
    __syncwarp();
    for (int i = lane; i < p.R / 2; i += 32) {
      const uint2 t = ld_global((const uint2*)(p.turns + i));
      const uint64_t turn = (((uint64_t)t.y << 32) | t.x) * (uint64_t)pos;
      float s, c;
      sincospif((float)(int32_t)(turn >> 32) * (1.0f / 2147483648.0f), &s, &c);
      table[i] = make_float2(c, s * p.sine);
    }
    __syncwarp();
  }
  __device__ __forceinline__ void take(const RotaryParams& p, const float2* table) {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int j = 0; j < V; j++) {
        // the unit's first pair: both layouts count pairs from half the first element on, or from the element itself
        const float2 t = j < turns[u] ? table[(PAIRS ? e[u][0] / 2 : e[u][0]) + j] : make_float2(1.f, 0.f);
        cs[u][j] = t.x; sn[u][j] = t.y;
      }
  }
  __device__ __forceinline__ void weights(const RotaryParams& p, int ti) {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        if constexpr (V > 1) {
          if (p.norm && p.weight_wide) {
            if (p.weight_f32) {
#pragma unroll
              for (int j = 0; j < V; j += 4) {
                RotRaw<EL_F32, 4> q;
                q.load(p.weight[ti] + (int64_t)(e[u][s] + j) * 4, e[u][s] >= 0);
#pragma unroll
                for (int i = 0; i < 4; i++) w[u][s][j + i] = __uint_as_float(q.w[i]);
              }
            } else {
              Raw q;
              q.load(p.weight[ti] + (int64_t)e[u][s] * ES, e[u][s] >= 0);
#pragma unroll
              for (int j = 0; j < V; j++) w[u][s][j] = rot_get<EL>(q.w, j);
            }
            continue;
          }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
          w[u][s][j] = 1.f;
          if (p.norm && e[u][s] >= 0) {
            if (p.weight_f32) w[u][s][j] = ld_global((const float*)p.weight[ti] + e[u][s] + j);
            else {
              const uint32_t h = ld_global((const uint16_t*)p.weight[ti] + e[u][s] + j);
              w[u][s][j] = rot_get<EL>(&h, 0);
            }
          }
        }
      }
  }
  __device__ __forceinline__ void load(const char* row, bool on, Raw (&v)[NU][2]) const {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        v[u][s].load(row + (int64_t)e[u][s] * ES, on && e[u][s] >= 0);
      }
  }
  static __device__ __forceinline__ void floats(const Raw (&r)[NU][2], float (&v)[NU][2][V]) {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int s = 0; s < 2; s++)
#pragma unroll
        for (int j = 0; j < V; j++) v[u][s][j] = rot_get<EL>(r[u][s].w, j);
  }
  __device__ __forceinline__ void store(char* row, const float (&v)[NU][2][V]) const {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int s = 0; s < 2; s++)
        if (e[u][s] >= 0) rot_store<EL, V>(row + (int64_t)e[u][s] * ES, v[u][s]);
  }
  // w (of the elements) times cos and sin: the pair (a, b) turns to f (a ca + b sb), f (b cb + a sa)
  __device__ __forceinline__ void fold(const RotaryParams& p, const float2* table) {
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int k = 0; k < V; k++) {
        const float2 t = k < turns[u] ? table[(PAIRS ? e[u][0] / 2 : e[u][0]) + k] : make_float2(1.f, 0.f);
        constexpr bool across = V == 1 || !PAIRS;
        const float wa = across ? w[u][0][k] : w[u][k / ((V + 1) / 2)][(2 * k) % V], wb = across ? w[u][1][k] : w[u][k / ((V + 1) / 2)][(2 * k + 1) % V];
        ca[u][k] = t.x * wa; sa[u][k] = t.y * wa; cb[u][k] = t.x * wb; sb[u][k] = -t.y * wb;
      }
  }
  __device__ __forceinline__ void turn_weighted(const RotaryParams& p, float (&v)[NU][2][V], float f) const {
#pragma unroll
    for (int u = 0; u < NU; u++) {
      if constexpr (V == 1 || !PAIRS) {
        // pieces turn as a whole or pass as a whole; sb carries its sign
        float a[V], b[V];
        rot_scale<V>(a, v[u][0], f);
        rot_scale<V>(b, v[u][1], f);
        rot_mul<V>(v[u][0], a, ca[u]);
        rot_mul<V>(v[u][1], b, cb[u]);
        if (turns[u] > 0) {
          rot_fma<V>(v[u][0], b, sb[u], v[u][0]);
          rot_fma<V>(v[u][1], a, sa[u], v[u][1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) {
          float &px = v[u][k / (V / 2)][2 * (k % (V / 2))], &py = v[u][k / (V / 2)][2 * (k % (V / 2)) + 1];
          const float a = px * f, b = py * f;
          float x = a * ca[u][k], y = b * cb[u][k];
          if (k < turns[u]) { x = fmaf(b, sb[u][k], x); y = fmaf(a, sa[u][k], y); }
          px = x; py = y;
        }
      }
    }
  }
  // pairs that pass are left alone: with a cosine of 1 and a sine of 0 an infinity in one element would make the other NaN
  __device__ __forceinline__ void turn(const RotaryParams& p, float (&v)[NU][2][V]) const {
#pragma unroll
    for (int u = 0; u < NU; u++) {
      if constexpr (V == 1 || !PAIRS) {
        if (turns[u] > 0) {
          float a[V], b[V];
          rot_mul<V>(a, v[u][1], sn[u]);
          rot_mul<V>(b, v[u][0], sn[u]);
          if constexpr (V == 1) a[0] = -a[0];
          else {
#pragma unroll
            for (int j = 0; j < V; j += 2) rot_put(a + j, rot_neg2(rot_two(a + j)));
          }
          rot_fma<V>(v[u][0], v[u][0], cs[u], a);
          rot_fma<V>(v[u][1], v[u][1], cs[u], b);
        }
      } else {
#pragma unroll
        for (int k = 0; k < V; k++) {
          float &x = v[u][k / (V / 2)][2 * (k % (V / 2))], &y = v[u][k / (V / 2)][2 * (k % (V / 2)) + 1];
          const float a = x, b = y;
          if (k < turns[u]) { x = a * cs[u][k] - b * sn[u][k]; y = b * cs[u][k] + a * sn[u][k]; }
        }
      }
    }
  }
  static __device__ __forceinline__ float dot(const float (&a)[NU][2][V], const float (&b)[NU][2][V], int lanes) {
    float s[2][V];
#pragma unroll
    for (int k = 0; k < 2; k++) {
      rot_mul<V>(s[k], a[0][k], b[0][k]);
#pragma unroll
      for (int u = 1; u < NU; u++) rot_fma<V>(s[k], a[u][k], b[u][k], s[k]);
    }
    float t = 0.f;
    if constexpr (V == 1) t = s[0][0] + s[1][0];
    else {
      uint64_t q = add2(rot_two(s[0]), rot_two(s[1]));
#pragma unroll
      for (int j = 2; j < V; j += 2) q = add2(q, add2(rot_two(s[0] + j), rot_two(s[1] + j)));
      uint32_t x, y;
      unpack2(q, x, y);
      t = __uint_as_float(x) + __uint_as_float(y);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) if (off < lanes) t += __shfl_xor_sync(0xffffffffu, t, off);
    return t;
  }
};

__device__ __forceinline__ int64_t rot_at(const B2xHeadStrides& s, int b, int h, int t) { return (int64_t)b * s.batch + (int64_t)h * s.head + (int64_t)t * s.token; }

// A warp: one token (of this CTA's eight), and the heads of share blockIdx.y of all its heads
template <int EL, int V, int NU, bool PAIRS>
__global__ void __launch_bounds__(kRotaryWarps * 32, 2) k_rotary(const __grid_constant__ RotaryParams p) {
  __shared__ float2 table[kRotaryWarps][128];
  constexpr int ES = EL == EL_F32 ? 4 : 2;
  constexpr int ROWS = NU == 1 ? kRotaryRows : 1;
  using Lane = RotLane<EL, V, NU, PAIRS>;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t token = blockIdx.x * kRotaryWarps + warp;
  if (token >= (uint32_t)p.tokens) return;
  const int b = (int)(token / (uint32_t)p.S), t = (int)(token - (uint32_t)b * (uint32_t)p.S);
  const int slots = 32 / p.lanes, slot = lane / p.lanes;
  Lane me;
  me.pieces(p, lane & (p.lanes - 1));
  bool angles = false;
#pragma unroll 1
  for (int ti = 0; ti < 2; ti++) {
    // this share's heads of the tensor
    const int h_begin = max((int)blockIdx.y * p.job_heads - (ti ? p.heads[0] : 0), 0), h_end = min(((int)blockIdx.y + 1) * p.job_heads - (ti ? p.heads[0] : 0), p.heads[ti]);
    if (h_begin >= h_end) continue;
    const char* in = p.x[ti] + rot_at(p.xs[ti], b, h_begin + slot, t) * ES;
    char* out = p.y[ti] + rot_at(p.ys[ti], b, h_begin + slot, t) * ES;
    const int64_t in_step = p.xs[ti].head * ES * slots, out_step = p.ys[ti].head * ES * slots;
    int left = h_end - h_begin - slot;             // heads from this slot's next on
    typename Lane::Raw raw[ROWS][NU][2];
    // the first heads are on their way while the angles are worked out
#pragma unroll
    for (int r = 0; r < ROWS; r++) { me.load(in, left > r * slots, raw[r]); in += in_step; }
    if (!angles) { me.angles(p, (int)token, table[warp]); angles = true; }
    me.weights(p, ti);
    me.fold(p, table[warp]);
    for (int n = h_begin; n < h_end; n += ROWS * slots) {
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        float v[NU][2][V];
        Lane::floats(raw[r], v);
        me.load(in, left > ROWS * slots, raw[r]);
        in += in_step;
        const float f = p.norm ? rsqrtf(Lane::dot(v, v, p.lanes) * p.inv_d + p.epsilon) : 1.f;
        me.turn_weighted(p, v, f);
        if (left > 0) me.store(out, v);
        out += out_step;
        left -= slots;
      }
    }
  }
}

// Gradient with norms: tensor blockIdx.y; a warp walks tokens in steps of the grid and keeps its elements' share of dw
template <int EL, int V, int NU, bool PAIRS>
__global__ void __launch_bounds__(kRotaryWarps * 32, 2) k_rotary_gradient(const __grid_constant__ RotaryParams p) {
  __shared__ float2 table[kRotaryWarps][128];
  __shared__ float sums[kRotaryWarps][256];
  constexpr int ES = EL == EL_F32 ? 4 : 2;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ti = blockIdx.y;
  const int slots = 32 / p.lanes, slot = lane / p.lanes;
  using Lane = RotLane<EL, V, NU, PAIRS>;
  Lane me;
  me.pieces(p, lane & (p.lanes - 1));
  me.weights(p, ti);
  float dw[NU][2][V];
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int j = 0; j < V; j++) dw[u][s][j] = 0.f;
  const uint32_t jobs = (uint32_t)((p.heads[ti] + p.job_heads - 1) / p.job_heads), work = (uint32_t)p.tokens * jobs;
  for (uint32_t id = blockIdx.x * kRotaryWarps + warp; id < work; id += gridDim.x * kRotaryWarps) {
    const int token = (int)(jobs == 1 ? id : id / jobs);
    const int first = (int)(id - (uint32_t)token * jobs) * p.job_heads, last = min(first + p.job_heads, p.heads[ti]);
    const int b = (int)((uint32_t)token / (uint32_t)p.S), t = token - b * p.S;
    const char* in = p.x[ti] + rot_at(p.xs[ti], b, 0, t) * ES;
    const char* din = p.dy[ti] + rot_at(p.dys[ti], b, 0, t) * ES;
    char* out = p.y[ti] + rot_at(p.ys[ti], b, 0, t) * ES;
    const int64_t in_head = p.xs[ti].head * ES, din_head = p.dys[ti].head * ES, out_head = p.ys[ti].head * ES;
    typename Lane::Raw rx[NU][2], rg[NU][2];
    me.load(in + (first + slot) * in_head, first + slot < last, rx);
    me.load(din + (first + slot) * din_head, first + slot < last, rg);
    me.angles(p, token, table[warp]);
    me.take(p, table[warp]);
    for (int h0 = first; h0 < last; h0 += slots) {
      const int h = h0 + slot, next = h + slots;
      float x[NU][2][V], g[NU][2][V];
      me.floats(rx, x);
      me.floats(rg, g);
      me.load(in + next * in_head, next < last, rx);
      me.load(din + next * din_head, next < last, rg);
      me.turn(p, g);
      const float f = rsqrtf(Lane::dot(x, x, p.lanes) * p.inv_d + p.epsilon);
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          rot_scale<V>(x[u][s], x[u][s], f);
          if (h < last) rot_fma<V>(dw[u][s], g[u][s], x[u][s], dw[u][s]);
          rot_mul<V>(g[u][s], g[u][s], me.w[u][s]);
        }
      const float m = Lane::dot(x, g, p.lanes) * p.inv_d;
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
          rot_fma<V>(g[u][s], x[u][s], -m, g[u][s]);
          rot_scale<V>(g[u][s], g[u][s], f);
        }
      if (h < last) me.store(out + h * out_head, g);
    }
  }
  // the warp's slots, then the CTA's warps, in a fixed order
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int j = 0; j < V; j++) {
        float d = dw[u][s][j];
        for (int off = p.lanes; off < 32; off <<= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
        if (slot == 0 && me.e[u][s] >= 0) sums[warp][me.e[u][s] + j] = d;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < p.D; i += kRotaryWarps * 32) {
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < kRotaryWarps; k++) d += sums[k][i];
    p.partial[((int64_t)ti * gridDim.x + blockIdx.x) * p.D + i] = d;
  }
}

// dw[i] = sum of the CTAs' partial sums: 32 columns per CTA, 32 threads per column
__global__ void __launch_bounds__(1024) k_rotary_fold(const float* partial, float* dw0, float* dw1, int rows, int D) {
  __shared__ float part[32][33];
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), r = threadIdx.x >> 5;
  const float* src = partial + (int64_t)blockIdx.y * rows * D;
  // sixteen loads of a thread in flight: the CTAs are few
  float s = 0.f;
  for (int i = r; i < rows; i += 32 * 16) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; k++) v[k] = c < D && i + 32 * k < rows ? ld_global(src + (int64_t)(i + 32 * k) * D + c) : 0.f;
#pragma unroll
    for (int k = 0; k < 16; k++) s += v[k];
  }
  part[r][threadIdx.x & 31] = s;
  __syncthreads();
  if (r == 0 && c < D) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; i++) t[i & 3] += part[i][threadIdx.x];
    (blockIdx.y ? dw1 : dw0)[c] = (t[0] + t[1]) + (t[2] + t[3]);
  }
}

int rot_elem_size(uint8_t e) { return e == EL_F32 ? 4 : 2; }

bool rot_valid(const B2xRotaryArgs* a, bool gradient) {
  constexpr int64_t most = 1ll << 31;
  const int64_t es = rot_elem_size(a->elem);
  auto at = [](const void* p, int64_t size) { return p && (uintptr_t)p % (size_t)size == 0; };
  if (!((a->elem == EL_BF16 || a->elem == EL_F16 || a->elem == EL_F32) && (a->weight_elem == EL_F32 || a->weight_elem == a->elem || !a->norm) && (a->n == 1 || a->n == 2) &&
        a->B >= 0 && a->B < most && a->S >= 0 && a->S < most && a->B * a->S < most && a->D >= 0 && a->D <= 256 && a->R >= 0 && a->R <= a->D && a->R % 2 == 0)) return false;
  if ((uintptr_t)a->positions % 4 != 0) return false;
  bool any = false;
  for (int i = 0; i < a->n; i++) {
    if (a->heads[i] < 0 || a->heads[i] >= (1 << 20)) return false;
    if (a->D > 0 && a->norm && gradient && !at(a->dweight[i], 4)) return false;
    if (a->B * a->S * a->D > 0 && a->norm && !at(a->weight[i], a->weight_elem == EL_F32 ? 4 : 2)) return false;
    if (a->B * a->S * a->heads[i] * a->D == 0) continue;
    any = true;
    if (!at(a->y[i], es) || ((!gradient || a->norm) && !at(a->x[i], es)) || (gradient && !at(a->dy[i], es))) return false;
  }
  return (!any || a->R == 0 || at(a->turns, 8)) && (!gradient || !a->norm || a->D == 0 || at(a->scratch, 4));
}

// Elements of a piece: 16 bytes where rows, pieces and partners start on that boundary, else 8 for 16-bit types, else one element.
int rot_piece(const B2xRotaryArgs* a, bool gradient) {
  const int es = rot_elem_size(a->elem);
  for (int v = 16 / es; v >= 4; v /= 2) {
    bool ok = a->D % v == 0 && (a->interleaved || (a->R / 2) % v == 0);
    auto row = [&](const void* p, const B2xHeadStrides& s) {
      if ((uintptr_t)p % (size_t)(v * es) != 0 || s.batch % v != 0 || s.head % v != 0 || s.token % v != 0) ok = false;
    };
    for (int i = 0; i < a->n; i++) {
      row(a->y[i], a->ys[i]);
      if (a->x[i]) row(a->x[i], a->xs[i]);
      if (gradient && a->dy[i]) row(a->dy[i], a->dys[i]);
    }
    if (ok) return v;
  }
  return 1;
}

RotaryParams rot_params(const B2xRotaryArgs* a, int V, bool each) {
  RotaryParams p{};
  p.positions = a->positions; p.turns = a->turns;
  p.tokens = (int32_t)(a->B * a->S); p.S = (int32_t)a->S; p.D = (int32_t)a->D; p.R = (int32_t)a->R;
  p.epsilon = a->epsilon; p.inv_d = 1.0f / (float)a->D; p.sine = 1.f;
  p.norm = a->norm; p.weight_f32 = a->weight_elem == EL_F32;
  p.weight_wide = 1;
  for (int i = 0; i < a->n; i++) if ((uintptr_t)a->weight[i] % 16 != 0) p.weight_wide = 0;
  const int pieces = (p.D + V - 1) / V;
  p.pair_units = a->interleaved ? 0 : p.R / 2 / V;
  p.units = a->interleaved ? (pieces + 1) / 2 : p.pair_units + (pieces - 2 * p.pair_units + 1) / 2;
  p.lanes = 1;
  while (p.lanes < p.units && p.lanes < 32) p.lanes *= 2;
  for (int i = 0; i < a->n; i++) {
    p.x[i] = (const char*)a->x[i]; p.xs[i] = a->xs[i];
    p.dy[i] = (const char*)a->dy[i]; p.dys[i] = a->dys[i];
    p.y[i] = (char*)a->y[i]; p.ys[i] = a->ys[i];
    p.weight[i] = (const char*)a->weight[i];
    p.heads[i] = (int32_t)a->heads[i];
  }
  // a warp walks all heads of its token, unless that leaves SMs without work: then as few as one round of its slots
  const int slots = 32 / p.lanes;
  const int most = each ? (p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1]) : p.heads[0] + p.heads[1];
  p.job_heads = (most + slots - 1) / slots * slots;
  if (p.job_heads < slots) p.job_heads = slots;
  while (p.job_heads > slots && (int64_t)p.tokens * ((most + p.job_heads - 1) / p.job_heads) < (int64_t)kNumSms * 16) p.job_heads = (p.job_heads / 2 + slots - 1) / slots * slots;
  return p;
}

int rot_gradient_ctas(const RotaryParams& p) {
  const int most = p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1];
  const int64_t ctas = ((int64_t)p.tokens * ((most + p.job_heads - 1) / p.job_heads) + kRotaryWarps - 1) / kRotaryWarps;
  return (int)(ctas < 1 ? 1 : ctas > kNumSms * 3 ? kNumSms * 3 : ctas);
}

template <int EL, int V, int NU, bool PAIRS>
int launch_rot_as(const B2xRotaryArgs* a, const RotaryParams& p, bool norm_gradient, cudaStream_t stream) {
  cudaError_t e;
  if (norm_gradient) e = launch_overlapped(k_rotary_gradient<EL, V, NU, PAIRS>, dim3((unsigned)rot_gradient_ctas(p), a->n), dim3(kRotaryWarps * 32), 0, stream, p);
  else {
    const unsigned jobs = (unsigned)((p.heads[0] + p.heads[1] + p.job_heads - 1) / p.job_heads);
    e = launch_overlapped(k_rotary<EL, V, NU, PAIRS>, dim3(((unsigned)p.tokens + kRotaryWarps - 1) / kRotaryWarps, jobs), dim3(kRotaryWarps * 32), 0, stream, p);
  }
  if (e != cudaSuccess) return (int)e;
  count_launch();
  return (int)cudaGetLastError();
}
template <int EL, int V, int NU>
int launch_rot(const B2xRotaryArgs* a, const RotaryParams& p, bool norm_gradient, cudaStream_t stream) {
  return a->interleaved ? launch_rot_as<EL, V, NU, true>(a, p, norm_gradient, stream) : launch_rot_as<EL, V, NU, false>(a, p, norm_gradient, stream);
}
template <int EL>
int launch_rot(const B2xRotaryArgs* a, const RotaryParams& p, int V, bool norm_gradient, cudaStream_t stream) {
  if constexpr (EL == EL_F32) {
    if (V == 4) return launch_rot<EL, 4, 1>(a, p, norm_gradient, stream);
  } else {
    if (V == 8) return launch_rot<EL, 8, 1>(a, p, norm_gradient, stream);
    if (V == 4) return launch_rot<EL, 4, 1>(a, p, norm_gradient, stream);
  }
  return launch_rot<EL, 1, 4>(a, p, norm_gradient, stream);
}
int launch_rot(const B2xRotaryArgs* a, const RotaryParams& p, int V, bool norm_gradient, cudaStream_t stream) {
  if (a->elem == EL_F32) return launch_rot<EL_F32>(a, p, V, norm_gradient, stream);
  if (a->elem == EL_BF16) return launch_rot<EL_BF16>(a, p, V, norm_gradient, stream);
  return launch_rot<EL_F16>(a, p, V, norm_gradient, stream);
}

}  // namespace
}  // namespace b2x

extern "C" int b2x_launch_rotary(const B2xRotaryArgs* a, b2x_stream_t stream) {
  using namespace b2x;
  if (!rot_valid(a, false)) return (int)cudaErrorInvalidValue;
  if (a->D == 0) return 0;
  const int V = rot_piece(a, false);
  const RotaryParams p = rot_params(a, V, false);
  if (p.tokens == 0 || p.heads[0] + p.heads[1] == 0) return 0;
  return launch_rot(a, p, V, false, (cudaStream_t)stream);
}

extern "C" int64_t b2x_rotary_scratch_bytes(const B2xRotaryArgs* a) {
  // the most CTAs of any piece size: addresses are not known yet when a program is compiled
  return a->norm ? (int64_t)a->n * b2x::kNumSms * 3 * a->D * 4 : 0;
}

extern "C" int b2x_rotary_launches(const B2xRotaryArgs* a, int gradient) {
  if (a->D == 0) return 0;
  if (gradient && a->norm) return a->B * a->S == 0 ? 1 : 2;
  return a->B * a->S * (a->heads[0] + a->heads[1]) > 0 ? 1 : 0;
}

extern "C" int b2x_launch_rotary_gradient(const B2xRotaryArgs* a, b2x_stream_t stream) {
  using namespace b2x;
  if (!rot_valid(a, true)) return (int)cudaErrorInvalidValue;
  if (a->D == 0) return 0;
  const int V = rot_piece(a, true);
  RotaryParams p = rot_params(a, V, a->norm);
  p.sine = -1.f;
  if (!a->norm) {
    // the rotation's transpose: the same kernel, turned the other way
    for (int i = 0; i < a->n; i++) { p.x[i] = p.dy[i]; p.xs[i] = p.dys[i]; }
    if (p.tokens == 0 || p.heads[0] + p.heads[1] == 0) return 0;
    return launch_rot(a, p, V, false, (cudaStream_t)stream);
  }
  p.partial = (float*)a->scratch;
  const int rows = p.tokens > 0 ? rot_gradient_ctas(p) : 0;
  if (rows > 0) {
    const int rc = launch_rot(a, p, V, true, (cudaStream_t)stream);
    if (rc) return rc;
  }
  const cudaError_t e = launch_overlapped(k_rotary_fold, dim3((unsigned)((p.D + 31) / 32), a->n), dim3(1024), 0, (cudaStream_t)stream, (const float*)p.partial,
                                          a->dweight[0], a->dweight[1], rows, p.D);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  return (int)cudaGetLastError();
}
