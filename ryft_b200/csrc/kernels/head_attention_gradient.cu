// The gradient of attention (head_attention.cu) on the tensor cores.
//
// Three launches, or up to five, after the ranges of documents: the row constants (delta = sum dO O, and the log sum in log2 units), dQ per tile of
// 128 queries, dK and dV per tile of 128 keys.  Both tile kernels compute scores again: seven products of a block of 128 x 128 in
// all where one kernel that adds dQ in memory would need five, but no sum depends on the order in which CTAs run, and no f32 copy
// of dQ is written and read.
//
// Where there are fewer tiles than SMs (few heads, short sequences) a tile's walk is cut into parts whose sums a further launch joins.
//
// Both are one kernel, k_attention_gradient: a tile of 128 rows (queries with their dO; or keys with their values) stays in shared
// memory, units of 64 of the other side pass by in five stages (eight at a width of 64).  Two products per unit, S and dP (transposed
// for keys), go into one of two or three pairs of TMEM buffers of 64 columns, so that four warps turn one pair into P and dS while the
// tensor pipe works for the others.
// P and dS are written in place as 16-bit words (a row's words take columns that it has read) and are the left operands of the
// second products, dQ += dS K, or dV += P^T dO and dK += dS^T Q: they never pass through shared memory, whose bandwidth bounds
// the products.  Accumulators and buffers fill TMEM at a width of 128.  Query heads that share a key head follow one another into the
// same accumulators of dK and dV.
//
// Rounded to 16 bits on the way: P and dS as those operands, and O, which delta is taken from as the caller hands it in.  Against 64 bits
// dq and dk are off by 2.6e-3 of their norm (bf16; 1.7e-3 is the rounding of the results alone), by up to 3.8e-3 where queries see a few
// dozen keys and dS is a difference of near equals.
//
// The arithmetic of a unit is a loop over 16 columns whose body is one of nine forms (cap, bias, mask), chosen once per unit: with
// the four steps unrolled, or with the forms' branches inside, the warps waited for instructions more than for anything else
// (dK and dV of 2 x 16/4 heads, 4096 x 128, causal, capped: 505 us with branches inside, 416 unrolled, 336 as a loop).
//
// What bounds it: a product of 128 x 64 x 16 takes the tensor pipe 48 cycles where both operands come from shared memory (32 would be
// its arithmetic; the rows of the tile are read again for every unit), so a unit cannot take less than 1003 cycles for dQ and
// 1259 for dK and dV.  At that size dQ takes 201 us, about 30 % above its products, and dK and dV 273 us, 50 % above: with two
// pairs a unit's arithmetic is on the way from its scores to its sums.  Capped they take 242 and 313 us: the cap's polynomial and its
// derivative double the instructions for the FMA pipe.  Both kernels and the row constants: 470 us, 731 TFLOP/s of the gradient's
// five products; capped 548 us; f16 17 us more, for the lengths of dO and V and the launches that no longer overlap.
//
// f16: P (dP - delta) passes f16's range at both ends where the gradients do not, so that it is rounded as a multiple of a power of
// two that its size allows (grad_shift): |P (dP - delta)| = P |dO (V - O)| <= 2 |dO| max|V|, as lengths of rows, is brought below f16's
// largest value, for dQ row by row, for dK with the largest dO of all query heads that share the key head.  The row constants' kernel
// finds the lengths (V is read once more); the factor sits in the sum dP - delta, and leaves with the last product.
//
// 384 threads, 512 with three pairs: warp 0 draws tiles and loads (TMA), warp 1 issues the MMAs, warps 4 and up do the arithmetic.
#include <atomic>
#include <type_traits>

#include "head_attention_tc.cuh"

namespace b2x {
namespace {

constexpr int GRAD_UNIT = 64;         // keys (dQ) or queries (dK, dV) per step

struct GradParams {
  HeadAttn a;
  const int2* ranges;                 // documents' ranges per block of 128 tokens; NULL: no documents, or too long to list
  const float* neg_lse;               // [B, Hq, rows]: -log sum in log2 units (-inf: nothing seen, or behind the last query)
  const float* neg_delta;             // [B, Hq, rows]
  int32_t rows;                       // queries, rounded up to 128
  int32_t tiles, group_heads, key_blocks, total, parts;   // total: tiles of all heads, times the parts of each (grad_parts)
  float* partial;                     // parts' sums: [part][tile][dQ, or dV and dK][128][D]
  uint64_t in2;                       // scale * log2(e)
  HeadCap cap;
  float scale;
  const float* row_size;              // f16: [B, Hq, rows] squared lengths of the rows of dO
  const float2* head_size;            // f16: [B, Hk] their largest over all queries that see something, and that of the rows of V within the length
  uint32_t idesc_s, idesc_acc;
};

// The power of two that P (dP - delta) is divided by, from the squared lengths of dO and V (1 % for their roundings and P's).  0
// where there is nothing to go by: zeros, and infinities or NaN, which come out as they are.
__device__ __forceinline__ int grad_shift(float dout, float v) {
  const float most = sqrtf(dout) * sqrtf(v) * (2.02f / 65504.f);
  return most > 0.f && most < INFINITY ? (int)(__float_as_uint(most) >> 23) - 126 : 0;
}
__device__ __forceinline__ float grad_power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Document ranges of the tokens at positions [lo, hi], from the blocks that hold them; nothing where there is no such token.
__device__ __forceinline__ int2 grad_range(const GradParams& p, const int2* rs, int lo, int hi) {
  lo = max(lo, 0); hi = min(hi, p.a.Sk - 1);
  if (lo > hi) return make_int2(0x7fffffff, (int)0x80000000);
  const int2 a = ha_range(rs + lo / HA_BLOCK), b = ha_range(rs + hi / HA_BLOCK);
  return make_int2(min(a.x, b.x), max(a.y, b.y));
}

// P and dS of 16 scores of a row as 16-bit words.  nl and nd are the row constants of the pair 2i, 2i + 1; far is the distance of
// the first, bits say which are seen.  f16: dS is worked out times `part`, nd included.  CAP: 0 none, 1 by the polynomial, 2 any.
template <int EL, int CAP, bool SLOPE, bool MASK, typename L, typename N>
__device__ __forceinline__ void grad_words(const GradParams& p, const uint32_t (&s)[16], const uint32_t (&dp)[16], const L& nl, const N& nd, float slope, float far, uint32_t bits,
                                           float part, uint32_t (&pw)[8], uint32_t (&dw)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) {
    uint64_t x2, bend2 = 0;
    const uint64_t s2 = pack2(s[2 * i], s[2 * i + 1]);
    uint32_t a0, a1;
    if constexpr (CAP == 1) {
      const uint64_t t2 = cap_small(p.cap, mul2(s2, p.cap.in2));
      bend2 = fma2(mul2(t2, t2), p.cap.back2, splat2(1.f));
      x2 = add2(t2, nl(i));
    } else if constexpr (CAP == 2) {
      const uint64_t c2 = mul2(s2, p.cap.in2);
      uint64_t e2;
      const uint64_t q2 = cap_rest<true>(c2, e2);
      // 1 - tanh^2 = 4 e^2x q^2
      bend2 = mul2(mul2(mul2(e2, q2), q2), splat2(4.f));
      x2 = add2(cap_choose(p.cap, c2, q2), nl(i));
    } else {
      x2 = fma2(s2, p.in2, nl(i));
    }
    unpack2(x2, a0, a1);
    float x0 = __uint_as_float(a0), x1 = __uint_as_float(a1);
    if constexpr (SLOPE) { x0 = fmaf(fabsf(far - (float)(2 * i)), -slope, x0); x1 = fmaf(fabsf(far - (float)(2 * i + 1)), -slope, x1); }
    const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
    uint64_t d2 = pack2(dp[2 * i], dp[2 * i + 1]);
    if constexpr (EL == EL_F16) d2 = fma2(d2, splat2(part), nd(i));
    else d2 = add2(d2, nd(i));
    d2 = mul2(pack2(__float_as_uint(p0), __float_as_uint(p1)), d2);
    if constexpr (CAP != 0) d2 = mul2(d2, bend2);
    unpack2(d2, a0, a1);
    pw[i] = ha_pack<EL>(p0, p1);
    dw[i] = ha_pack<EL>(__uint_as_float(a0), __uint_as_float(a1));
    if constexpr (MASK) {
      // both words' halves: what is not seen is 0, whatever was computed there
      const uint32_t keep = ((bits >> (2 * i)) & 1u ? 0xffffu : 0u) | ((bits >> (2 * i + 1)) & 1u ? 0xffff0000u : 0u);
      pw[i] &= keep; dw[i] &= keep;
    }
  }
}
// Runs body<CAP, SLOPE, MASK>: every form is a stretch of straight code of its own, chosen once per block, because branches inside it
// left the warps waiting for instructions.
template <typename F> __device__ __forceinline__ void grad_choose(int cap, bool slope, bool mask, const F& body) {
  using std::integral_constant;
#define B2X_GRAD_FORM(C, S, M) body(integral_constant<int, C>{}, integral_constant<bool, S>{}, integral_constant<bool, M>{})
#define B2X_GRAD_CAP(C) if (slope) B2X_GRAD_FORM(C, true, true); else if (mask) B2X_GRAD_FORM(C, false, true); else B2X_GRAD_FORM(C, false, false)
  if (cap == 1) { B2X_GRAD_CAP(1); }
  else if (cap == 0) { B2X_GRAD_CAP(0); }
  else { B2X_GRAD_CAP(2); }
#undef B2X_GRAD_CAP
#undef B2X_GRAD_FORM
}
// Waits for the loads behind two sets of registers; naming them keeps their uses behind the wait.
__device__ __forceinline__ void grad_wait(uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]), "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]),
                 "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15])
               :
               : "memory");
  asm volatile("" : "+r"(b[0]), "+r"(b[1]), "+r"(b[2]), "+r"(b[3]), "+r"(b[4]), "+r"(b[5]), "+r"(b[6]), "+r"(b[7]), "+r"(b[8]), "+r"(b[9]), "+r"(b[10]), "+r"(b[11]),
                    "+r"(b[12]), "+r"(b[13]), "+r"(b[14]), "+r"(b[15])
               :
               : "memory");
}

// Sixteen columns of a row of an accumulator times `f`, as 16-bit values; `width` of them exist
template <int EL>
__device__ __forceinline__ void grad_write(uint32_t taddr, char* row, bool there, int width, float f, bool zero) {
  uint32_t x[16];
  if (!zero) { sm100::tmem_ld_32x16(taddr, x); sm100::tc_wait_ld(); }
  else {
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = 0;
  }
  uint32_t wd[8];
#pragma unroll
  for (int k = 0; k < 8; k++) wd[k] = ha_pack<EL>(__uint_as_float(x[2 * k]) * f, __uint_as_float(x[2 * k + 1]) * f);
  if (there) ha_store_row(row, width, wd);
}

// The same as f32, of a part of the tile's units
__device__ __forceinline__ void grad_part(uint32_t taddr, float* row, float f, bool zero) {
  uint32_t x[16];
  if (!zero) { sm100::tmem_ld_32x16(taddr, x); sm100::tc_wait_ld(); }
  else {
#pragma unroll
    for (int i = 0; i < 16; i++) x[i] = 0;
  }
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    *(float4*)(row + i) = make_float4(__uint_as_float(x[i]) * f, __uint_as_float(x[i + 1]) * f, __uint_as_float(x[i + 2]) * f, __uint_as_float(x[i + 3]) * f);
}

// Parts that a tile's units are cut into.  Where there are fewer tiles than SMs, the longest walk takes the whole time; parts of nine
// units and more, as many as fill the SMs (twice under a causal mask, which leaves half of the units), are summed in f32 and joined in
// their order by k_gradient_join.  Whole gradients, causal: 8 query heads of one key head, 4096 x 128, 534 -> 150 us; 16/4 heads, 2048 x 128,
// 167 -> 101; 2 heads, 3766 x 80, cap and bias, 151 -> 91.  4 heads, 1024 x 128, without a mask: two parts of eight units 47 us, one 46.
template <typename Args> int grad_parts(const Args& a, bool keys) {
  const int64_t tiles = (int64_t)a.B * (keys ? a.Hk : a.Hq) * (((keys ? a.Sk : a.Sq) + HA_BLOCK - 1) / HA_BLOCK);
  const int64_t units = (((keys ? a.Sq : a.Sk) + GRAD_UNIT - 1) / GRAD_UNIT) * (keys && a.Hk > 0 ? a.Hq / a.Hk : 1);
  if (tiles <= 0) return 1;
  int64_t parts = (a.causal ? 2 : 1) * kNumSms / tiles;
  if (parts > units / 9) parts = units / 9;
  return parts < 1 ? 1 : (int)(parts < 16 ? parts : 16);
}
// bytes of the parts' sums of one side
template <typename Args> int64_t grad_part_bytes(const Args& a, bool keys) {
  const int parts = grad_parts(a, keys);
  return parts == 1 ? 0 : (int64_t)parts * a.B * (keys ? 2 * a.Hk : a.Hq) * (((keys ? a.Sk : a.Sq) + HA_BLOCK - 1) / HA_BLOCK) * HA_BLOCK * (a.D <= 64 ? 64 : 128) * 4;
}

// One warp per row: the parts' sums in their order, as 16-bit values
template <int D, int EL, bool KEYS>
__global__ void __launch_bounds__(256) k_gradient_join(const __grid_constant__ GradParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int col = (threadIdx.x & 31) * 4;
  const int64_t tiles = p.total / p.parts;
  const int heads = KEYS ? p.a.Hk : p.a.Hq, tokens = KEYS ? p.a.Sk : p.a.Sq;
  const int row = (int)(id % HA_BLOCK);
  const int64_t rest = id / HA_BLOCK, tile = KEYS ? rest >> 1 : rest;
  const bool second = KEYS && (rest & 1);
  const int bh = (int)(tile / p.tiles), token = (int)(tile - (int64_t)bh * p.tiles) * HA_BLOCK + row, b = bh / heads, h = bh - b * heads;
  if (tile < tiles && token < tokens && col < p.a.D) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.parts; k++) {
      const uint4 x = ld_global((const uint4*)(p.partial + (((k * tiles + tile) * (KEYS ? 2 : 1) + second) * HA_BLOCK + row) * D + col));
      v.x += __uint_as_float(x.x); v.y += __uint_as_float(x.y); v.z += __uint_as_float(x.z); v.w += __uint_as_float(x.w);
    }
    const B2xHeadStrides& o = !KEYS ? p.a.dqs : second ? p.a.dks : p.a.dvs;
    char* out = (!KEYS ? p.a.dq : second ? p.a.dk : p.a.dv) + 2 * ((int64_t)b * o.batch + (int64_t)h * o.head + (int64_t)token * o.token + col);
    *(uint2*)out = make_uint2(ha_pack<EL>(v.x, v.y), ha_pack<EL>(v.z, v.w));
  }
}

// ---- the tile kernel -------------------------------------------------------------------------------------------------------
// Pairs of score buffers in TMEM, each with four warps of its own: as many as the accumulators leave room for
template <int D, bool KEYS> struct GradShape {
  static constexpr int GROUPS = KEYS && D == 128 ? 2 : 3;
  static constexpr int THREADS = 128 + 128 * GROUPS;
};

template <int D> struct GradSmem {
  static constexpr int T_BYTES = HA_BLOCK * D * 2;         // the tile's Q and dO, or K and V
  static constexpr int U_BYTES = GRAD_UNIT * D * 2;        // a unit's K and V, or Q and dO
  static constexpr int STAGES = D == 64 ? 8 : 5;           // what fits; the units are there before they are needed
  static constexpr int T0_OFF = 0, T1_OFF = T_BYTES;
  static constexpr int U_OFF = 2 * T_BYTES;                // STAGES x 2
  static constexpr int ROW_OFF = U_OFF + STAGES * 2 * U_BYTES;   // row constants of keys' tiles: groups x 2 turns x (64 + 64) floats
  static constexpr int BAR_OFF = ROW_OFF + GradShape<D, true>::GROUPS * 2 * 512;
  static constexpr int SLOT_OFF = BAR_OFF + 288;            // 18 + 2 x STAGES barriers, TMEM slot, abort flag
  static constexpr int TOTAL = SLOT_OFF + 2 * (int)sizeof(TileSlot);
};

// KEYS: tiles of keys (dK, dV); else tiles of queries (dQ).  t0, t1: Q and dO, or K and V; u0, u1: K and V, or Q and dO.
template <int D, int EL, bool KEYS>
__global__ void __launch_bounds__(GradShape<D, KEYS>::THREADS, 1)
k_attention_gradient(const __grid_constant__ CUtensorMap tmT0, const __grid_constant__ CUtensorMap tmT1, const __grid_constant__ CUtensorMap tmU0,
                     const __grid_constant__ CUtensorMap tmU1, const __grid_constant__ GradParams p, int32_t* sched, int32_t* status) {
  using namespace sm100;
  using SM = GradSmem<D>;
  constexpr int DC = D / 64, STAGES = SM::STAGES, GROUPS = GradShape<D, KEYS>::GROUPS;
  constexpr uint32_t U_CHUNK = GRAD_UNIT * 128;            // one [64 rows x 128 bytes] swizzled sub-tile
  constexpr uint32_t TMEM_COLS = 512;          // pair g: S [128 g, +64), dP [128 g + 64, +64); behind the pairs dQ, or dV and dK
  constexpr uint32_t ACC = GROUPS * 128;
  // swizzled tiles start on 1024 bytes; there is no room to round up to them
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  const uint32_t b0 = sbase + SM::BAR_OFF;
  const uint32_t bar_tl = b0, bar_tu = b0 + 8 /* tile loaded, tile used */, bar_end = b0 + 16, bar_of = b0 + 24, bar_tf = b0 + 32 /* [2] */, bar_te = b0 + 48 /* [2] */,
                 bar_drain = b0 + 64, bar_sf = b0 + 72 /* [3] */, bar_pf = b0 + 96 /* [3] */, bar_rf = b0 + 120 /* [3] */, bar_uf = b0 + 144 /* [STAGES] */,
                 bar_ue = bar_uf + 8 * STAGES;
  uint32_t* tmem_slot = (uint32_t*)(smem + SM::BAR_OFF + 272);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile TileSlot* slots = (volatile TileSlot*)(smem + SM::SLOT_OFF);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool listed = p.ranges != nullptr;
  const int repeat = KEYS ? p.a.group : 1;     // heads that pass by a tile

  if (threadIdx.x == 0) {
    mbar_init(bar_tl, 1); mbar_init(bar_tu, 1); mbar_init(bar_end, 1); mbar_init(bar_of, 4 * GROUPS); mbar_init(bar_drain, 1);
    for (uint32_t s = 0; s < 8 * STAGES; s += 8) { mbar_init(bar_uf + s, 1); mbar_init(bar_ue + s, 1); }
    for (uint32_t s = 0; s < 8 * GROUPS; s += 8) { mbar_init(bar_sf + s, 1); mbar_init(bar_pf + s, 4); mbar_init(bar_rf + s, 4); }
    for (uint32_t s = 0; s < 16; s += 8) { mbar_init(bar_tf + s, 1); mbar_init(bar_te + s, 1 + 4 * GROUPS); }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmT0); tma_prefetch_desc(&tmT1); tma_prefetch_desc(&tmU0); tma_prefetch_desc(&tmU1);
  }
  if (warp == 1) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();          // everything above touched this SM only

  if (warp == 0) {
    // ---------------------------------------------- tiles and loads ------------------------------------------------
    uint32_t uc = 0, nt = 0;       // units loaded, tiles with work
    int fixed = (int)blockIdx.x;
    for (int n = 0;; n++) {
      if (n >= 2 && !ha_barrier_warp(bar_te + 8 * (n & 1), (uint32_t)(((n >> 1) - 1) & 1), abort_flag, status, 61)) break;
      int t = 0;
      if (sched) {
        if (lane == 0) t = atomicAdd(sched, 1);
        t = __shfl_sync(0xffffffffu, t, 0);
      } else { t = fixed; fixed += (int)gridDim.x; }
      if ((sbase & 1023u) != 0) { t = -1; if (lane == 0 && status) atomicCAS(status, 0, 60); }   // nothing is touched
      if (t >= p.total) t = -1;
      volatile TileSlot* s = slots + (n & 1);
      int b = 0, h = 0, at = 0, begin = 0, units = 0;
      HeadSequence seq{};
      if (t >= 0) {
        // the tiles with the most units first: the last queries, the first keys; inside a group of heads that stay in L2 together
        const int all = KEYS ? p.a.Hk : p.a.Hq;
        const int per_group = p.group_heads * p.tiles;
        const int tile = t / p.parts;
        const int g = tile / per_group, in = tile - g * per_group;
        const int heads = min(p.group_heads, p.a.B * all - g * p.group_heads);
        const int rank = in / heads, bh = g * p.group_heads + (in - rank * heads);
        b = bh / all; h = bh - b * all;
        at = (KEYS ? rank : p.tiles - 1 - rank) * HA_BLOCK;
        seq = head_sequence(p.a, b);
        int stop;                                // the unit behind the last
        if constexpr (KEYS) {
          stop = (p.a.Sq + GRAD_UNIT - 1) / GRAD_UNIT;
          if (at >= seq.length) stop = 0;
          else if (p.a.causal && at >= seq.prefix) begin = min(max(at - seq.first, 0) / GRAD_UNIT, stop);
        } else {
          const int last = min(at + HA_BLOCK, p.a.Sq) - 1;
          stop = (max(head_limit(p.a, seq, seq.first + last), 0) + GRAD_UNIT - 1) / GRAD_UNIT;
        }
        units = stop - begin;
        if (listed) {
          const int2* rs = p.ranges + (int64_t)b * p.key_blocks;
          int2 mine;
          if constexpr (KEYS) mine = ha_range(rs + at / HA_BLOCK);
          else mine = grad_range(p, rs, seq.first + at, seq.first + min(at + HA_BLOCK, p.a.Sq) - 1);
          int count = 0;
          for (int i = 0; i < HA_MASK_WORDS; i++) {
            const int k = i * 32 + lane;
            bool visit = false, compare = false;
            if (k >= begin && k < stop) {
              int2 r;
              bool all_there = true;
              if constexpr (KEYS) {
                const int lo = seq.first + k * GRAD_UNIT;
                r = grad_range(p, rs, lo, min(lo + GRAD_UNIT, seq.first + p.a.Sq) - 1);
                all_there = lo >= 0 && lo + GRAD_UNIT <= p.a.Sk;
              } else {
                r = ha_range(rs + k * GRAD_UNIT / HA_BLOCK);
              }
              visit = !ha_apart(mine, r);
              compare = !ha_one_document(mine, r) || !all_there;
            }
            const uint32_t mv = __ballot_sync(0xffffffffu, visit), mc = __ballot_sync(0xffffffffu, compare);
            if (lane == 0) { s->visit[i] = mv; s->compare[i] = mc; }
            count += __popc(mv);
          }
          units = count;
        }
      }
      // this part's share of the units
      const int whole = units * repeat, share = (whole + p.parts - 1) / p.parts, part = t >= 0 ? t % p.parts : 0;
      const int skip = min(part * share, whole), count = min(share, whole - skip);
      if (lane == 0) {
        s->skip = skip; s->count = count; s->part = part;
        s->tile = t; s->b = b; s->h = h; s->at = at; s->begin = begin; s->blocks = units;
        s->length = seq.length; s->first = seq.first; s->prefix = seq.prefix;
        mbar_arrive(bar_tf + 8 * (n & 1));
      }
      __syncwarp();
      if (t < 0) break;
      if (count == 0) continue;
      if (elect_one()) {
        bool ok = nt == 0 || ha_barrier(bar_tu, (nt - 1) & 1, abort_flag, status, 62);
        if (ok) {
          mbar_expect_tx(bar_tl, 2 * SM::T_BYTES);
#pragma unroll
          for (int c = 0; c < DC; c++) {
            tma_load_4d(sbase + SM::T0_OFF + c * HA_CHUNK, &tmT0, bar_tl, c * 64, at, h, b);
            tma_load_4d(sbase + SM::T1_OFF + c * HA_CHUNK, &tmT1, bar_tl, c * 64, at, h, b);
          }
          int hh = skip / units, it = skip - hh * units;
          BlockWalk walk;
          walk.start(s, listed);
          for (int i = 0; i < it; i++) walk.next();
          for (uint32_t k = uc; k < uc + (uint32_t)count; k++) {
            const uint32_t st = k % STAGES, turn = k / STAGES;
            const int uh = KEYS ? h * p.a.group + hh : h / p.a.group;
            if (turn > 0 && !ha_barrier(bar_ue + 8 * st, (turn - 1) & 1, abort_flag, status, 63)) { ok = false; break; }
            mbar_expect_tx(bar_uf + 8 * st, 2 * SM::U_BYTES);
            const uint32_t ua = sbase + SM::U_OFF + st * 2 * SM::U_BYTES;
#pragma unroll
            for (int c = 0; c < DC; c++) {
              tma_load_4d(ua + c * U_CHUNK, &tmU0, bar_uf + 8 * st, c * 64, walk.j * GRAD_UNIT, uh, b);
              tma_load_4d(ua + SM::U_BYTES + c * U_CHUNK, &tmU1, bar_uf + 8 * st, c * 64, walk.j * GRAD_UNIT, uh, b);
            }
            // the next unit, over the end of a head
            if (++it < units) walk.next();
            else { it = 0; hh++; walk.start(s, listed); }
          }
        }
      }
      __syncwarp();
      uc += (uint32_t)count; nt++;
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
    }
  } else if (warp == 1) {
    // ---------------------------------------------- MMA issuer ------------------------------------------------------
    if (elect_one()) {
      // The tensor pipe's queue holds a few products, less work than a wait takes that is over already.  So the questions of the next
      // unit, is the one behind the pairs loaded and are its dS there, are asked in the middle of this one's scores, and their answers
      // are looked at after them; only a no is waited for.  With two pairs the dS are hardly ever there so early, and are not asked
      // for.  dQ of 2 x 16/4 heads, 4096 x 128, causal: 225 -> 201 us; products alone (without waits and arithmetic) would take 140.
      uint32_t stage = 0, stage_parity = 0, pair = 0;      // of the next unit whose scores are issued
      uint32_t held = 0, from_pair = 0, pair_parity = 0;   // of the next unit added to the accumulators
      uint32_t nt = 0;                                     // tiles with work
      const uint32_t dta = ha_desc(sbase + SM::T0_OFF, 16), dtb = ha_desc(sbase + SM::T1_OFF, 16);
      const uint32_t du = ha_desc(sbase + SM::U_OFF, 16), dm = ha_desc(sbase + SM::U_OFF, U_CHUNK);
      bool ok = true, loaded = false, arrived = false;
      auto issue_scores = [&](bool last_of_tile) -> bool {
        if (!loaded && !ha_barrier(bar_uf + 8 * stage, stage_parity, abort_flag, status, 71)) return false;
        tc_fence_after();
        const uint32_t da = du + stage * (2 * SM::U_BYTES / 16), db = da + SM::U_BYTES / 16, to = tmem_base + pair * 128u;
#pragma unroll
        for (int k = 0; k < D / 16; k++) ha_mma(to, dta + ((k >> 2) * HA_CHUNK + (k & 3) * 32) / 16, da + ((k >> 2) * U_CHUNK + (k & 3) * 32) / 16, p.idesc_s, k > 0);
        const uint32_t done = pair;
        if (++stage == STAGES) { stage = 0; stage_parity ^= 1; }
        if (++pair == GROUPS) pair = 0;
        loaded = mbar_test_wait(bar_uf + 8 * stage, stage_parity);
        if (GROUPS > 2) arrived = mbar_test_wait(bar_pf + 8 * from_pair, pair_parity);
#pragma unroll
        for (int k = 0; k < D / 16; k++) ha_mma(to + 64u, dtb + ((k >> 2) * HA_CHUNK + (k & 3) * 32) / 16, db + ((k >> 2) * U_CHUNK + (k & 3) * 32) / 16, p.idesc_s, k > 0);
        tc_commit(bar_sf + 8 * done);
        if (last_of_tile) tc_commit(bar_tu);
        return true;
      };
      for (int n = 0; ok; n++) {
        if (!ha_barrier(bar_tf + 8 * (n & 1), (uint32_t)((n >> 1) & 1), abort_flag, status, 72)) { ok = false; break; }
        const int t = slots[n & 1].tile, total = slots[n & 1].count;
        mbar_arrive(bar_te + 8 * (n & 1));
        if (t < 0) break;
        if (total == 0) continue;
        if (!ha_barrier(bar_tl, nt & 1, abort_flag, status, 73)) { ok = false; break; }
        for (int it = 0; it < GROUPS && it < total && ok; it++) ok = issue_scores(it + 1 == total);
        for (int it = 0; it < total && ok; it++) {
          if (!arrived && !ha_barrier(bar_pf + 8 * from_pair, pair_parity, abort_flag, status, 74)) { ok = false; break; }
          // the previous tile's rows have been read out of the accumulators
          if (it == 0 && nt > 0 && !ha_barrier(bar_of, (nt - 1) & 1, abort_flag, status, 75)) { ok = false; break; }
          tc_fence_after();
          // A = P or dS from TMEM: 16 of the unit are 8 columns; B = the unit's rows (MN-major: chunks of 64 of the width are U_CHUNK apart)
          const uint32_t da = dm + held * (2 * SM::U_BYTES / 16), db = da + SM::U_BYTES / 16, from = tmem_base + from_pair * 128u;
          if constexpr (KEYS) {
#pragma unroll
            for (int k = 0; k < GRAD_UNIT / 16; k++) ha_mma_ts(tmem_base + ACC, from + (uint32_t)(k * 8), db + k * 128, p.idesc_acc, it > 0 || k > 0);
          }
#pragma unroll
          for (int k = 0; k < GRAD_UNIT / 16; k++) ha_mma_ts(tmem_base + ACC + (KEYS ? (uint32_t)D : 0u), from + 64u + (uint32_t)(k * 8), da + k * 128, p.idesc_acc, it > 0 || k > 0);
          tc_commit(bar_ue + 8 * held);
          if (it + 1 == total) tc_commit(bar_end);
          if (++held == STAGES) held = 0;
          if (++from_pair == GROUPS) { from_pair = 0; pair_parity ^= 1; }
          arrived = false;
          // the tensor pipe keeps this thread's order: the pair's next scores come after the products that read it
          if (it + GROUPS < total && !issue_scores(it + GROUPS + 1 == total)) { ok = false; break; }
        }
        nt++;
      }
      // everything this thread issued must retire before TMEM is released
      tc_commit(bar_drain);
      ha_barrier(bar_drain, 0, abort_flag, nullptr, 0);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------- P and dS --------------------------------------------------------
    const int g = (warp - 4) >> 2;                // this group's pair of buffers: every GROUPS-th unit
    const int quad = warp & 3, row = quad * 32 + lane, tid = (int)threadIdx.x - 128 - g * 128;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + (uint32_t)(g * 128);
    uint32_t uc = 0, mine = 0, nt = 0;            // units of all groups before this tile, this group's units, tiles with work
    // A wait inside a tile that runs out lets its lane go on with what is there: the lanes of a warp have to stay together for its
    // votes and TMEM loads.  They leave as one in front of the next tile, which nobody publishes any more.  (Looking for it at the tile's
    // end, or a vote behind every wait, cost 1.5 %.)
    auto wait = [&](uint32_t bar, uint32_t parity, int code) { ha_barrier(bar, parity & 1, abort_flag, status, code); };
    for (int n = 0;; n++) {
      if (!ha_barrier_warp(bar_tf + 8 * (n & 1), (uint32_t)((n >> 1) & 1), abort_flag, status, 81)) break;
      volatile TileSlot* s = slots + (n & 1);
      const int t = s->tile, units = s->blocks, b = s->b, th = s->h, at = s->at;
      const HeadSequence seq{s->length, s->first, s->prefix};
      if (t < 0) break;
      const int total = s->count, skip = s->skip, part = s->part, self = at + row;   // this part's units; this row's query or key
      // queries: keys up to `edge` are seen; keys: queries from `edge` on see this key
      const int pos = KEYS ? self : seq.first + self;
      int edge;
      bool there;
      if constexpr (KEYS) {
        there = self < seq.length;
        edge = !there ? 0x3fffffff : p.a.causal && self >= seq.prefix ? self - seq.first : -0x3fffffff;
      } else {
        there = !p.a.documents || (pos >= 0 && pos < p.a.Sk);
        edge = there ? head_limit(p.a, seq, pos) - 1 : -1;
      }
      const int doc = p.a.documents && pos >= 0 && pos < p.a.Sk ? (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + pos) : 0;
      uint64_t nl2 = 0, nd2 = 0;
      float part_of = 1.f, whole = p.scale;        // f16: dS is held as this part of itself; what the sums are multiplied by
      const int64_t rc = ((int64_t)b * p.a.Hq + th) * p.rows + self;
      if constexpr (EL == EL_F16) {
        if (total > 0) {
          const uint2 size = ld_global((const uint2*)(p.head_size + (int64_t)b * p.a.Hk + (KEYS ? th : th / p.a.group)));
          const int shift = grad_shift(KEYS ? __uint_as_float(size.x) : ld_global(p.row_size + rc), __uint_as_float(size.y));
          part_of = grad_power(-shift); whole *= grad_power(shift);
        }
      }
      if constexpr (!KEYS) { nl2 = splat2(ld_global(p.neg_lse + rc)); nd2 = splat2(ld_global(p.neg_delta + rc) * part_of); }
      BlockWalk walk;
      int hh = 0, it = 0;                          // head that passes by, unit of the head
      // keys: a unit's row constants, one value per thread, fetched a unit ahead
      auto fetch = [&](int head, int unit) {
        const int64_t rc = ((int64_t)b * p.a.Hq + th * p.a.group + head) * p.rows + unit * GRAD_UNIT + (tid & 63);
        return tid < 64 ? ld_global(p.neg_lse + rc) : ld_global(p.neg_delta + rc) * part_of;
      };
      auto advance = [&]() {                       // to the next unit, over the end of a head
        if (++it == units) { it = 0; hh++; if (hh < repeat) walk.start(s, listed); }
        else walk.next();
      };
      int k = 0;
      float ahead = 0.f;
      if (total > 0) {
        hh = skip / units; it = skip - hh * units;
        walk.start(s, listed);
        for (int i = 0; i < it; i++) walk.next();
        for (uint32_t first = ((uint32_t)g + GROUPS - uc % GROUPS) % GROUPS; k < (int)first && k < total; k++) advance();
        if (KEYS && k < total) ahead = fetch(hh, walk.j);
      }
      while (k < total) {
        const int unit = walk.j, head = KEYS ? th * p.a.group + hh : th;
        const uint32_t stage = (uc + (uint32_t)k) % STAGES;
        const bool compare = listed ? (s->compare[unit >> 5] >> (unit & 31)) & 1 : p.a.documents != nullptr;
        const uint32_t rows_at = sbase + (uint32_t)(SM::ROW_OFF + (g * 2 + (int)(mine & 1)) * 512);
        if constexpr (KEYS) {
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(rows_at + (uint32_t)tid * 4), "f"(ahead) : "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_rf + 8 * g);
        }
        for (int i = 0; i < GROUPS && k < total; i++, k++) advance();
        if (KEYS && k < total) ahead = fetch(hh, walk.j);
        // the group's four warps have stored theirs (and read those of two units ago)
        if (KEYS) wait(bar_rf + 8 * g, mine, 84);
        wait(bar_sf + 8 * g, mine, 82);
        tc_fence_after();
        const int u0 = unit * GRAD_UNIT;           // the unit's first key or query
        const float slope = p.a.slopes ? ld_global(p.a.slopes + head) * kLog2e : 0.f;
        const bool masked = compare || __any_sync(0xffffffffu, KEYS ? edge > u0 : edge < u0 + GRAD_UNIT - 1);
        if constexpr (!KEYS) {
          if (p.a.lengths && seq.length < p.a.Sk && seq.length < u0 + GRAD_UNIT) {
            // keys behind the sequence's end: zero before they meet their dS of zero (the scores have been computed: K has landed)
            if (tid < GRAD_UNIT && u0 + tid >= seq.length) {
#pragma unroll 1
              for (int c = 0; c < DC; c++)
#pragma unroll
                for (int q = 0; q < 8; q++) sts_v4(sbase + (uint32_t)SM::U_OFF + stage * 2 * SM::U_BYTES + (uint32_t)(c * U_CHUNK + tid * 128 + q * 16), 0, 0, 0, 0);
            }
            fence_async_shared();
          }
        }
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
        if (masked) {
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const int first = u0 + c * 32;
            seen[c] = KEYS ? ~ha_bits(min(max(edge - first, 0), 32) - 1) : ha_bits(edge - first);
            if (compare) {
              const int other = KEYS ? seq.first + first + lane : first + lane;    // position
              const bool has = other >= 0 && other < p.a.Sk && (!KEYS || first + lane < p.a.Sq);
              const int theirs = has ? (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + other) : 0;
              seen[c] &= ha_same_document(doc, theirs, has);
            }
          }
        }
        int cap = 0;
        if (p.cap.cap > 0.f) {
          uint32_t v[32];
          tmem_ld_32x32(s_addr, v);
          tc_wait_ld();
          float largest = ha_largest(v);
          tmem_ld_32x32(s_addr + 32u, v);
          tc_wait_ld();
          largest = max3(largest, ha_largest(v), 0.f);
          cap = __all_sync(0xffffffffu, largest <= p.cap.small) ? 1 : 2;
        }
        // distance of this row from the unit's first
        const float far = (float)(KEYS ? self - seq.first - u0 : pos - u0);
        grad_choose(cap, slope != 0.f, masked, [&](auto C, auto S, auto M) {
#pragma unroll 1
          for (int c = 0; c < 4; c++) {
            uint32_t sr[16], dr[16], pw[8], dw[8];
            tmem_ld_32x16(s_addr + (uint32_t)(c * 16), sr);
            tmem_ld_32x16(s_addr + 64u + (uint32_t)(c * 16), dr);
            const uint32_t bits = (c < 2 ? seen[0] : seen[1]) >> (16 * (c & 1));
            if constexpr (KEYS) {
              const uint32_t nl_at = rows_at + (uint32_t)(c * 64), nd_at = nl_at + 256;
              uint64_t nlv[8], ndv[8];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                uint32_t w0, w1, w2, w3;
                lds_v4(nl_at + (uint32_t)(i * 16), w0, w1, w2, w3);
                nlv[2 * i] = pack2(w0, w1); nlv[2 * i + 1] = pack2(w2, w3);
                lds_v4(nd_at + (uint32_t)(i * 16), w0, w1, w2, w3);
                ndv[2 * i] = pack2(w0, w1); ndv[2 * i + 1] = pack2(w2, w3);
              }
              grad_wait(sr, dr);
              grad_words<EL, decltype(C)::value, decltype(S)::value, decltype(M)::value>(p, sr, dr, [&](int i) { return nlv[i]; }, [&](int i) { return ndv[i]; }, slope, far - (float)(c * 16),
                                                                                         bits, part_of, pw, dw);
              // words of 16 queries into 8 columns that this row has read
              tmem_st_32x8(s_addr + (uint32_t)(c * 8), pw);
            } else {
              grad_wait(sr, dr);
              grad_words<EL, decltype(C)::value, decltype(S)::value, decltype(M)::value>(p, sr, dr, [&](int) { return nl2; }, [&](int) { return nd2; }, slope, far - (float)(c * 16), bits, part_of, pw, dw);
            }
            tmem_st_32x8(s_addr + 64u + (uint32_t)(c * 8), dw);
          }
        });
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_pf + 8 * g);
        mine++;
      }
      uc += (uint32_t)total;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_te + 8 * (n & 1));   // the tile's list has been walked
      if (total > 0) {
        wait(bar_end, nt, 83);
        tc_fence_after();
        nt++;
      }
      // sixteen columns at a time, the groups in turn: dQ, or dV and then dK
#pragma unroll 1
      for (int c = g; c < (KEYS ? 2 : 1) * (D / 16); c += GROUPS) {
        const bool second = c >= D / 16;
        const int first = (second ? c - D / 16 : c) * 16;
        if (p.parts > 1) {
          const int64_t tiles = p.total / p.parts, tile = ((int64_t)b * (KEYS ? p.a.Hk : p.a.Hq) + th) * p.tiles + at / HA_BLOCK;
          grad_part(tmem_base + lane_addr + ACC + (uint32_t)(c * 16), p.partial + (((part * tiles + tile) * (KEYS ? 2 : 1) + second) * HA_BLOCK + row) * D + first,
                    KEYS && !second ? 1.f : whole, total == 0);
          continue;
        }
        const B2xHeadStrides& o = !KEYS ? p.a.dqs : second ? p.a.dks : p.a.dvs;
        char* out = (!KEYS ? p.a.dq : second ? p.a.dk : p.a.dv) + 2 * ((int64_t)b * o.batch + (int64_t)th * o.head + (int64_t)self * o.token + first);
        grad_write<EL>(tmem_base + lane_addr + ACC + (uint32_t)(c * 16), out, self < (KEYS ? p.a.Sk : p.a.Sq), p.a.D - first, KEYS && !second ? 1.f : whole, total == 0);
      }
      tc_fence_before();
      __syncwarp();
      if (total > 0 && lane == 0) mbar_arrive(bar_of);
    }
  }

  ha_linger(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc(tmem_base, TMEM_COLS); }
  // the last CTA to leave puts the tile counter back for the stream's next launch
  if (sched && threadIdx.x == 0 && atomicAdd(sched + 1, 1) == (int)gridDim.x - 1) { sched[0] = 0; sched[1] = 0; __threadfence(); }
}

// ---- row constants: -log sum in log2 units and -delta; rows behind the last query weigh nothing ---------------------------------
// 32 rows of a head per block (`rows` is a multiple of 128), two per half warp, so that a thread has four loads of 16 bytes in flight;
// a sequence's heads follow one another, for where tokens come before heads their rows are neighbours in memory.  2 x 16 heads of
// 4096 rows of 128, 67 MB: 16 us with nothing in L2 (18 with one row per half warp, head by head).  f16: the squared lengths of the
// rows of dO and, by further blocks, of V; the bits of floats that are not negative are ordered as they are (NaN above infinity), so
// that the largest is one of whole numbers and does not depend on the order in which blocks find it.
template <int EL> __device__ __forceinline__ void rows_floats(const uint4& w, float (&f)[8]) {
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int k = 0; k < 4; k++) {
    float2 u;
    if constexpr (EL == EL_BF16) u = __bfloat1622float2(*(const __nv_bfloat162*)&ws[k]);
    else u = __half22float2(*(const __half2*)&ws[k]);
    f[2 * k] = u.x; f[2 * k + 1] = u.y;
  }
}
// over the half warp that holds a row
__device__ __forceinline__ float rows_dot(const float (&a)[8], const float (&b)[8]) {
  float d = 0.f;
#pragma unroll
  for (int k = 0; k < 8; k++) d = fmaf(a[k], b[k], d);
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
  return d;
}
// Most warps find a larger value there and leave the address to the others.
__device__ __forceinline__ void rows_raise(uint32_t* at, uint32_t most) { if (most > ld_global(at)) atomicMax(at, most); }
template <int EL>
__global__ void __launch_bounds__(256) k_attention_rows(const __grid_constant__ HeadAttn p, float* neg_lse, float* neg_delta, int32_t rows, float* row_size, uint32_t* head_size) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, part = lane & 15;
  const uint32_t per_head = (uint32_t)rows / 32u;
  const int in_block = ((int)(threadIdx.x >> 5) * 2 + (lane >> 4)) * 2;
  if constexpr (EL == EL_F16) {
    const uint32_t query_blocks = (uint32_t)p.B * (uint32_t)p.Hq * per_head;
    if (blockIdx.x >= query_blocks) {
      // 32 rows of a head of V
      const uint32_t key_blocks = ((uint32_t)p.Sk + 31u) / 32u, id = blockIdx.x - query_blocks, head = id / key_blocks;
      const int b = (int)(head / (uint32_t)p.Hk), u = (int)(head - (uint32_t)b * (uint32_t)p.Hk), length = head_sequence(p, b).length;
      const int first = (int)(id - head * key_blocks) * 32 + in_block;
      uint32_t most = 0;
#pragma unroll
      for (int r = 0; r < 2; r++) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (first + r < length && part * 8 < p.D) x = ld_global((const uint4*)(p.v + 2 * ((int64_t)b * p.vs.batch + (int64_t)u * p.vs.head + (int64_t)(first + r) * p.vs.token)) + part);
        float f[8];
        rows_floats<EL>(x, f);
        most = max(most, __float_as_uint(rows_dot(f, f)));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) rows_raise(head_size + 2 * head + 1, most);
      return;
    }
  }
  const uint32_t at = blockIdx.x / (uint32_t)p.Hq;
  const int h = (int)(blockIdx.x - at * (uint32_t)p.Hq), b = (int)(at / per_head), bh = b * p.Hq + h;
  const int first = (int)(at - (uint32_t)b * per_head) * 32 + in_block;
  uint4 x[2], y[2];
#pragma unroll
  for (int r = 0; r < 2; r++) {
    x[r] = y[r] = make_uint4(0, 0, 0, 0);
    if (first + r < p.Sq && part * 8 < p.D) {
      x[r] = ld_global((const uint4*)(p.o + 2 * ((int64_t)b * p.os.batch + (int64_t)h * p.os.head + (int64_t)(first + r) * p.os.token)) + part);
      y[r] = ld_global((const uint4*)(p.dout + 2 * ((int64_t)b * p.dos.batch + (int64_t)h * p.dos.head + (int64_t)(first + r) * p.dos.token)) + part);
    }
  }
  uint32_t most = 0;
#pragma unroll
  for (int r = 0; r < 2; r++) {
    float u[8], v[8];
    rows_floats<EL>(x[r], u);
    rows_floats<EL>(y[r], v);
    const float d = rows_dot(u, v);
    float size = 0.f;
    if constexpr (EL == EL_F16) size = rows_dot(v, v);
    if (part == 0) {
      // a query that saw nothing has a log sum of -inf: its weights are 0
      const bool there = first + r < p.Sq;
      const int64_t id = (int64_t)bh * rows + first + r;
      const float l = there ? ld_global(p.lse + (int64_t)bh * p.Sq + first + r) : -INFINITY;
      neg_lse[id] = l == -INFINITY ? -INFINITY : -l * kLog2e;
      neg_delta[id] = there ? -d : 0.f;
      if constexpr (EL == EL_F16) {
        row_size[id] = size;
        if (l != -INFINITY) most = max(most, __float_as_uint(size));
      }
    }
  }
  if constexpr (EL == EL_F16) {
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) rows_raise(head_size + 2 * ((uint32_t)b * (uint32_t)p.Hk + (uint32_t)(h / p.group)), most);
  }
}

// The tiles of one side: dQ, or with KEYS dK and dV
template <int D, int EL, bool KEYS>
int launch_side(const HeadAttn& a, GradParams p, const int2* ranges, int32_t* status, cudaStream_t stream) {
  static std::atomic<bool> ready[64];
  const int tokens = KEYS ? a.Sk : a.Sq, others = KEYS ? a.Sq : a.Sk;
  if (tokens == 0) return 0;
  const int64_t all = (int64_t)a.B * (KEYS ? a.Hk : a.Hq);
  p.tiles = (tokens + HA_BLOCK - 1) / HA_BLOCK;
  if (all * p.tiles > 0x7fffff00) return (int)cudaErrorInvalidValue;
  p.parts = grad_parts(a, KEYS);
  p.total = (int)(all * p.tiles) * p.parts;
  // what passes by (K and V of a key head, or Q and dO of its query heads) stays in L2 for a group of heads: 32 MiB, as in the
  // forward pass
  const int64_t fit = (32ll << 20) / ((int64_t)(others > 0 ? others : 1) * a.D * 4), heads = KEYS ? fit / a.group : fit * a.group, least = KEYS ? 1 : a.group;
  p.group_heads = (int)(heads < least ? (least < all ? least : all) : heads > all ? all : heads);
  // longer sequences than a list of units covers walk all of theirs, and compare in each
  p.ranges = a.documents && (others + GRAD_UNIT - 1) / GRAD_UNIT <= HA_MASK_WORDS * 32 ? ranges : nullptr;
  const uint32_t format = EL == EL_BF16 ? 1u : 0u;
  p.idesc_s = sm100::make_idesc(format, false, false, HA_BLOCK, GRAD_UNIT);
  p.idesc_acc = sm100::make_idesc(format, false, true, HA_BLOCK, D);
  CUtensorMap t0, t1, u0, u1;
  const uint32_t q_rows = KEYS ? GRAD_UNIT : HA_BLOCK, k_rows = KEYS ? HA_BLOCK : GRAD_UNIT;
  CUtensorMap &q = KEYS ? u0 : t0, &d = KEYS ? u1 : t1, &k = KEYS ? t0 : u0, &v = KEYS ? t1 : u1;
  if (a.Sq > 0 && (!ha_encode(&q, EL, a.q, a.qs, a.B, a.Hq, a.Sq, a.D, q_rows) || !ha_encode(&d, EL, a.dout, a.dos, a.B, a.Hq, a.Sq, a.D, q_rows))) return (int)cudaErrorInvalidValue;
  if (a.Sk > 0 && (!ha_encode(&k, EL, a.k, a.ks, a.B, a.Hk, a.Sk, a.D, k_rows) || !ha_encode(&v, EL, a.v, a.vs, a.B, a.Hk, a.Sk, a.D, k_rows))) return (int)cudaErrorInvalidValue;
  if (others == 0) { u0 = t0; u1 = t1; }      // nothing is loaded
  auto kern = k_attention_gradient<D, EL, KEYS>;
  using SM = GradSmem<D>;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const cudaError_t e = launch_overlapped(kern, dim3((unsigned)(p.total < kNumSms ? p.total : kNumSms)), dim3(GradShape<D, KEYS>::THREADS), SM::TOTAL, stream, t0, t1, u0, u1, p, ha_sched(stream), status);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  if (p.parts > 1) {
    const int64_t rows = (int64_t)(p.total / p.parts) * (KEYS ? 2 : 1) * HA_BLOCK;
    const cudaError_t f = launch_overlapped(k_gradient_join<D, EL, KEYS>, dim3((unsigned)(rows / 8)), dim3(256), 0, stream, p);
    if (f != cudaSuccess) return (int)f;
    count_launch();
  }
  return (int)cudaGetLastError();
}
template <int D, int EL>
int launch_gradient(const HeadAttn& a, const GradParams& p, const int2* ranges, int32_t* status, cudaStream_t stream) {
  const int rc = launch_side<D, EL, false>(a, p, ranges, status, stream);
  return rc ? rc : launch_side<D, EL, true>(a, p, ranges, status, stream);
}

int grad_rows(int64_t Sq) { return (int)((Sq + HA_BLOCK - 1) / HA_BLOCK * HA_BLOCK); }

}  // namespace

// row constants [2][B, Hq, rows], the documents' ranges, for f16 the sizes of heads [B, Hk, 2] and rows [B, Hq, rows], and from a
// multiple of 16 bytes on the sums of parts, of one side at a time
int64_t grad_size_bytes(int elem, int64_t B, int64_t Hq, int64_t Hk, int64_t rows) { return elem == EL_F16 ? B * (Hk * 8 + Hq * rows * 4) : 0; }
int64_t ha_gradient_scratch(const B2xHeadAttentionArgs* a, int64_t ranges) {
  const int64_t rows = grad_rows(a->Sq), head = a->B * a->Hq * rows * 8 + ranges + grad_size_bytes(a->elem, a->B, a->Hq, a->Hk, rows), q = grad_part_bytes(*a, false), k = grad_part_bytes(*a, true);
  return q > 0 || k > 0 ? (head + 15) / 16 * 16 + (q > k ? q : k) : head;
}
int ha_gradient_launches(const B2xHeadAttentionArgs* a) {
  const int q = a->B * a->Hq * a->Sq > 0, k = a->B * a->Hk * a->Sk > 0;
  return (q ? 2 + (grad_parts(*a, false) > 1) : 0) + (k ? 1 + (grad_parts(*a, true) > 1) : 0);
}

// scratch: ha_gradient_scratch
int ha_launch_gradient(const HeadAttn& call, int elem, void* scratch, int32_t* status, cudaStream_t stream) {
  HeadAttn a = call;
  if (a.B == 0 || a.Hk == 0) return 0;
  if (a.Hq == 0) { a.Hq = a.Hk; a.group = 1; a.Sq = 0; }   // keys that no head reads: gradients of zero, as without queries
  GradParams p{};
  p.a = a;
  p.rows = grad_rows(a.Sq);
  const int64_t n = (int64_t)a.B * a.Hq * p.rows;
  p.neg_lse = (const float*)scratch;
  p.neg_delta = p.neg_lse + n;
  int2* ranges = (int2*)(p.neg_delta + n);
  p.key_blocks = (a.Sk + HA_BLOCK - 1) / HA_BLOCK;
  const int64_t fixed = n * 8 + (a.documents ? (int64_t)a.B * p.key_blocks * 8 : 0), heads = (int64_t)a.B * a.Hk;
  uint32_t* head_size = (uint32_t*)((char*)scratch + fixed);
  p.head_size = (const float2*)head_size;
  p.row_size = (const float*)head_size + 2 * heads;
  p.partial = (float*)((char*)scratch + (fixed + grad_size_bytes(elem, a.B, a.Hq, a.Hk, p.rows) + 15) / 16 * 16);
  p.scale = a.scale;
  p.in2 = ha_pair(a.scale * kLog2e);
  p.cap = ha_cap(a.softcap, a.scale);
  if (a.documents) {
    const int rc = ha_launch_ranges(a, ranges, stream);
    if (rc) return rc;
  }
  if (n > 0) {
    int64_t blocks = n / 32;
    if (elem == EL_F16) {
      blocks += heads * ((a.Sk + 31) / 32);
      const cudaError_t z = cudaMemsetAsync(head_size, 0, (size_t)heads * 8, stream);
      if (z != cudaSuccess) return (int)z;
    }
    if (blocks > 0x7fffffff) return (int)cudaErrorInvalidValue;
    const cudaError_t e = launch_overlapped(elem == EL_BF16 ? k_attention_rows<EL_BF16> : k_attention_rows<EL_F16>, dim3((unsigned)blocks), dim3(256), 0, stream, a,
                                            const_cast<float*>(p.neg_lse), const_cast<float*>(p.neg_delta), p.rows, const_cast<float*>(p.row_size), head_size);
    if (e != cudaSuccess) return (int)e;
    count_launch();
  }
  if (a.D <= 64) return elem == EL_BF16 ? launch_gradient<64, EL_BF16>(a, p, ranges, status, stream) : launch_gradient<64, EL_F16>(a, p, ranges, status, stream);
  return elem == EL_BF16 ? launch_gradient<128, EL_BF16>(a, p, ranges, status, stream) : launch_gradient<128, EL_F16>(a, p, ranges, status, stream);
}

}  // namespace b2x
