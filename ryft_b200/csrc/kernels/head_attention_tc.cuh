// What the tensor-core kernels of head_attention share: tensor maps over tensors of heads, the ranges of document numbers that
// let whole blocks be skipped, and masks as bits.
#pragma once
#include <cstring>

#include "attention_math.cuh"
#include "head_attention.cuh"
#include "sm100.cuh"

namespace b2x {

constexpr int HA_BLOCK = 128;                 // queries of a tile, keys of a block
constexpr int HA_MASK_WORDS = 32;             // blocks that a tile's skip list covers: 1024, 131072 tokens
constexpr uint32_t HA_CHUNK = 128 * 128;      // one [128 rows x 128 bytes] swizzled sub-tile

// Two f32 as one word of 16-bit values, `lo` in the lower half.
template <int EL> __device__ __forceinline__ uint32_t ha_pack(float lo, float hi) {
  if constexpr (EL == EL_BF16) { __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&t); }
  else { __half2 t = __floats2half2_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&t); }
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Keys 0..31 of a chunk that lie at or below `lim` (relative to the chunk's first key).
__device__ __forceinline__ uint32_t ha_bits(int lim) { return lim >= 31 ? 0xffffffffu : lim < 0 ? 0u : (2u << lim) - 1u; }

// Which of 32 keys lie in the lane's document: lane l holds key l's (`key`; `there` says whether there is such a key).  The lanes
// of a warp are neighbouring queries (or keys), so the loop over their distinct documents is short.
__device__ __forceinline__ uint32_t ha_same_document(int mine, int key, bool there) {
  uint32_t todo = 0xffffffffu, bits = 0;
  const uint32_t valid = __ballot_sync(0xffffffffu, there);
  while (todo) {
    const int d = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
    const uint32_t b = __ballot_sync(0xffffffffu, key == d) & valid;
    const bool hit = mine == d;
    if (hit) bits = b;
    todo &= ~__ballot_sync(0xffffffffu, hit);
  }
  return bits;
}

// Smallest and largest document of every block of 128 tokens: one warp per block.  [B][blocks]
__device__ __forceinline__ bool ha_apart(int2 a, int2 b) { return a.y < b.x || b.y < a.x; }
__device__ __forceinline__ bool ha_one_document(int2 a, int2 b) { return a.x == a.y && b.x == b.y && a.x == b.x; }
__device__ __forceinline__ int2 ha_range(const int2* r) {
  const uint2 v = ld_global((const uint2*)r);
  return make_int2((int)v.x, (int)v.y);
}

// 4-D tensor map (width, tokens, heads, sequences) with a box of 64 elements x `rows` tokens; elements behind the width read as 0.
inline bool ha_encode(CUtensorMap* m, int elem, const void* base, const B2xHeadStrides& s, int64_t B, int64_t H, int64_t S, int64_t D, uint32_t rows = HA_BLOCK) {
  PFN_encodeTiled fn = get_encode_tiled();
  if (!fn || ((uintptr_t)base & 15) != 0) return false;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  // the stride of a dimension of one is never used, but has to be a legal one
  int64_t st = S > 1 ? s.token : D, sh = H > 1 ? s.head : D, sb = B > 1 ? s.batch : D;
  if (st % 8 != 0 || sh % 8 != 0 || sb % 8 != 0 || st <= 0 || sh <= 0 || sb <= 0) return false;
  cuuint64_t strides[3] = {(cuuint64_t)st * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {64, rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  return fn(m, elem == EL_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr float kLog2e = 1.4426950408889634f;

// softcap * tanh(x) in log2 units, x = scale / softcap times the product.  Two ways:
//   |x| <= 0.75 (scores up to 0.75 caps, the usual case): an odd polynomial of degree 9, the minimax fit of tanh(x) / x in x^2
//     (exchange algorithm of Remez, relative error 6e-7), seven packed instructions for two scores on the FMA pipe;
//   beyond: cap - 2 cap q with q = 1 / (1 + e^2x), two special-function instructions per score, right for infinities, too.  Its error
//     goes with the cap, not with the score (2e-7 caps), so that it is for scores of the cap's size only.
// Where all scores of a warp's block are small only the polynomial is worked out; else both, and each score takes its own.
// The special-function pipe does 16 a clock and SM and has the softmax's exponential to do for every score as it is: with the
// second way alone a block of 128 x 128 keeps it busy three times as long as the tensor pipe (1024 cycles).
//
// Constants are held as pairs, so that packed instructions take them as they are: splitting one value in front of every use cost
// two moves each.
struct HeadCap {
  float cap;                   // cap * log2(e); 0: none
  float small;                 // products up to this magnitude take the polynomial: 0.75 caps
  uint64_t in2;                // scale / softcap
  uint64_t c0, c1, c2, c3, c4; // the polynomial's coefficients times `cap`
  uint64_t back2;              // -1 / cap^2: 1 - tanh^2 = 1 + back * (cap tanh)^2
  uint64_t out2, twice2;       // cap, -2 cap
};
inline uint64_t ha_pair(float v) {
  uint32_t u;
  memcpy(&u, &v, 4);
  return ((uint64_t)u << 32) | u;
}
inline HeadCap ha_cap(float softcap, float scale) {
  HeadCap h{};
  if (!(softcap > 0.f)) return h;
  h.cap = softcap * kLog2e;
  h.in2 = ha_pair(scale / softcap);
  h.small = scale != 0.f ? fminf(0.75f * softcap / fabsf(scale), 3e38f) : 0.f;   // infinite products are beyond it
  h.c0 = ha_pair(0.99999946f * h.cap); h.c1 = ha_pair(-0.3332825f * h.cap); h.c2 = ha_pair(0.13258983f * h.cap);
  h.c3 = ha_pair(-0.0500563f * h.cap); h.c4 = ha_pair(0.012929632f * h.cap);
  h.back2 = ha_pair(-1.0f / (h.cap * h.cap));
  h.out2 = ha_pair(h.cap); h.twice2 = ha_pair(-2.0f * h.cap);
  return h;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// cap * tanh(x) of a pair, and the same plus something
__device__ __forceinline__ uint64_t cap_share(const HeadCap& h, uint64_t x) {
  const uint64_t y = mul2(x, x);
  uint64_t c = fma2(y, h.c4, h.c3);
  c = fma2(y, c, h.c2);
  c = fma2(y, c, h.c1);
  return fma2(y, c, h.c0);
}
__device__ __forceinline__ uint64_t cap_small(const HeadCap& h, uint64_t x) { return mul2(x, cap_share(h, x)); }
__device__ __forceinline__ uint64_t cap_small_plus(const HeadCap& h, uint64_t x, uint64_t plus) { return fma2(x, cap_share(h, x), plus); }
// e^2x and q = 1 / (1 + e^2x); with BOUNDED e^2x stays finite (2^126 at most), as products with q need it
template <bool BOUNDED> __device__ __forceinline__ uint64_t cap_rest(uint64_t x, uint64_t& e2) {
  uint32_t a0, a1;
  unpack2(mul2(x, splat2(2.f * kLog2e)), a0, a1);
  float x0 = __uint_as_float(a0), x1 = __uint_as_float(a1);
  if constexpr (BOUNDED) { x0 = min3(x0, 126.f, 126.f); x1 = min3(x1, 126.f, 126.f); }
  e2 = pack2(__float_as_uint(fast_exp2(x0)), __float_as_uint(fast_exp2(x1)));
  unpack2(add2(e2, splat2(1.f)), a0, a1);
  return pack2(__float_as_uint(fast_rcp(__uint_as_float(a0))), __float_as_uint(fast_rcp(__uint_as_float(a1))));
}
// cap * tanh(x) of a pair of any size: of the polynomial's and the other, each x takes its own
__device__ __forceinline__ uint64_t cap_choose(const HeadCap& h, uint64_t x, uint64_t q) {
  uint32_t x0, x1, s0, s1, l0, l1;
  unpack2(x, x0, x1);
  unpack2(cap_small(h, x), s0, s1);
  unpack2(fma2(q, h.twice2, h.out2), l0, l1);
  return pack2(fabsf(__uint_as_float(x0)) <= 0.75f ? s0 : l0, fabsf(__uint_as_float(x1)) <= 0.75f ? s1 : l1);
}
__device__ __forceinline__ uint64_t cap_any(const HeadCap& h, uint64_t x) {
  uint64_t e2;
  const uint64_t q = cap_rest<false>(x, e2);
  return cap_choose(h, x, q);
}
// Waits for a TMEM load; naming its registers keeps their uses behind the wait.
__device__ __forceinline__ void ha_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
  asm volatile("" : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                    "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
// Largest magnitude of 32 products, NaN if one is
__device__ __forceinline__ float ha_largest(const uint32_t (&r)[32]) {
  float m[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 16; i++) m[i & 1] = max3(m[i & 1], fabsf(__uint_as_float(r[2 * i])), fabsf(__uint_as_float(r[2 * i + 1])));
  return max3(m[0], m[1], 0.f);
}

// Matrix products with descriptors as their lower words (address and leading offset; make_smem_desc): the upper word is the same for
// all tiles here (128-byte swizzle, groups of eight rows 1024 bytes apart), and a step on is one addition.  Against 64-bit
// descriptors built for every product: a capped causal step and its gradient of 2 x 16/4 heads, 4096 x 128, 870 -> 858 us.
__device__ __forceinline__ uint32_t ha_desc(uint32_t addr, uint32_t lbo_bytes) { return ((addr >> 4) & 0x3fffu) | (((lbo_bytes >> 4) & 0x3fffu) << 16); }
constexpr uint32_t HA_DESC_UPPER = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void ha_mma(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n"
      ::"r"(d_tmem), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(HA_DESC_UPPER)
      : "memory");
}
__device__ __forceinline__ void ha_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 y;\n mov.b64 y, {%2, %5};\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "n"(HA_DESC_UPPER)
      : "memory");
}

// Sixteen 16-bit values of a row, `width` of which exist: 32 bytes at once where the row lies on that boundary (a sector in one
// access, half as many of them), else 16 bytes at a time.
__device__ __forceinline__ void ha_store_row(char* row, int width, const uint32_t (&w)[8]) {
  if (width >= 16 && ((uintptr_t)row & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(__cvta_generic_to_global(row)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
    return;
  }
  if (width > 0) *reinterpret_cast<uint4*>(row) = make_uint4(w[0], w[1], w[2], w[3]);
  if (width > 8) *reinterpret_cast<uint4*>(row + 16) = make_uint4(w[4], w[5], w[6], w[7]);
}

// sm100::mbar_wait with the thread asleep in between: most of a CTA's warps wait most of the time here, and what they poll with
// is taken from the warps that compute.
__device__ __forceinline__ bool ha_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(2000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool ha_barrier(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int code) {
  for (uint32_t i = 0; i < (1u << 21); i++) {
    if (ha_try_wait(bar, parity)) return true;
    if (i > 4 && *abort_flag) return false;
  }
  *abort_flag = 1;
  if (status) atomicCAS(status, 0, code);
  return false;
}

// The same for all lanes of a warp, with one answer: lanes that gave up by themselves would miss from the votes of the others.
__device__ __forceinline__ bool ha_barrier_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status, int code) {
  return __all_sync(0xffffffffu, ha_barrier(bar, parity, abort_flag, status, code));
}
// Before a CTA that has given up leaves: what it has in flight (copies, products) ends while shared memory and TMEM are still its own.
__device__ __forceinline__ void ha_linger(const volatile int* abort_flag) {
  if (*abort_flag) for (uint32_t i = 0; i < 4096; i++) __nanosleep(256);
}

// A tile as its loading warp publishes it.
struct TileSlot {
  int tile;                    // -1: no more
  int b, h, at;                // sequence, head, first query (or key) of the tile
  int begin, blocks;           // first block to walk, and how many
  int part, skip, count;       // number of this part of the tile; gradient: of the units of all heads that pass by, those before and of this part
  int length, first, prefix;   // HeadSequence
  uint32_t visit[HA_MASK_WORDS], compare[HA_MASK_WORDS];   // with documents: blocks to walk, and those whose documents have to be compared
};

// A tile's blocks in their order: all from `begin`, or those whose bits are set
struct BlockWalk {
  const volatile TileSlot* s;
  int j;
  bool listed;
  __device__ __forceinline__ void start(const volatile TileSlot* slot, bool list) { s = slot; listed = list; j = slot->begin - 1; next(); }
  __device__ __forceinline__ void next() {
    j++;
    if (!listed) return;
    int w = j >> 5;
    uint32_t m = w < HA_MASK_WORDS ? s->visit[w] & (0xffffffffu << (j & 31)) : 0u;
    while (m == 0 && ++w < HA_MASK_WORDS) m = s->visit[w];
    j = m ? w * 32 + __ffs(m) - 1 : HA_MASK_WORDS * 32;
  }
};


int32_t* sched_slot(cudaStream_t stream);   // gemm_tc.cu: a (tile counter, finished CTAs) pair per stream
// The same, or nullptr (tiles dealt out in a fixed order) where launches that share a handle may run side by side and would share the
// counter: while the stream is captured (graphs of one stream may later run at once), and on the per-thread default stream, one
// handle for every thread's own stream.
inline int32_t* ha_sched(cudaStream_t stream) {
  if (stream == cudaStreamPerThread) return nullptr;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(stream, &status) != cudaSuccess || status != cudaStreamCaptureStatusNone) return nullptr;
  return sched_slot(stream);
}

// Blocks of 128 tokens and the launches of the entry points.
int ha_launch_ranges(const HeadAttn& p, int2* ranges, cudaStream_t stream);
bool ha_token_takes(const HeadAttn& p);
int64_t ha_token_scratch(const HeadAttn& p);
int ha_token_launches(const HeadAttn& p);
int ha_launch_token(const HeadAttn& p, int elem, void* scratch, cudaStream_t stream);
int64_t ha_gradient_scratch(const B2xHeadAttentionArgs* a, int64_t ranges);
int ha_gradient_launches(const B2xHeadAttentionArgs* a);
int64_t ha_forward_scratch(const HeadAttn& p, int64_t ranges);
int ha_forward_launches(const HeadAttn& p);
int ha_launch_gradient(const HeadAttn& p, int elem, void* scratch, int32_t* status, cudaStream_t stream);
int ha_launch_forward(const HeadAttn& p, int elem, int2* ranges, int32_t* status, cudaStream_t stream);

}  // namespace b2x
