// Attention over tiles of 128 queries on the tensor cores: persistent, one CTA per SM, two independent workers per CTA.
//
// A worker owns a tile at a time (drawn from a device-wide counter), walks its blocks of 128 keys with the running maximum and
// sum of a softmax, normalises and writes its rows, and draws the next; while one worker starts or ends a tile the tensor and
// special-function pipes work for the other.  384 threads: warps 0, 1 draw tiles and load (TMA), warps 2, 3 issue the MMAs,
// warps 4-7 and 8-11 are the workers' softmax, one thread per query: its 128 scores are read from TMEM once and stay in registers
// through bias, mask, maximum and exponential; capped scores without a bias are read twice, 32 at a time.  Per worker Q, one K and
// one V stage, half a buffer of weights (the second half's first keys are exponentiated while the first half multiplies), 128 score
// columns and the accumulator in TMEM.
//
// Where there are fewer tiles than workers a tile's walk is cut into parts (tile_parts), which a second launch joins.
//
// What masks leave out is left out in three grades: blocks that no query of the tile sees are neither loaded nor multiplied (the
// keys' end follows from the last query; with documents the loading warp compares ranges of document numbers and publishes the
// tile's blocks as bits); blocks that every query sees run without a test; in the others a row's keys are 128 bits, from the
// row's last key and, by ballots over the warp's distinct documents, from the document numbers.
//
// What bounds it: the softmax warps, two for each of the SM's four schedulers, whose instructions wait for one another more than
// the tensor pipe (42 % busy) waits for operands.  2 x 16/8 heads, 4096 x 128, causal: 150 us, 915 TFLOP/s; with a bias by
// distance 216 us, with a cap 225, with both 276.
//
// Scores, maxima, sums and the accumulator are f32; the weights are rounded to the operands' 16 bits before they multiply V: o is off by
// 2.1e-3 of its norm against 64 bits (bf16; 1.6e-3 is the rounding of the result alone).
//
// Rows of V behind a sequence's length are set to zero in shared memory before they meet their zero weights: a product of 0 and
// what happens to lie there might be NaN.
#include <atomic>
#include <type_traits>

#include "head_attention_tc.cuh"

namespace b2x {
namespace {

struct TileParams {
  HeadAttn a;
  const int2* ranges;          // documents' ranges per block, [B][key blocks]
  int32_t q_tiles, group_heads, key_blocks, total, parts;   // total: tiles of all heads, times the parts of each (tile_parts)
  float* part_o;               // parts' accumulators: [part][tile][128][D]
  float2* part_ml;             // parts' maxima (log2 units) and sums: [part][tile][128]
  float mult;                  // scores in registers times this are log2 units: scale * log2(e), or 1 where cap or bias made them so
  uint64_t in2;                // scale * log2(e)
  HeadCap cap;
  int32_t scaled;              // scores are brought to log2 units before anything else (cap; bias; scale not positive)
  uint32_t idesc_qk, idesc_pv;
};

template <int D> struct TileSmem {
  static constexpr int Q_BYTES = HA_BLOCK * D * 2;
  static constexpr int KV_BYTES = HA_BLOCK * D * 2;
  static constexpr int P_BYTES = HA_BLOCK * 64 * 2;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + Q_BYTES;
  static constexpr int V_OFF = K_OFF + KV_BYTES;
  static constexpr int P_OFF = V_OFF + KV_BYTES;
  static constexpr int W_BYTES = P_OFF + P_BYTES;
  static constexpr int BAR_OFF = 2 * W_BYTES;              // 2 x 16 barriers, TMEM slot, abort flag
  static constexpr int SLOT_OFF = BAR_OFF + 288;
  static constexpr int TOTAL = SLOT_OFF + 4 * (int)sizeof(TileSlot) + 1024;
};

// What a kernel can do beside causal, prefix and length masks.  One kernel for everything left the warps of a plain problem waiting
// for instructions and its registers spilled (2 x 16 heads of 4096 x 128, causal: 199 us where the
// plain form took 157).  What is left of that: TILE_ANY spills 8 to 11 registers, TILE_DOCUMENTS two.
enum TileMode { TILE_PLAIN, TILE_CAP /* and documents */, TILE_DOCUMENTS, TILE_ANY /* a bias by distance, scales that are not positive */ };

template <int D, int EL, int MODE>
__global__ void __launch_bounds__(384, 1)
k_head_attention(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ TileParams p, int32_t* sched, int32_t* status) {
  using namespace sm100;
  using SM = TileSmem<D>;
  constexpr bool TWO_PASS = MODE == TILE_CAP;   // how the softmax warps go over a block
  constexpr bool CAP = MODE == TILE_CAP || MODE == TILE_ANY, SLOPES = MODE == TILE_ANY, DOCUMENTS = MODE != TILE_PLAIN;
  constexpr int DC = D / 64;
  constexpr uint32_t TMEM_COLS = 512;          // S0 [0,128), S1 [128,256), O0 [256, 256 + D), O1 [256 + D, 256 + 2 D)

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = (uint64_t*)(smem + SM::BAR_OFF);
  uint32_t* tmem_slot = (uint32_t*)(bars + 32);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = warp < 4 ? (warp & 1) : ((warp - 4) >> 2);   // worker
  volatile TileSlot* slots = (volatile TileSlot*)(smem + SM::SLOT_OFF) + 2 * w;   // the worker's current and next tile
  const uint32_t wb = smem_u32(bars) + (uint32_t)w * 128u;
  const uint32_t bar_qf = wb, bar_qe = wb + 8, bar_kf = wb + 16, bar_ke = wb + 24, bar_vf = wb + 32, bar_ve = wb + 40, bar_sf = wb + 48,
                 bar_se = wb + 56, bar_pf = wb + 64, bar_pv = wb + 72, bar_of = wb + 80, bar_tf = wb + 88 /* [2] */, bar_te = wb + 104 /* [2] */,
                 bar_drain = wb + 120;
  const uint32_t wbase = sbase + (uint32_t)w * SM::W_BYTES;
  const bool listed = DOCUMENTS && p.ranges != nullptr;

  if (threadIdx.x == 0) {
    for (int v = 0; v < 2; v++) {
      const uint32_t b = smem_u32(bars) + (uint32_t)v * 128u;
      mbar_init(b, 1); mbar_init(b + 8, 1); mbar_init(b + 16, 1); mbar_init(b + 24, 1); mbar_init(b + 32, 1); mbar_init(b + 40, 1);
      mbar_init(b + 48, 1); mbar_init(b + 56, 4); mbar_init(b + 64, 4); mbar_init(b + 72, 1); mbar_init(b + 80, 4);
      mbar_init(b + 88, 1); mbar_init(b + 96, 1); mbar_init(b + 104, 5); mbar_init(b + 112, 5); mbar_init(b + 120, 1);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmQ); tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
  }
  if (warp == 2) { tmem_alloc(smem_u32(tmem_slot), TMEM_COLS); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_trigger();
  pdl_wait();          // everything above touched this SM only

  if (warp < 2) {
    // ---------------------------------------------- tiles and loads ------------------------------------------------
    uint32_t kc = 0, vc = 0;       // K and V blocks loaded so far
    uint32_t nq = 0;               // tiles with work so far
    int fixed = (int)blockIdx.x + w * (int)gridDim.x;   // without a counter: every worker takes tiles in steps of all workers
    for (int n = 0;; n++) {
      // the slot's previous tile has been read by the issuer and the four softmax warps (all lanes wait: they leave together)
      if (n >= 2 && !ha_barrier_warp(bar_te + 8 * (n & 1), (uint32_t)(((n >> 1) - 1) & 1), abort_flag, status, 21)) break;
      int t = 0;
      if (w == 1 && p.total <= (int)gridDim.x) t = -1;     // one tile per SM: the first workers take them
      else if (sched) {
        if (lane == 0) t = atomicAdd(sched, 1);
        t = __shfl_sync(0xffffffffu, t, 0);
      } else { t = fixed; fixed += 2 * (int)gridDim.x; }
      if (t >= p.total) t = -1;
      volatile TileSlot* s = slots + (n & 1);
      int bh = 0, qt = 0, blocks = 0, begin = 0;
      HeadSequence seq{};
      if (t >= 0) {
        // groups of heads whose keys stay in L2 together; inside a group the tiles with the longest causal prefix first
        const int per_group = p.group_heads * p.q_tiles;
        const int tile = t / p.parts;
        const int g = tile / per_group, in = tile - g * per_group;
        const int heads = min(p.group_heads, p.a.B * p.a.Hq - g * p.group_heads);
        const int rank = in / heads;
        bh = g * p.group_heads + (in - rank * heads);
        qt = p.q_tiles - 1 - rank;
        const int b = bh / p.a.Hq, q0 = qt * HA_BLOCK, last = min(q0 + HA_BLOCK, p.a.Sq) - 1;
        seq = head_sequence(p.a, b);
        const int end = head_limit(p.a, seq, seq.first + last);
        blocks = (max(end, 0) + HA_BLOCK - 1) / HA_BLOCK;
        if (listed) {
          // documents of the tile's queries: the blocks that hold their positions
          const int lo = max(seq.first + q0, 0), hi = min(seq.first + last, p.a.Sk - 1);
          const int2* rs = p.ranges + (int64_t)b * p.key_blocks;
          int2 mine = make_int2(0x7fffffff, (int)0x80000000);
          if (lo <= hi) {
            const int2 r0 = ha_range(rs + lo / HA_BLOCK), r1 = ha_range(rs + hi / HA_BLOCK);
            mine = make_int2(min(r0.x, r1.x), max(r0.y, r1.y));
          }
          int count = 0;
          for (int i = 0; i < HA_MASK_WORDS; i++) {
            const int j = i * 32 + lane;
            bool visit = false, compare = false;
            if (j < blocks) {
              const int2 r = ha_range(rs + j);
              visit = !ha_apart(mine, r);
              compare = !ha_one_document(mine, r);
            }
            const uint32_t mv = __ballot_sync(0xffffffffu, visit), mc = __ballot_sync(0xffffffffu, compare);
            if (lane == 0) { s->visit[i] = mv; s->compare[i] = mc; }
            count += __popc(mv);
            if ((i + 1) * 32 >= blocks && lane == 0) { for (int k = i + 1; k < HA_MASK_WORDS; k++) s->visit[k] = 0; }
            if ((i + 1) * 32 >= blocks) break;
          }
          blocks = count;
        }
        if (p.parts > 1) {
          // this part's share of the blocks
          const int share = (blocks + p.parts - 1) / p.parts, skip = min((t - tile * p.parts) * share, blocks);
          blocks = min(share, blocks - skip);
          begin = skip;
          if (listed && lane == 0) {
            s->begin = 0;
            BlockWalk walk;
            walk.start(s, true);
            for (int i = 0; i < skip; i++) walk.next();
            begin = walk.j;
          }
        }
      }
      if (lane == 0) {
        s->tile = t; s->b = bh / max(p.a.Hq, 1); s->h = bh % max(p.a.Hq, 1); s->at = qt * HA_BLOCK; s->begin = begin; s->blocks = blocks;
        s->part = t >= 0 ? t % p.parts : 0;
        s->length = seq.length; s->first = seq.first; s->prefix = seq.prefix;
        mbar_arrive(bar_tf + 8 * (n & 1));
      }
      __syncwarp();
      if (t < 0) break;
      if (blocks == 0) continue;
      bool ok = true;
      if (elect_one()) {
        const int b = bh / p.a.Hq, h = bh - b * p.a.Hq, u = h / p.a.group;
        // Q is free once the previous tile's last Q K^T has retired
        if (nq > 0 && !ha_barrier(bar_qe, (nq - 1) & 1, abort_flag, status, 22)) ok = false;
        if (ok) {
          mbar_expect_tx(bar_qf, SM::Q_BYTES);
#pragma unroll
          for (int c = 0; c < DC; c++) tma_load_4d(wbase + SM::Q_OFF + c * HA_CHUNK, &tmQ, bar_qf, c * 64, qt * HA_BLOCK, h, b);
          BlockWalk wk, wv;
          wk.start(s, listed); wv.start(s, listed);
          uint32_t k_c = kc, v_c = vc;
          int jk = 0, jv = 0;
          uint32_t idle = 0;
          while (jk < blocks || jv < blocks) {
            bool progress = false;
            if (jk < blocks && (k_c == 0 || mbar_try_wait(bar_ke, (k_c - 1) & 1))) {
              mbar_expect_tx(bar_kf, SM::KV_BYTES);
#pragma unroll
              for (int c = 0; c < DC; c++) tma_load_4d(wbase + SM::K_OFF + c * HA_CHUNK, &tmK, bar_kf, c * 64, wk.j * HA_BLOCK, u, b);
              jk++; k_c++; progress = true;
              wk.next();
            }
            if (jv < blocks && (v_c == 0 || mbar_try_wait(bar_ve, (v_c - 1) & 1))) {
              mbar_expect_tx(bar_vf, SM::KV_BYTES);
#pragma unroll
              for (int c = 0; c < DC; c++) tma_load_4d(wbase + SM::V_OFF + c * HA_CHUNK, &tmV, bar_vf, c * 64, wv.j * HA_BLOCK, u, b);
              jv++; v_c++; progress = true;
              wv.next();
            }
            if (progress) { idle = 0; continue; }
            if (++idle > (1u << 22)) { *abort_flag = 1; if (status) atomicCAS(status, 0, 11); ok = false; break; }
            if (idle > 16) { if (*abort_flag) { ok = false; break; } __nanosleep(idle > 4096 ? 256 : 32); }
          }
        }
      }
      __syncwarp();
      kc += (uint32_t)blocks; vc += (uint32_t)blocks; nq++;
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
    }
  } else if (warp < 4) {
    // ---------------------------------------------- MMA issuer ------------------------------------------------------
    if (elect_one()) {
      uint32_t kc = 0, vc = 0, hc = 0, nq = 0;     // score blocks issued, V blocks consumed, P V half-steps issued, tiles with work
      const uint32_t s_tmem = tmem_base + (uint32_t)(w * 128), o_tmem = tmem_base + 256u + (uint32_t)(w * D);
      const uint32_t dq = ha_desc(wbase + SM::Q_OFF, 16), dk = ha_desc(wbase + SM::K_OFF, 16), dv = ha_desc(wbase + SM::V_OFF, HA_CHUNK), dp = ha_desc(wbase + SM::P_OFF, 16);
      bool ok = true;
      auto issue_qk = [&](bool last_of_tile) -> bool {
        if (!ha_barrier(bar_kf, kc & 1, abort_flag, status, 13)) return false;
        // the worker's softmax has copied the previous block's scores into registers
        if (kc > 0 && !ha_barrier(bar_se, (kc - 1) & 1, abort_flag, status, 14)) return false;
        tc_fence_after();
#pragma unroll
        for (int k = 0; k < D / 16; k++) ha_mma(s_tmem, dq + ((k >> 2) * HA_CHUNK + (k & 3) * 32) / 16, dk + ((k >> 2) * HA_CHUNK + (k & 3) * 32) / 16, p.idesc_qk, k > 0);
        tc_commit(bar_sf);
        tc_commit(bar_ke);
        if (last_of_tile) tc_commit(bar_qe);
        kc++;
        return true;
      };
      for (int n = 0; ok; n++) {
        if (!ha_barrier(bar_tf + 8 * (n & 1), (uint32_t)((n >> 1) & 1), abort_flag, status, 23)) { ok = false; break; }
        const int t = slots[n & 1].tile, blocks = slots[n & 1].blocks;
        mbar_arrive(bar_te + 8 * (n & 1));
        if (t < 0) break;
        if (blocks == 0) continue;
        if (!ha_barrier(bar_qf, nq & 1, abort_flag, status, 12)) { ok = false; break; }
        if (!issue_qk(blocks == 1)) { ok = false; break; }
        for (int it = 0; it < blocks && ok; it++) {
          // the block's scores are in the softmax warps' registers early: the next score block goes ahead of this
          // block's products.  In two passes they are read to the end only while the first half multiplies: it goes between.
          if (!TWO_PASS && it + 1 < blocks && !issue_qk(it + 2 == blocks)) { ok = false; break; }
          if (!ha_barrier(bar_vf, vc & 1, abort_flag, status, 15)) { ok = false; break; }
          // the previous tile's rows have been read out of the accumulator
          if (it == 0 && nq > 0 && !ha_barrier(bar_of, (nq - 1) & 1, abort_flag, status, 24)) { ok = false; break; }
#pragma unroll
          for (int h = 0; h < 2; h++) {
            if (!ha_barrier(bar_pf, hc & 1, abort_flag, status, 16)) { ok = false; break; }
            tc_fence_after();
            // A = P (K-major: 64 keys contiguous per row); B = V (MN-major: head-dim chunks of 64 are HA_CHUNK apart)
#pragma unroll
            for (int k = 0; k < 4; k++) ha_mma(o_tmem, dp + k * 2, dv + (4 * h + k) * 128, p.idesc_pv, it > 0 || h > 0 || k > 0);
            tc_commit(bar_pv);     // the half's weights have been read; the accumulator holds them
            hc++;
            if (h == 0 && TWO_PASS && it + 1 < blocks && !issue_qk(it + 2 == blocks)) { ok = false; break; }
          }
          if (!ok) break;
          tc_commit(bar_ve);
          vc++;
        }
        nq++;
      }
      // everything this thread issued must retire before TMEM is released
      tc_commit(bar_drain);
      ha_barrier(bar_drain, 0, abort_flag, nullptr, 0);
    }
  } else {
    // ---------------------------------------------- softmax ---------------------------------------------------------
    const int quad = warp & 3;                    // TMEM lanes [32 * quad, 32 * quad + 32): fixed by the warp's number
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_addr + (uint32_t)(w * 128);
    const uint32_t o_addr = tmem_base + lane_addr + 256u + (uint32_t)(w * D);
    const uint32_t prow_s = wbase + (uint32_t)(SM::P_OFF + row * 128);
    const uint32_t sw = (uint32_t)(row & 7);
    uint32_t sc = 0, hc = 0;                      // score blocks consumed, half-steps of weights published
    const uint64_t mult2 = splat2(p.mult);
    // 32 scores -> exp2, partial row sums, 16 words of 16-bit pairs
    auto exps = [&](const uint32_t (&r)[32], uint64_t mn2, uint64_t (&ps2)[2], uint32_t (&pw)[16]) {
#pragma unroll
      for (int h = 0; h < 16; h++) {
        const uint64_t x2 = fma2(pack2(r[2 * h], r[2 * h + 1]), mult2, mn2);
        uint32_t t0, t1;
        unpack2(x2, t0, t1);
        const float e0 = fast_exp2(__uint_as_float(t0)), e1 = fast_exp2(__uint_as_float(t1));
        ps2[h & 1] = add2(ps2[h & 1], pack2(__float_as_uint(e0), __float_as_uint(e1)));
        pw[h] = ha_pack<EL>(e0, e1);
      }
    };
    // chunk c (32 keys = four 16-byte pieces) of the 64-key half into the swizzled buffer of weights
    auto store = [&](int c, const uint32_t (&pw)[16]) {
#pragma unroll
      for (int q = 0; q < 4; q++)
        sts_v4(prow_s + ((((uint32_t)((c & 1) * 4 + q)) ^ sw) << 4), pw[4 * q], pw[4 * q + 1], pw[4 * q + 2], pw[4 * q + 3]);
    };
    auto publish = [&]() {
      tc_fence_before();
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_pf);
      hc++;
    };
    for (int n = 0;; n++) {
      if (!ha_barrier_warp(bar_tf + 8 * (n & 1), (uint32_t)((n >> 1) & 1), abort_flag, status, 25)) break;
      volatile TileSlot* s = slots + (n & 1);
      const int t = s->tile, blocks = s->blocks;
      if (t < 0) break;
      // what is needed again at the tile's end is read again there: the slot stays this tile's until then
      int pos = 0, end, doc = 0;
      float slope = 0.f;
      {
        const HeadSequence seq{s->length, s->first, s->prefix};
        pos = seq.first + s->at + row;
        end = head_limit(p.a, seq, pos);
        if constexpr (SLOPES) slope = p.a.slopes ? ld_global(p.a.slopes + s->h) * kLog2e : 0.f;
        if constexpr (DOCUMENTS) {
          if (p.a.documents) {
            if (pos >= 0 && pos < p.a.Sk) doc = (int)ld_global((const uint32_t*)p.a.documents + (int64_t)s->b * p.a.Sk + pos);
            else end = 0;
          }
        }
      }
      float m_used = -INFINITY, l = 0.f;
      bool poisoned = false;
      // A wait inside the tile that runs out lets its lane go on with what is there: the lanes of a warp have to stay together for
      // its votes and TMEM loads.  They leave as one at the tile's end, to which no wait is long any more, and its rows are not written.
      // (With a vote behind every wait a capped prompt took 1 % longer, with one every 64 blocks the gradient 1.5 %.)
      auto wait = [&](uint32_t bar, uint32_t parity, int code) { ha_barrier(bar, parity & 1, abort_flag, status, code); };
      auto given_up = [&]() -> bool { return __any_sync(0xffffffffu, *abort_flag != 0); };
      // the previous block's second half-product has retired: the buffer of weights is free and the accumulator at rest
      auto settle = [&](int it, bool rescale, float alpha) {
        if (it == 0) return;
        wait(bar_pv, hc - 1, 18);
        tc_fence_after();
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int c = 0; c < D / 16; c++) {
            uint32_t o[16];
            tmem_ld_32x16(o_addr + (uint32_t)(c * 16), o);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x16(o_addr + (uint32_t)(c * 16), o);
          }
          tc_wait_st();
        }
      };
      // values behind the sequence's end: zero before they meet their weights of zero
      uint32_t vc = sc;                           // the tile's first V block; its count goes with the score blocks
      auto clear_tail = [&](int j) {
        const uint32_t turn = vc++;
        if (!p.a.lengths || s->length >= p.a.Sk || s->length >= (j + 1) * HA_BLOCK) return;
        wait(bar_vf, turn, 26);
        if (j * HA_BLOCK + row >= s->length) {
#pragma unroll 1
          for (int c = 0; c < DC; c++)
#pragma unroll
            for (int q = 0; q < 8; q++) sts_v4(wbase + (uint32_t)(SM::V_OFF + c * HA_CHUNK + row * 128 + q * 16), 0, 0, 0, 0);
        }
      };
      BlockWalk walk;
      if (blocks > 0) walk.start(s, listed);
      for (int it = 0; it < blocks; it++) {
        const int j = walk.j;
        bool compare = false;
        if constexpr (DOCUMENTS) compare = listed ? (s->compare[j >> 5] >> (j & 31)) & 1 : p.a.documents != nullptr;
        if (it + 1 < blocks) walk.next();
        wait(bar_sf, sc, 17);
        tc_fence_after();
        // keys of this block that this row sees: [0, lim], and among them those of its document
        const int lim = end - 1 - j * HA_BLOCK;
        const bool need_mask = compare || __any_sync(0xffffffffu, lim < HA_BLOCK - 1);
        if constexpr (TWO_PASS) {
          // Capped scores: the cap is monotonic, so a first pass finds the row's maximum among the products, a second caps, weighs and
          // stores 32 columns at a time, a loop of a few registers and little code.  The score buffer is handed back late, which
          // this much arithmetic hides.  (With all 128 scores in registers, as below, 235 us
          // where this takes 220; with two warps for every 32 queries, a half of the keys each, 282.)
          uint32_t seen[4];
          float hi = -INFINITY, lo = INFINITY;
          if (need_mask) {
#pragma unroll
            for (int c = 0; c < 4; c++) {
              seen[c] = ha_bits(lim - c * 32);
              if (DOCUMENTS && compare) {
                const int key = j * HA_BLOCK + c * 32 + lane;
                const int theirs = key < p.a.Sk ? (int)ld_global((const uint32_t*)p.a.documents + (int64_t)s->b * p.a.Sk + key) : 0;
                seen[c] &= ha_same_document(doc, theirs, key < p.a.Sk);
              }
            }
          }
#pragma unroll 1
          for (int c = 0; c < 4; c++) {
            uint32_t r[32];
            tmem_ld_32x32(s_addr + (uint32_t)(c * 32), r);
            ha_wait(r);
            if (need_mask) {
              const uint32_t bits = c == 0 ? seen[0] : c == 1 ? seen[1] : c == 2 ? seen[2] : seen[3];
#pragma unroll
              for (int i = 0; i < 32; i++)
                if ((bits >> i) & 1u) { hi = max3(hi, __uint_as_float(r[i]), hi); lo = min3(lo, __uint_as_float(r[i]), lo); }
            } else {
              float h2[2] = {hi, hi}, l2[2] = {lo, lo};
#pragma unroll
              for (int i = 0; i < 16; i++) {
                h2[i & 1] = max3(h2[i & 1], __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                l2[i & 1] = min3(l2[i & 1], __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
              }
              hi = max3(h2[0], h2[1], h2[0]); lo = min3(l2[0], l2[1], l2[0]);
            }
          }
          const bool small = __all_sync(0xffffffffu, hi <= p.cap.small && lo >= -p.cap.small);
          float mx = -INFINITY;
          if (!need_mask || (seen[0] | seen[1] | seen[2] | seen[3]) != 0) {   // products of -inf are scores of -cap
            const uint64_t x = mul2(splat2(hi), p.cap.in2);
            uint32_t v0, v1;
            unpack2(small ? cap_small(p.cap, x) : cap_any(p.cap, x), v0, v1);
            mx = __uint_as_float(v0);
          }
          if (hi != hi || lo != lo) { poisoned = true; mx = 0.f; }
          float alpha = 1.f;
          bool rescale = false;
          if (it == 0) m_used = mx;
          else if (mx - m_used > 8.0f) { alpha = fast_exp2(m_used - mx); l *= alpha; m_used = mx; rescale = true; }
          settle(it, rescale, alpha);
          clear_tail(j);
          const uint64_t mn2 = splat2(m_used == -INFINITY ? 0.f : -m_used);
          uint64_t ps2[2] = {0ull, 0ull};
          auto chunks = [&](auto SMALL, auto MASK) {
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
              uint32_t r[32], pw[16];
              tmem_ld_32x32(s_addr + (uint32_t)(c * 32), r);
              ha_wait(r);
              if (c == 3) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_se);
              }
              const uint32_t bits = c == 0 ? seen[0] : c == 1 ? seen[1] : c == 2 ? seen[2] : seen[3];
#pragma unroll
              for (int h2 = 0; h2 < 16; h2++) {
                const uint64_t x = mul2(pack2(r[2 * h2], r[2 * h2 + 1]), p.cap.in2);
                uint64_t y;
                if constexpr (decltype(SMALL)::value) y = cap_small_plus(p.cap, x, mn2);
                else y = add2(cap_any(p.cap, x), mn2);
                uint32_t t0, t1;
                unpack2(y, t0, t1);
                if constexpr (decltype(MASK)::value) {
                  if (!((bits >> (2 * h2)) & 1u)) t0 = 0xff800000u;
                  if (!((bits >> (2 * h2 + 1)) & 1u)) t1 = 0xff800000u;
                }
                const float e0 = fast_exp2(__uint_as_float(t0)), e1 = fast_exp2(__uint_as_float(t1));
                ps2[h2 & 1] = add2(ps2[h2 & 1], pack2(__float_as_uint(e0), __float_as_uint(e1)));
                pw[h2] = ha_pack<EL>(e0, e1);
              }
              // the first half's product has retired: its buffer takes the second half
              if (c == 2) wait(bar_pv, hc - 1, 19);
              store(c & 1, pw);
              if (c & 1) publish();
            }
          };
          using std::bool_constant;
          if (small) { if (need_mask) chunks(bool_constant<true>{}, bool_constant<true>{}); else chunks(bool_constant<true>{}, bool_constant<false>{}); }
          else { if (need_mask) chunks(bool_constant<false>{}, bool_constant<true>{}); else chunks(bool_constant<false>{}, bool_constant<false>{}); }
          sc++;
          uint32_t a0, a1, b0, b1;
          unpack2(ps2[0], a0, a1); unpack2(ps2[1], b0, b1);
          l += (__uint_as_float(a0) + __uint_as_float(a1)) + (__uint_as_float(b0) + __uint_as_float(b1));
        } else {
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; c++) tmem_ld_32x32(s_addr + (uint32_t)(c * 32), r[c]);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_se);
        sc++;
        if (CAP && p.cap.cap > 0.f) {
          const float largest = max3(max3(ha_largest(r[0]), ha_largest(r[1]), 0.f), ha_largest(r[2]), ha_largest(r[3]));
          if (__all_sync(0xffffffffu, largest <= p.cap.small)) {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
              for (int i = 0; i < 16; i++) unpack2(cap_small(p.cap, mul2(pack2(r[c][2 * i], r[c][2 * i + 1]), p.cap.in2)), r[c][2 * i], r[c][2 * i + 1]);
          } else {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
              for (int i = 0; i < 16; i++) unpack2(cap_any(p.cap, mul2(pack2(r[c][2 * i], r[c][2 * i + 1]), p.cap.in2)), r[c][2 * i], r[c][2 * i + 1]);
          }
        } else if (MODE == TILE_ANY && !p.a.slopes) {
#pragma unroll
          for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) unpack2(mul2(pack2(r[c][2 * i], r[c][2 * i + 1]), p.in2), r[c][2 * i], r[c][2 * i + 1]);
        }
        float near = 0.f, grow = 0.f;              // SLOPES: what 32 keys' scores lack of their bias
        auto lacking = [&](int c) -> float { return fmaf((float)(32 * c), grow, near); };
        if (SLOPES && p.a.slopes) {
          const int far = pos - j * HA_BLOCK;
          const uint64_t m2 = p.cap.cap > 0.f ? splat2(1.f) : p.in2;
          const bool before = __all_sync(0xffffffffu, far >= HA_BLOCK - 1), behind = __all_sync(0xffffffffu, far <= 0);
          if (before || behind) {
            // All keys on one side of all the warp's queries: the bias grows by the slope from key to key.  Its growth within 32 keys is added
            // here, what is the same for all of them where a maximum is taken off anyway: added up along the keys, a bias far from its
            // query lost a rounding with every key.
            grow = before ? slope : -slope;
            near = -(float)far * grow;
            const uint64_t step2 = splat2(2.f * grow);
#pragma unroll
            for (int c = 0; c < 4; c++) {
              uint64_t on2 = pack2(0u, __float_as_uint(grow));
#pragma unroll
              for (int i = 0; i < 16; i++) {
                unpack2(fma2(pack2(r[c][2 * i], r[c][2 * i + 1]), m2, on2), r[c][2 * i], r[c][2 * i + 1]);
                on2 = add2(on2, step2);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
              for (int i = 0; i < 16; i++) {
                const float d0 = -slope * fabsf((float)(far - c * 32 - 2 * i)), d1 = -slope * fabsf((float)(far - c * 32 - 2 * i - 1));
                unpack2(fma2(pack2(r[c][2 * i], r[c][2 * i + 1]), m2, pack2(__float_as_uint(d0), __float_as_uint(d1))), r[c][2 * i], r[c][2 * i + 1]);
              }
          }
        }
        if (need_mask) {
#pragma unroll
          for (int c = 0; c < 4; c++) {
            uint32_t bits = ha_bits(lim - c * 32);
            if (DOCUMENTS && compare) {
              const int key = j * HA_BLOCK + c * 32 + lane;
              const int theirs = key < p.a.Sk ? (int)ld_global((const uint32_t*)p.a.documents + (int64_t)s->b * p.a.Sk + key) : 0;
              bits &= ha_same_document(doc, theirs, key < p.a.Sk);
            }
#pragma unroll
            for (int i = 0; i < 32; i++) if (!((bits >> i) & 1u)) r[c][i] = 0xff800000u;
          }
        }
        float mx;
        {
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx4[SLOPES ? c : i & 3] = max3(mx4[SLOPES ? c : i & 3], __uint_as_float(r[c][2 * i]), __uint_as_float(r[c][2 * i + 1]));
          if constexpr (SLOPES) {
#pragma unroll
            for (int c = 0; c < 4; c++) mx4[c] += lacking(c);
          }
          mx = max3(mx4[0], mx4[1], max3(mx4[2], mx4[3], -INFINITY));
        }
        // a NaN score makes the whole row NaN; keep the arithmetic finite and poison the row sum at the end
        if (mx != mx) { poisoned = true; mx = 0.f; }
        float alpha = 1.f;
        bool rescale = false;
        if (it == 0) m_used = mx;
        else if ((mx - m_used) * p.mult > 8.0f) { alpha = fast_exp2((m_used - mx) * p.mult); l *= alpha; m_used = mx; rescale = true; }
        settle(it, rescale, alpha);
        clear_tail(j);
        const float mneg = (m_used == -INFINITY) ? 0.f : -m_used * p.mult;
        const uint64_t same2 = splat2(mneg);
        auto less = [&](int c) -> uint64_t { return SLOPES ? splat2(mneg + lacking(c)) : same2; };
        uint64_t ps2[2] = {0ull, 0ull};
        {
          uint32_t pw[16];
          exps(r[0], less(0), ps2, pw); store(0, pw);
          exps(r[1], less(1), ps2, pw); store(1, pw);
        }
        publish();
        {
          // the second half: its first 32 keys are exponentiated while the first half multiplies
          uint32_t pw[16];
          exps(r[2], less(2), ps2, pw);
          wait(bar_pv, hc - 1, 19);
          store(0, pw);
          exps(r[3], less(3), ps2, pw); store(1, pw);
        }
        publish();
        {
          uint32_t a0, a1, b0, b1;
          unpack2(ps2[0], a0, a1); unpack2(ps2[1], b0, b1);
          l += (__uint_as_float(a0) + __uint_as_float(a1)) + (__uint_as_float(b0) + __uint_as_float(b1));
        }
        }
      }
      // ---- the tile's last product has retired: normalise and write the rows ----
      if (blocks > 0) {
        wait(bar_pv, hc - 1, 20);
        tc_fence_after();
      }
      if (given_up()) break;
      if (poisoned) l = __int_as_float(0x7fc00000);
      if (p.parts > 1) {
        const int64_t at = ((int64_t)s->part * (p.total / p.parts) + ((int64_t)s->b * p.a.Hq + s->h) * p.q_tiles + s->at / HA_BLOCK) * HA_BLOCK + row;
#pragma unroll 1
        for (int c = 0; c < D / 16; c++) {
          uint32_t x[16];
          if (blocks > 0) {
            tmem_ld_32x16(o_addr + (uint32_t)(c * 16), x);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = 0;
          }
#pragma unroll
          for (int i = 0; i < 16; i += 4) *(uint4*)(p.part_o + at * D + c * 16 + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        }
        p.part_ml[at] = make_float2(m_used * p.mult, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_te + 8 * (n & 1));
          if (blocks > 0) mbar_arrive(bar_of);
        }
        continue;
      }
      const float inv = !(l <= 0.f) ? 1.0f / l : 0.f;   // a NaN sum stays NaN
      const int b = s->b, h = s->h, qrow = s->at + row;
      char* orow = p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)h * p.a.os.head + (int64_t)qrow * p.a.os.token);
#pragma unroll 1
      for (int c = 0; c < D / 16; c++) {
        uint32_t x[16];
        if (blocks > 0) {
          tmem_ld_32x16(o_addr + (uint32_t)(c * 16), x);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) x[i] = 0;
        }
        if (qrow < p.a.Sq) {
          uint32_t wd[8];
          // a row that sees nothing is 0, whatever weights of zero were multiplied with
#pragma unroll
          for (int k = 0; k < 8; k++) wd[k] = inv == 0.f ? 0u : ha_pack<EL>(__uint_as_float(x[2 * k]) * inv, __uint_as_float(x[2 * k + 1]) * inv);
          ha_store_row(orow + 2 * (c * 16), p.a.D - c * 16, wd);
        }
      }
      if (p.a.lse && qrow < p.a.Sq)
        p.a.lse[((int64_t)b * p.a.Hq + h) * p.a.Sq + qrow] = l == 0.f ? -INFINITY : (m_used * p.mult + fast_log2(l)) * 0.6931471805599453f;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar_te + 8 * (n & 1));
        if (blocks > 0) mbar_arrive(bar_of);
      }
    }
  }

  ha_linger(abort_flag);
  tc_fence_before();
  __syncthreads();
  if (warp == 2) { tc_fence_after(); tmem_dealloc(tmem_base, TMEM_COLS); }
  // the last CTA to leave puts the tile counter back for the stream's next launch
  if (sched && threadIdx.x == 0 && atomicAdd(sched + 1, 1) == (int)gridDim.x - 1) { sched[0] = 0; sched[1] = 0; __threadfence(); }
}

// Parts that a tile's blocks are cut into.  Where there are fewer tiles than workers, the longest walk takes the whole time; parts of
// four blocks and more, as many as give every worker one (two under a causal mask, which leaves half of the blocks).  2 heads, 3766 x 80,
// cap and bias, causal: 162 -> 47 us; 2/1 heads, 2692 x 64, bias, 75 -> 31; 4 heads, 1024 x 128, 28 -> 20.  Where every SM has a tile as
// it is, writing and joining the parts has to be worth it: 256 causal tiles of up to 32 blocks 84 -> 66 us, of up to 16 blocks 47 -> 51.
template <typename Args> int tile_parts(const Args& a) {
  const int64_t tiles = (int64_t)a.B * a.Hq * ((a.Sq + HA_BLOCK - 1) / HA_BLOCK), blocks = (a.Sk + HA_BLOCK - 1) / HA_BLOCK;
  if (tiles <= 0) return 1;
  int64_t parts = (a.causal ? 4 : 2) * kNumSms / tiles;
  if (parts > blocks / 4) parts = blocks / 4;
  if (tiles > kNumSms && blocks < 24) parts = 1;
  return parts < 1 ? 1 : (int)(parts < 16 ? parts : 16);
}
// Parts are joined as the blocks of a walk are: by their maxima.  One warp per row.
template <int D, int EL>
__global__ void __launch_bounds__(256) k_attention_join(const __grid_constant__ TileParams p) {
  pdl_trigger();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (int64_t)(p.total / p.parts) * HA_BLOCK;
  const int lane = threadIdx.x & 31, col = lane * 4;
  const int tile = (int)(id / HA_BLOCK), bh = tile / p.q_tiles, i = (tile - bh * p.q_tiles) * HA_BLOCK + (int)(id % HA_BLOCK), b = bh / p.a.Hq, h = bh - b * p.a.Hq;
  if (id < rows && i < p.a.Sq) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < p.parts) { const uint2 v = ld_global((const uint2*)(p.part_ml + lane * rows + id)); ml = make_float2(__uint_as_float(v.x), __uint_as_float(v.y)); }
    // a part that saw nothing has a sum of 0 and is left out, whatever its accumulator holds
    float m = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    const float w = ml.y == 0.f ? 0.f : fast_exp2(ml.x - m);
    float l = ml.y == 0.f ? 0.f : ml.y * w;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.parts; k++) {
      const float wk = __shfl_sync(0xffffffffu, w, k);
      if (wk != 0.f && col < p.a.D) {
        const uint4 x = ld_global((const uint4*)(p.part_o + (k * rows + id) * D + col));
        o.x = fmaf(__uint_as_float(x.x), wk, o.x); o.y = fmaf(__uint_as_float(x.y), wk, o.y);
        o.z = fmaf(__uint_as_float(x.z), wk, o.z); o.w = fmaf(__uint_as_float(x.w), wk, o.w);
      }
    }
    const float inv = !(l <= 0.f) ? 1.0f / l : 0.f;   // a NaN sum stays NaN
    if (col < p.a.D)
      *(uint2*)(p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)h * p.a.os.head + (int64_t)i * p.a.os.token + col)) =
          inv == 0.f ? make_uint2(0, 0) : make_uint2(ha_pack<EL>(o.x * inv, o.y * inv), ha_pack<EL>(o.z * inv, o.w * inv));
    if (lane == 0 && p.a.lse) p.a.lse[(int64_t)bh * p.a.Sq + i] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * 0.6931471805599453f;
  }
}

// One warp per block of 128 tokens
__global__ void __launch_bounds__(256) k_document_ranges(const int32_t* documents, int2* ranges, int32_t B, int32_t Sk, int32_t blocks) {
  pdl_trigger();
  pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (id < (int64_t)B * blocks) {
    const int b = (int)(id / blocks), j = (int)(id - (int64_t)b * blocks);
    int lo = 0x7fffffff, hi = (int)0x80000000;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int t = j * HA_BLOCK + i * 32 + lane;
      if (t < Sk) { const int d = (int)ld_global((const uint32_t*)documents + (int64_t)b * Sk + t); lo = min(lo, d); hi = max(hi, d); }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) ranges[id] = make_int2(lo, hi);
  }
}

template <int D, int EL, int MODE>
int launch_tiles(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileParams& p, int32_t* sched, int32_t* status, cudaStream_t stream) {
  using SM = TileSmem<D>;
  auto kern = k_head_attention<D, EL, MODE>;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> configured[64];
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::TOTAL);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  const int ctas = p.total < kNumSms ? p.total : kNumSms;
  const cudaError_t e = launch_overlapped(kern, dim3((unsigned)ctas), dim3(384), SM::TOTAL, stream, q, k, v, p, sched, status);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  if (p.parts > 1) {
    const cudaError_t f = launch_overlapped(k_attention_join<D, EL>, dim3((unsigned)((int64_t)(p.total / p.parts) * HA_BLOCK / 8)), dim3(256), 0, stream, p);
    if (f != cudaSuccess) return (int)f;
    count_launch();
  }
  return (int)cudaGetLastError();
}

template <int D, int EL>
int launch_tiles(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TileParams& p, int32_t* sched, int32_t* status, cudaStream_t stream) {
  const bool cap = p.cap.cap > 0.f;
  if (p.a.slopes || !(p.a.scale > 0.f)) return launch_tiles<D, EL, TILE_ANY>(q, k, v, p, sched, status, stream);
  if (cap) return launch_tiles<D, EL, TILE_CAP>(q, k, v, p, sched, status, stream);
  if (p.a.documents) return launch_tiles<D, EL, TILE_DOCUMENTS>(q, k, v, p, sched, status, stream);
  return launch_tiles<D, EL, TILE_PLAIN>(q, k, v, p, sched, status, stream);
}

}  // namespace

int ha_launch_ranges(const HeadAttn& p, int2* ranges, cudaStream_t stream) {
  const int blocks = (p.Sk + HA_BLOCK - 1) / HA_BLOCK;
  const int64_t n = (int64_t)p.B * blocks;
  if (n == 0) return 0;
  const cudaError_t e = launch_overlapped(k_document_ranges, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, stream, p.documents, ranges, p.B, p.Sk, blocks);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  return (int)cudaGetLastError();
}

int64_t ha_forward_scratch(const HeadAttn& a, int64_t ranges) {
  const int parts = tile_parts(a);
  return parts == 1 ? ranges : (ranges + 15) / 16 * 16 + (int64_t)parts * a.B * a.Hq * ((a.Sq + HA_BLOCK - 1) / HA_BLOCK) * HA_BLOCK * ((a.D <= 64 ? 64 : 128) * 4 + 8);
}
int ha_forward_launches(const HeadAttn& a) { return 1 + (tile_parts(a) > 1); }

int ha_launch_forward(const HeadAttn& a, int elem, int2* ranges, int32_t* status, cudaStream_t stream) {
  TileParams p{};
  p.a = a;
  p.q_tiles = (a.Sq + HA_BLOCK - 1) / HA_BLOCK;
  p.key_blocks = (a.Sk + HA_BLOCK - 1) / HA_BLOCK;
  const int64_t total = (int64_t)a.B * a.Hq * p.q_tiles;
  if (total == 0) return 0;
  if (total > 0x7fffff00) return (int)cudaErrorInvalidValue;
  p.parts = tile_parts(a);
  p.total = (int)total * p.parts;
  if (a.documents) {
    const int rc = ha_launch_ranges(a, ranges, stream);
    if (rc) return rc;
  }
  // scratch: ranges, then from a multiple of 16 bytes on the parts
  const int D = a.D <= 64 ? 64 : 128;
  p.part_o = (float*)((char*)ranges + ((a.documents ? (int64_t)a.B * p.key_blocks * 8 : 0) + 15) / 16 * 16);
  p.part_ml = (float2*)(p.part_o + (int64_t)p.total * HA_BLOCK * D);
  // longer sequences than a skip list covers walk all their blocks, and compare in each
  p.ranges = a.documents && p.key_blocks <= HA_MASK_WORDS * 32 ? ranges : nullptr;
  const int64_t kv_heads = (32ll << 20) / ((int64_t)(a.Sk > 0 ? a.Sk : 1) * a.D * 4);
  const int64_t heads = kv_heads < 1 ? a.group : kv_heads * a.group;
  p.group_heads = (int)(heads > (int64_t)a.B * a.Hq ? (int64_t)a.B * a.Hq : heads);
  p.scaled = a.softcap > 0.f || a.slopes || !(a.scale > 0.f);
  p.mult = p.scaled ? 1.0f : a.scale * kLog2e;
  p.in2 = ha_pair(a.scale * kLog2e);
  p.cap = ha_cap(a.softcap, a.scale);
  const uint32_t format = elem == EL_BF16 ? 1u : 0u;
  p.idesc_qk = sm100::make_idesc(format, false, false, HA_BLOCK, HA_BLOCK);
  p.idesc_pv = sm100::make_idesc(format, false, true, HA_BLOCK, (uint32_t)D);
  CUtensorMap q, k, v;
  if (!ha_encode(&q, elem, a.q, a.qs, a.B, a.Hq, a.Sq, a.D)) return (int)cudaErrorInvalidValue;
  if (a.Sk == 0) k = v = q;      // nothing is loaded
  else if (!ha_encode(&k, elem, a.k, a.ks, a.B, a.Hk, a.Sk, a.D) || !ha_encode(&v, elem, a.v, a.vs, a.B, a.Hk, a.Sk, a.D)) return (int)cudaErrorInvalidValue;
  int32_t* sched = ha_sched(stream);
  if (D == 64) return elem == EL_BF16 ? launch_tiles<64, EL_BF16>(q, k, v, p, sched, status, stream) : launch_tiles<64, EL_F16>(q, k, v, p, sched, status, stream);
  return elem == EL_BF16 ? launch_tiles<128, EL_BF16>(q, k, v, p, sched, status, stream) : launch_tiles<128, EL_F16>(q, k, v, p, sched, status, stream);
}

}  // namespace b2x
