// Attention of a few queries per sequence (up to 16; one, where a model answers) against a long cache.
//
// Bound by HBM: keys and values are read once for every 16 rows, 4 * rows flops for every 2 bytes of them.  The queries of all heads that
// share a key head are the rows of tiles of 16, so that a cache line serves 16 of them; 16 queries of 8 heads are 8 tiles, each of
// which reads the cache for itself.  The keys of a sequence are cut into chunks, a CTA of four
// warps each, whatever the batch: long sequences spread over the chip, chunks behind a short one's end leave at once.  A warp walks
// steps of 16 keys through a ring of its own in shared memory, filled two steps ahead by asynchronous copies of 16 bytes (keys
// behind the sequence's end are filled with zeros, so that nothing that lies there meets a product), and multiplies with m16n8k16
// from there; no warp waits for another before the end.  (The 128-row tiles of tcgen05 would be empty but for a few rows; the
// products here are a fifth of the time that the loads take.)  Straight into registers, with one step in flight, the loads
// reached 3.2 TB/s: their latency showed, and 520 instructions per step went into placing them.  32 sequences with caches of
// various lengths up to 8192, 32/8 heads of 128, capped: 93 us, 5.9 TB/s (6.5 where all lengths are 8192).
//
// Each warp keeps its own maximum (raised only when a score passes it by 2^8), sum and accumulator; the four meet in shared memory,
// chunks in a second launch that weighs them by their maxima.  Order of sums: fixed.
#include <atomic>

#include "head_attention_tc.cuh"

namespace b2x {
namespace {

constexpr int TOKEN_ROWS = 16, TOKEN_WARPS = 4, TOKEN_STAGES = 3;

struct TokenParams {
  HeadAttn a;
  int32_t rows, row_tiles;     // of a key head: Sq * group, and tiles of 16
  int32_t tiles;               // of all key heads and sequences
  int32_t chunk, chunks;       // keys per CTA; CTAs per tile
  float mult;                  // scale * log2(e)
  HeadCap cap;
  float* part_o;               // [tile][chunk][16][D]
  float2* part_ml;             // [tile][chunk][16]: maximum (log2 units) and sum
};

template <int EL> __device__ __forceinline__ void token_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (EL == EL_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void token_ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void token_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes to shared memory, or zeros
__device__ __forceinline__ void token_copy(uint32_t dst, const char* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(on ? 16 : 0) : "memory");
}
template <int N> __device__ __forceinline__ void token_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// row of a tile -> query head and query
struct TokenRow { int h, i; bool there; };
__device__ __forceinline__ TokenRow token_row(const TokenParams& p, int u, int row) {
  const bool there = row < p.rows;
  const int i = there ? row / p.a.group : 0;
  return {u * p.a.group + (there ? row - i * p.a.group : 0), i, there};
}

template <int D> struct TokenSmem {
  static constexpr int STEP_BYTES = 2 * 16 * D * 2;            // 16 keys and their values
  static constexpr int RING_BYTES = TOKEN_STAGES * STEP_BYTES; // of a warp
  static constexpr int ROW = D + 4;                            // floats per row where the warps meet (in the rings' place)
  static constexpr int MEET_BYTES = TOKEN_WARPS * TOKEN_ROWS * ROW * 4 + TOKEN_WARPS * TOKEN_ROWS * 8;
  static constexpr int TOTAL = TOKEN_WARPS * RING_BYTES > MEET_BYTES ? TOKEN_WARPS * RING_BYTES : MEET_BYTES;
};

template <int D, int EL>
__global__ void __launch_bounds__(TOKEN_WARPS * 32, 2) k_attention_token(const __grid_constant__ TokenParams p) {
  using SM = TokenSmem<D>;
  constexpr int PIECES = D / 8;                // 16-byte pieces of a row
  constexpr int LOADS = 16 * PIECES / 32;      // copies of a lane for 16 rows
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  // chunks of all heads and sequences in turn: heads that lie side by side in memory are read at the same time
  const int tile = (int)(blockIdx.x % (unsigned)p.tiles), chunk = (int)(blockIdx.x / (unsigned)p.tiles);
  const int rt = tile % p.row_tiles, bu = tile / p.row_tiles, b = bu / p.a.Hk, u = bu - b * p.a.Hk;
  const HeadSequence seq = head_sequence(p.a, b);
  const int r0 = rt * TOKEN_ROWS, r_last = min(r0 + TOKEN_ROWS, p.rows) - 1;
  const int end = max(head_limit(p.a, seq, seq.first + r_last / p.a.group), 0);
  const int k_begin = chunk * p.chunk, k_end = min(k_begin + p.chunk, end);
  const bool work = k_begin < k_end;
  if (work || p.chunks == 1) {
    const uint32_t ring = sm100::smem_u32(smem) + (uint32_t)warp * SM::RING_BYTES;
    // copies: this lane's pieces are rows (lane / PIECES) + i * (32 / PIECES), swizzled within groups of eight pieces
    const int piece = lane % PIECES, row_in = lane / PIECES;
    const bool wide = piece * 8 < p.a.D;
    const char* kp = p.a.k + 2 * ((int64_t)b * p.a.ks.batch + (int64_t)u * p.a.ks.head + piece * 8);
    const char* vp = p.a.v + 2 * ((int64_t)b * p.a.vs.batch + (int64_t)u * p.a.vs.head + piece * 8);
    auto fill = [&](int stage, int k0) {       // the 16 keys from k0 on; always one group, of nothing behind the chunk
      if (k0 < k_end) {
        const uint32_t at = ring + (uint32_t)stage * SM::STEP_BYTES;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
          const int row = row_in + i * (32 / PIECES), key = k0 + row;
          const uint32_t dst = at + (uint32_t)(row * D * 2 + (piece & ~7) * 16 + (((piece ^ row) & 7) << 4));
          const bool on = wide && key < k_end;
          const int64_t from = on ? key : k_begin;
          token_copy(dst, kp + (wide ? 2 * from * p.a.ks.token : 0), on);
          token_copy(dst + 16 * D * 2, vp + (wide ? 2 * from * p.a.vs.token : 0), on);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int k0 = k_begin + warp * 16;
#pragma unroll
    for (int st = 0; st < TOKEN_STAGES - 1; st++) fill(st, k0 + st * TOKEN_WARPS * 16);

    // this lane's rows r and r + 8
    TokenRow row[2];
    int lim[2], doc[2], pos[2];
    float slope[2];
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      row[x] = token_row(p, u, r0 + r + 8 * x);
      const int at = seq.first + row[x].i;
      lim[x] = row[x].there ? head_limit(p.a, seq, at) : 0x7fffffff;    // a row that is not there may see what it likes
      doc[x] = 0;
      if (p.a.documents) {
        if (at >= 0 && at < p.a.Sk) doc[x] = (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + at);
        else if (row[x].there) lim[x] = 0;
      }
      slope[x] = p.a.slopes ? ld_global(p.a.slopes + row[x].h) * kLog2e : 0.f;
      pos[x] = at;
      const char* q = p.a.q + 2 * ((int64_t)b * p.a.qs.batch + (int64_t)row[x].h * p.a.qs.head + (int64_t)row[x].i * p.a.qs.token);
#pragma unroll
      for (int k = 0; k < D / 16; k++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const int d = 16 * k + 8 * y + 2 * c;
          qf[k][x + 2 * y] = row[x].there && d < p.a.D ? ld_global((const uint32_t*)(q + 2 * d)) : 0u;
        }
    }
    // keys below `open` are seen by every row
    const int open = !p.a.slopes && !p.a.documents ? __reduce_min_sync(0xffffffffu, min(lim[0], lim[1])) : 0;
    float acc[PIECES][4], m_used[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool poisoned[2] = {false, false};
#pragma unroll
    for (int i = 0; i < PIECES; i++)
#pragma unroll
      for (int x = 0; x < 4; x++) acc[i][x] = 0.f;
    // fragments: keys as they lie (matrix lane / 8 of a load: pieces 4 q + lane / 8 of eight keys), values turned (keys 8 * (bit 3 of the
    // lane), piece 2 q + (bit 4))
    const uint32_t k_row = (uint32_t)(lane & 7), v_row = (uint32_t)((lane & 7) + (lane & 8));
    int stage = 0;
    for (; k0 < k_end; k0 += TOKEN_WARPS * 16) {
      token_arrived<TOKEN_STAGES - 2>();
      __syncwarp();
      // the stage that the previous step read
      fill(stage == 0 ? TOKEN_STAGES - 1 : stage - 1, k0 + (TOKEN_STAGES - 1) * TOKEN_WARPS * 16);
      const uint32_t at = ring + (uint32_t)stage * SM::STEP_BYTES, vat = at + 16 * D * 2;
      stage = stage == TOKEN_STAGES - 1 ? 0 : stage + 1;
      float s[2][4];
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int x = 0; x < 4; x++) s[m][x] = 0.f;
#pragma unroll
      for (int q = 0; q < D / 32; q++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
          uint32_t f[4];
          const uint32_t pc = (uint32_t)(4 * q) + (uint32_t)(lane >> 3);
          token_ldsm(at + (k_row + 8 * m) * (D * 2) + (pc & ~7u) * 16 + (((pc ^ k_row) & 7) << 4), f);
          token_mma<EL>(s[m], qf[2 * q], f[0], f[1]);
          token_mma<EL>(s[m], qf[2 * q + 1], f[2], f[3]);
        }
      // element x of s[m]: row x >> 1, key k0 + 8 m + 2 c + (x & 1)
      if (p.cap.cap > 0.f) {
        float largest = 0.f;
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int x = 0; x < 4; x += 2) largest = max3(largest, fabsf(s[m][x]), fabsf(s[m][x + 1]));
        const bool small = __all_sync(0xffffffffu, largest <= p.cap.small);
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int x = 0; x < 4; x += 2) {
            const uint64_t v = mul2(pack2(__float_as_uint(s[m][x]), __float_as_uint(s[m][x + 1])), p.cap.in2);
            uint32_t a, b;
            unpack2(small ? cap_small(p.cap, v) : cap_any(p.cap, v), a, b);
            s[m][x] = __uint_as_float(a); s[m][x + 1] = __uint_as_float(b);
          }
      } else {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int x = 0; x < 4; x++) s[m][x] *= p.mult;
      }
      if (k0 + 16 > open) {
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            const int key = k0 + 8 * m + 2 * c + (x & 1), w = x >> 1;
            float v = s[m][x];
            if (p.a.slopes) v = fmaf(fabsf((float)(pos[w] - key)), -slope[w], v);
            bool see = key < lim[w] && key < k_end;
            if (p.a.documents) see = see && (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + min(key, p.a.Sk - 1)) == doc[w];
            s[m][x] = see ? v : -INFINITY;
          }
      }
      float most[2];
#pragma unroll
      for (int w = 0; w < 2; w++) most[w] = max3(max3(s[0][2 * w], s[0][2 * w + 1], s[1][2 * w]), s[1][2 * w + 1], -INFINITY);
      // a NaN score makes its row NaN: noted here, kept out of the arithmetic
#pragma unroll
      for (int w = 0; w < 2; w++) if (most[w] != most[w]) { poisoned[w] = true; most[w] = 0.f; }
      if (__any_sync(0xffffffffu, most[0] > m_used[0] + 8.f || most[1] > m_used[1] + 8.f)) {
        float f[2];
#pragma unroll
        for (int w = 0; w < 2; w++) {
          float m = fmaxf(most[w], m_used[w]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
          f[w] = m_used[w] == -INFINITY ? 0.f : fast_exp2(m_used[w] - m);
          l[w] *= f[w];
          m_used[w] = m;
        }
#pragma unroll
        for (int i = 0; i < PIECES; i++) { acc[i][0] *= f[0]; acc[i][1] *= f[0]; acc[i][2] *= f[1]; acc[i][3] *= f[1]; }
      }
      uint32_t pf[4];
      {
        const float base[2] = {m_used[0] == -INFINITY ? 0.f : m_used[0], m_used[1] == -INFINITY ? 0.f : m_used[1]};
        float e[2][4];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
          for (int x = 0; x < 4; x++) { e[m][x] = fast_exp2(s[m][x] - base[x >> 1]); l[x >> 1] += e[m][x]; }
        pf[0] = ha_pack<EL>(e[0][0], e[0][1]); pf[1] = ha_pack<EL>(e[0][2], e[0][3]);
        pf[2] = ha_pack<EL>(e[1][0], e[1][1]); pf[3] = ha_pack<EL>(e[1][2], e[1][3]);
      }
#pragma unroll
      for (int q = 0; q < PIECES / 2; q++) {
        uint32_t f[4];
        const uint32_t pc = (uint32_t)(2 * q) + (uint32_t)(lane >> 4);
        token_ldsm_t(vat + v_row * (D * 2) + (pc & ~7u) * 16 + (((pc ^ v_row) & 7) << 4), f);
        token_mma<EL>(acc[2 * q], pf, f[0], f[1]);
        token_mma<EL>(acc[2 * q + 1], pf, f[2], f[3]);
      }
    }
    // ---- the four warps meet, in the rings' place ----
    token_arrived<0>();
    __syncthreads();
    float (*so)[TOKEN_ROWS][SM::ROW] = (float (*)[TOKEN_ROWS][SM::ROW])smem;
    float2 (*sml)[TOKEN_ROWS] = (float2 (*)[TOKEN_ROWS])(smem + TOKEN_WARPS * TOKEN_ROWS * SM::ROW * 4);
#pragma unroll
    for (int w = 0; w < 2; w++) {
      if (poisoned[w]) l[w] = __int_as_float(0x7fc00000);
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 1);
      l[w] += __shfl_xor_sync(0xffffffffu, l[w], 2);
      if (c == 0) sml[warp][r + 8 * w] = make_float2(m_used[w], l[w]);
    }
    __syncthreads();
    float f[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      float most = -INFINITY;
#pragma unroll
      for (int k = 0; k < TOKEN_WARPS; k++) most = fmaxf(most, sml[k][r + 8 * w].x);
      f[w] = m_used[w] == -INFINITY ? 0.f : fast_exp2(m_used[w] - most);
    }
#pragma unroll
    for (int i = 0; i < PIECES; i++)
#pragma unroll
      for (int w = 0; w < 2; w++) *(float2*)&so[warp][r + 8 * w][8 * i + 2 * c] = make_float2(acc[i][2 * w] * f[w], acc[i][2 * w + 1] * f[w]);
    __syncthreads();
    // eight threads per row, two adjacent elements of every sixteen each
    const int orow = threadIdx.x >> 3;
    const TokenRow o = token_row(p, u, r0 + orow);
    if (o.there) {
      float rm = -INFINITY, rl = 0.f;
#pragma unroll
      for (int k = 0; k < TOKEN_WARPS; k++) rm = fmaxf(rm, sml[k][orow].x);
#pragma unroll
      for (int k = 0; k < TOKEN_WARPS; k++) { const float2 v = sml[k][orow]; rl += v.x == -INFINITY ? v.y : v.y * fast_exp2(v.x - rm); }
      const float inv = 1.0f / rl;
      float* part = p.part_o + (((int64_t)tile * p.chunks + chunk) * TOKEN_ROWS + orow) * D;
      char* out = p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)o.h * p.a.os.head + (int64_t)o.i * p.a.os.token);
      for (int d = (threadIdx.x & 7) * 2; d < p.a.D; d += 16) {
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int k = 0; k < TOKEN_WARPS; k++) { const float2 v = *(const float2*)&so[k][orow][d]; v0 += v.x; v1 += v.y; }
        if (p.chunks > 1) *(float2*)(part + d) = make_float2(v0, v1);
        else *(uint32_t*)(out + 2 * d) = rl == 0.f ? 0u : ha_pack<EL>(rl != rl ? rl : v0 * inv, rl != rl ? rl : v1 * inv);   // sees nothing: 0, whatever was multiplied
      }
      if ((threadIdx.x & 7) == 0) {
        if (p.chunks > 1) p.part_ml[((int64_t)tile * p.chunks + chunk) * TOKEN_ROWS + orow] = make_float2(rm, rl);
        else if (p.a.lse) p.a.lse[((int64_t)b * p.a.Hq + o.h) * p.a.Sq + o.i] = rl == 0.f ? -INFINITY : (rm + fast_log2(rl)) * 0.6931471805599453f;
      }
    }
  }
}

// One CTA per row: the chunks' maxima and sums, then their accumulators by weight
template <int D, int EL>
__global__ void __launch_bounds__(128) k_attention_token_join(const __grid_constant__ TokenParams p) {
  __shared__ float weight[128];
  __shared__ float red[8];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile_rows = min(p.rows, TOKEN_ROWS * p.row_tiles);
  const int bu = (int)(blockIdx.x / (unsigned)tile_rows), row = (int)(blockIdx.x - (unsigned)bu * (unsigned)tile_rows);
  const int b = bu / p.a.Hk, u = bu - b * p.a.Hk, rt = row / TOKEN_ROWS, tile = bu * p.row_tiles + rt;
  const HeadSequence seq = head_sequence(p.a, b);
  const int r_last = min((rt + 1) * TOKEN_ROWS, p.rows) - 1;
  const int end = max(head_limit(p.a, seq, seq.first + r_last / p.a.group), 0);
  const int n = (end + p.chunk - 1) / p.chunk;         // chunks that were worked on; at most 128
  const int64_t base = (int64_t)tile * p.chunks * TOKEN_ROWS + row % TOKEN_ROWS;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (tid < n) { const uint2 v = ld_global((const uint2*)(p.part_ml + base + (int64_t)tid * TOKEN_ROWS)); ml = make_float2(__uint_as_float(v.x), __uint_as_float(v.y)); }
  float m = ml.x;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m);
  float l = ml.x == -INFINITY ? ml.y : ml.y * w;
  weight[tid] = w;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (lane == 0) red[4 + warp] = l;
  __syncthreads();
  l = (red[4] + red[5]) + (red[6] + red[7]);
  const TokenRow o = token_row(p, u, row);
  if (tid < p.a.D) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    const float* src = p.part_o + base * D + tid;
    int k = 0;
    for (; k + 4 <= n; k += 4)
#pragma unroll
      for (int x = 0; x < 4; x++) v[x] = fmaf(ld_global(src + (int64_t)(k + x) * TOKEN_ROWS * D), weight[k + x], v[x]);
    for (; k < n; k++) v[0] = fmaf(ld_global(src + (int64_t)k * TOKEN_ROWS * D), weight[k], v[0]);
    const float f = l == 0.f ? 0.f : l != l ? l : ((v[0] + v[1]) + (v[2] + v[3])) * (1.0f / l);
    *(uint16_t*)(p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)o.h * p.a.os.head + (int64_t)o.i * p.a.os.token + tid)) = (uint16_t)(ha_pack<EL>(f, 0.f) & 0xffffu);
  }
  if (tid == 0 && p.a.lse) p.a.lse[((int64_t)b * p.a.Hq + o.h) * p.a.Sq + o.i] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * 0.6931471805599453f;
}

void token_shape(const HeadAttn& a, TokenParams* p) {
  p->rows = a.Sq * a.group;
  p->row_tiles = (p->rows + TOKEN_ROWS - 1) / TOKEN_ROWS;
  const int64_t tiles = (int64_t)a.B * a.Hk * p->row_tiles;
  p->tiles = (int)tiles;
  // about eight CTAs per SM where the keys allow (two run at a time: sequences of different lengths even out), one step of the four
  // warps at least, and at most the 128 chunks that are joined
  int64_t chunk = tiles * a.Sk / (kNumSms * 8);
  const int64_t least = (a.Sk + 127) / 128;
  if (chunk < least) chunk = least;
  chunk = (chunk + 63) / 64 * 64;
  if (chunk < 64) chunk = 64;
  p->chunk = (int)(chunk < (1 << 30) ? chunk : 1 << 30);
  p->chunks = a.Sk > 0 ? (int)((a.Sk + p->chunk - 1) / p->chunk) : 1;
}

template <int D, int EL>
int launch_token(const TokenParams& p, cudaStream_t stream) {
  const int64_t tiles = (int64_t)p.a.B * p.a.Hk * p.row_tiles, ctas = tiles * p.chunks, rows = (int64_t)p.a.B * p.a.Hk * p.rows;
  if (ctas > 0x7fffffff || rows > 0x7fffffff) return (int)cudaErrorInvalidValue;
  auto kern = k_attention_token<D, EL>;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<bool> configured[64];
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TokenSmem<D>::TOTAL);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  cudaError_t e = launch_overlapped(kern, dim3((unsigned)ctas), dim3(TOKEN_WARPS * 32), TokenSmem<D>::TOTAL, stream, p);
  if (e != cudaSuccess) return (int)e;
  count_launch();
  if (p.chunks > 1) {
    e = launch_overlapped(k_attention_token_join<D, EL>, dim3((unsigned)rows), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return (int)e;
    count_launch();
  }
  return (int)cudaGetLastError();
}

}  // namespace

// Few queries: tiles of 128 would be nearly empty, and there is one per head for a whole sequence of keys.
bool ha_token_takes(const HeadAttn& a) { return a.Sq <= 16; }

int64_t ha_token_scratch(const HeadAttn& a) {
  TokenParams p{};
  token_shape(a, &p);
  const int64_t parts = (int64_t)a.B * a.Hk * p.row_tiles * p.chunks * TOKEN_ROWS;
  return p.chunks > 1 ? parts * ((a.D <= 64 ? 64 : 128) * 4 + 8) : 0;
}
int ha_token_launches(const HeadAttn& a) {
  TokenParams p{};
  token_shape(a, &p);
  return p.chunks > 1 ? 2 : 1;
}

int ha_launch_token(const HeadAttn& a, int elem, void* scratch, cudaStream_t stream) {
  if (a.B == 0 || a.Hq == 0 || a.Sq == 0) return 0;
  TokenParams p{};
  p.a = a;
  token_shape(a, &p);
  const int D = a.D <= 64 ? 64 : 128;
  p.part_o = (float*)scratch;
  p.part_ml = (float2*)(p.part_o + (int64_t)a.B * a.Hk * p.row_tiles * p.chunks * TOKEN_ROWS * D);
  p.mult = a.scale * kLog2e;
  p.cap = ha_cap(a.softcap, a.scale);
  if (D == 64) return elem == EL_BF16 ? launch_token<64, EL_BF16>(p, stream) : launch_token<64, EL_F16>(p, stream);
  return elem == EL_BF16 ? launch_token<128, EL_BF16>(p, stream) : launch_token<128, EL_F16>(p, stream);
}

}  // namespace b2x
