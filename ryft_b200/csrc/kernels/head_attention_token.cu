// Attention of a few queries per sequence (up to 16; one, where a model answers) against a long cache.
//
// Bound by HBM: keys and values are read once, 4 * rows flops for every 2 bytes of them.  The query heads that share a key head are
// the rows of one tile of 16, so that a cache line serves all of them.  The keys of a sequence are cut into chunks, a CTA of four
// warps each, whatever the batch: long sequences spread over the chip, chunks behind a short one's end leave at once.  A warp takes
// 16 keys at a time from memory straight into the fragments of m16n8k16 products, the next 16 in flight meanwhile; nothing passes
// through shared memory and no warp waits for another before the end.  (The 128-row tiles of tcgen05 would be empty but for a few
// rows; the products here are a fifth of the time that the loads take.)
//
// 16-byte loads without shuffles: a product over d does not depend on the order of d, so four neighbouring lanes take 8 adjacent
// elements each of a key's row (and of a query's) for two k-steps; and the columns of a result may come in any order, so eight
// lanes take 8 adjacent elements each of a value's row, element i of each belonging to product i.  A lane ends up with 16 adjacent
// elements of its two rows.
//
// Each warp keeps its own maximum (raised only when a score passes it by 2^8), sum and accumulator; the four meet in shared memory,
// chunks in a second launch that weighs them by their maxima.  Order of sums: fixed.
#include "head_attention_tc.cuh"

namespace b2x {
namespace {

constexpr int TOKEN_ROWS = 16, TOKEN_WARPS = 4;

struct TokenParams {
  HeadAttn a;
  int32_t rows, row_tiles;     // of a key head: Sq * group, and tiles of 16
  int32_t chunk, chunks;       // keys per CTA; CTAs per tile
  float mult;                  // scale * log2(e)
  float cap, cap_in;           // cap * log2(e) and the exponent 2 * scale / cap * log2(e); 0: none
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
__device__ __forceinline__ uint32_t token_low(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t token_high(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// row of a tile -> query head and query
struct TokenRow { int h, i; bool there; };
__device__ __forceinline__ TokenRow token_row(const TokenParams& p, int u, int row) {
  const bool there = row < p.rows;
  const int i = there ? row / p.a.group : 0;
  return {u * p.a.group + (there ? row - i * p.a.group : 0), i, there};
}

template <int D, int EL>
__global__ void __launch_bounds__(TOKEN_WARPS * 32, 2) k_attention_token(const __grid_constant__ TokenParams p) {
  constexpr int KJ = D / 32, VJ = D / 64;
  __shared__ float so[TOKEN_WARPS][TOKEN_ROWS][D + 4];
  __shared__ float2 sml[TOKEN_WARPS][TOKEN_ROWS];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const int tile = (int)(blockIdx.x / (unsigned)p.chunks), chunk = (int)(blockIdx.x - (unsigned)tile * (unsigned)p.chunks);
  const int rt = tile % p.row_tiles, bu = tile / p.row_tiles, b = bu / p.a.Hk, u = bu - b * p.a.Hk;
  const HeadSequence seq = head_sequence(p.a, b);
  const int r0 = rt * TOKEN_ROWS, r_last = min(r0 + TOKEN_ROWS, p.rows) - 1;
  const int end = max(head_limit(p.a, seq, seq.first + r_last / p.a.group), 0);
  const int k_begin = chunk * p.chunk, k_end = min(k_begin + p.chunk, end);
  const bool work = k_begin < k_end;
  if (work || p.chunks == 1) {
    // this lane's rows r and r + 8
    TokenRow row[2];
    int lim[2], doc[2];
    float slope[2], pos[2];
    uint32_t qf[2 * KJ][4];
#pragma unroll
    for (int x = 0; x < 2; x++) {
      row[x] = token_row(p, u, r0 + r + 8 * x);
      const int at = seq.first + row[x].i;
      lim[x] = row[x].there ? head_limit(p.a, seq, at) : 0;
      doc[x] = 0;
      if (p.a.documents) {
        if (at >= 0 && at < p.a.Sk) doc[x] = (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + at);
        else lim[x] = 0;
      }
      slope[x] = p.a.slopes ? ld_global(p.a.slopes + row[x].h) * kLog2e : 0.f;
      pos[x] = (float)at;
      const char* q = p.a.q + 2 * ((int64_t)b * p.a.qs.batch + (int64_t)row[x].h * p.a.qs.head + (int64_t)row[x].i * p.a.qs.token);
#pragma unroll
      for (int j = 0; j < KJ; j++) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (row[x].there && 32 * j + 8 * c < p.a.D) v = ld_global((const uint4*)(q + 2 * (32 * j + 8 * c)));
        qf[2 * j][x] = v.x; qf[2 * j][2 + x] = v.y; qf[2 * j + 1][x] = v.z; qf[2 * j + 1][2 + x] = v.w;
      }
    }
    const char* kp = p.a.k + 2 * ((int64_t)b * p.a.ks.batch + (int64_t)u * p.a.ks.head);
    const char* vp = p.a.v + 2 * ((int64_t)b * p.a.vs.batch + (int64_t)u * p.a.vs.head);
    uint4 kf[2][KJ], vf[4][VJ];
    auto load_k = [&](int k0) {
#pragma unroll
      for (int m = 0; m < 2; m++) {
        const int key = k0 + 8 * m + r;
#pragma unroll
        for (int j = 0; j < KJ; j++) {
          kf[m][j] = make_uint4(0, 0, 0, 0);
          if (key < k_end && 32 * j + 8 * c < p.a.D) kf[m][j] = ld_global((const uint4*)(kp + 2 * ((int64_t)key * p.a.ks.token + 32 * j + 8 * c)));
        }
      }
    };
    auto load_v = [&](int k0) {
#pragma unroll
      for (int m = 0; m < 4; m++) {
        const int key = k0 + 2 * c + (m & 1) + 8 * (m >> 1);
#pragma unroll
        for (int j = 0; j < VJ; j++) {
          vf[m][j] = make_uint4(0, 0, 0, 0);
          if (key < k_end && 64 * j + 8 * r < p.a.D) vf[m][j] = ld_global((const uint4*)(vp + 2 * ((int64_t)key * p.a.vs.token + 64 * j + 8 * r)));
        }
      }
    };
    float acc[8 * VJ][4], m_used[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool poisoned[2] = {false, false};
#pragma unroll
    for (int i = 0; i < 8 * VJ; i++)
#pragma unroll
      for (int x = 0; x < 4; x++) acc[i][x] = 0.f;
    int k0 = k_begin + warp * 16;
    if (k0 < k_end) { load_k(k0); load_v(k0); }
    for (; k0 < k_end; k0 += TOKEN_WARPS * 16) {
      const int next = k0 + TOKEN_WARPS * 16;
      float s[2][4];
#pragma unroll
      for (int m = 0; m < 2; m++) {
#pragma unroll
        for (int x = 0; x < 4; x++) s[m][x] = 0.f;
#pragma unroll
        for (int j = 0; j < KJ; j++) {
          token_mma<EL>(s[m], qf[2 * j], kf[m][j].x, kf[m][j].y);
          token_mma<EL>(s[m], qf[2 * j + 1], kf[m][j].z, kf[m][j].w);
        }
      }
      if (next < k_end) load_k(next);
      // element x of s[m]: row x >> 1, key k0 + 8 m + 2 c + (x & 1)
      float most[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const int key = k0 + 8 * m + 2 * c + (x & 1), w = x >> 1;
          float v = s[m][x];
          if (p.cap > 0.f) v = p.cap - 2.f * p.cap * fast_rcp(1.f + fast_exp2(v * p.cap_in));
          else v *= p.mult;
          if (p.a.slopes) v = fmaf(fabsf(pos[w] - (float)key), -slope[w], v);
          bool see = key < lim[w];
          if (p.a.documents) see = see && (int)ld_global((const uint32_t*)p.a.documents + (int64_t)b * p.a.Sk + min(key, p.a.Sk - 1)) == doc[w];
          s[m][x] = see ? v : -INFINITY;
          most[w] = max3(most[w], s[m][x], -INFINITY);
        }
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
        for (int i = 0; i < 8 * VJ; i++) { acc[i][0] *= f[0]; acc[i][1] *= f[0]; acc[i][2] *= f[1]; acc[i][3] *= f[1]; }
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
      for (int j = 0; j < VJ; j++) {
        const uint32_t v0[4] = {vf[0][j].x, vf[0][j].y, vf[0][j].z, vf[0][j].w}, v1[4] = {vf[1][j].x, vf[1][j].y, vf[1][j].z, vf[1][j].w};
        const uint32_t v2[4] = {vf[2][j].x, vf[2][j].y, vf[2][j].z, vf[2][j].w}, v3[4] = {vf[3][j].x, vf[3][j].y, vf[3][j].z, vf[3][j].w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
          token_mma<EL>(acc[8 * j + 2 * i], pf, token_low(v0[i], v1[i]), token_low(v2[i], v3[i]));
          token_mma<EL>(acc[8 * j + 2 * i + 1], pf, token_high(v0[i], v1[i]), token_high(v2[i], v3[i]));
        }
      }
      if (next < k_end) load_v(next);
    }
    // ---- the four warps meet ----
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
    for (int j = 0; j < VJ; j++)
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int x = 0; x < 4; x++) so[warp][r + 8 * (x >> 1)][64 * j + 16 * c + 8 * (x & 1) + i] = acc[8 * j + i][x] * f[x >> 1];
    __syncthreads();
    // thread: row, and every eighth element of it
    const int orow = threadIdx.x >> 3;
    const TokenRow o = token_row(p, u, r0 + orow);
    if (o.there) {
      float rm = -INFINITY, rl = 0.f;
#pragma unroll
      for (int k = 0; k < TOKEN_WARPS; k++) rm = fmaxf(rm, sml[k][orow].x);
#pragma unroll
      for (int k = 0; k < TOKEN_WARPS; k++) { const float2 v = sml[k][orow]; rl += v.x == -INFINITY ? v.y : v.y * fast_exp2(v.x - rm); }
      const float inv = p.chunks > 1 ? 1.f : rl == 0.f ? 0.f : 1.0f / rl;
      float* part = p.part_o + (((int64_t)tile * p.chunks + chunk) * TOKEN_ROWS + orow) * D;
      char* out = p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)o.h * p.a.os.head + (int64_t)o.i * p.a.os.token);
      for (int d = (threadIdx.x & 7) * 2; d < p.a.D; d += 16) {
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int k = 0; k < TOKEN_WARPS; k++) { v0 += so[k][orow][d]; v1 += so[k][orow][d + 1]; }
        if (p.chunks > 1) *(float2*)(part + d) = make_float2(v0, v1);
        else *(uint32_t*)(out + 2 * d) = ha_pack<EL>(rl != rl ? rl : v0 * inv, rl != rl ? rl : v1 * inv);
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
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const float f = l != l ? l : ((v[0] + v[1]) + (v[2] + v[3])) * inv;
    *(uint16_t*)(p.a.o + 2 * ((int64_t)b * p.a.os.batch + (int64_t)o.h * p.a.os.head + (int64_t)o.i * p.a.os.token + tid)) = (uint16_t)(ha_pack<EL>(f, 0.f) & 0xffffu);
  }
  if (tid == 0 && p.a.lse) p.a.lse[((int64_t)b * p.a.Hq + o.h) * p.a.Sq + o.i] = l == 0.f ? -INFINITY : (m + fast_log2(l)) * 0.6931471805599453f;
}

void token_shape(const HeadAttn& a, TokenParams* p) {
  p->rows = a.Sq * a.group;
  p->row_tiles = (p->rows + TOKEN_ROWS - 1) / TOKEN_ROWS;
  const int64_t tiles = (int64_t)a.B * a.Hk * p->row_tiles;
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
  cudaError_t e = launch_overlapped(k_attention_token<D, EL>, dim3((unsigned)ctas), dim3(TOKEN_WARPS * 32), 0, stream, p);
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
  p.cap = a.softcap > 0.f ? a.softcap * kLog2e : 0.f;
  p.cap_in = a.softcap > 0.f ? 2.0f * a.scale / a.softcap * kLog2e : 0.f;
  if (D == 64) return elem == EL_BF16 ? launch_token<64, EL_BF16>(p, stream) : launch_token<64, EL_F16>(p, stream);
  return elem == EL_BF16 ? launch_token<128, EL_BF16>(p, stream) : launch_token<128, EL_F16>(p, stream);
}

}  // namespace b2x
