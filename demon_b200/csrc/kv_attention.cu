// kv_attention.cu -- attention of new queries over a paged E4M3 K/V cache:
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]   over the keys j that query i sees
// (j < length, causal and band limits; a query that sees no key gives zeros).
//
// Small kernel (few query rows per kv head: single tokens, short chunks).  Bound by reading the
// codes, 256 bytes per key and kv head.  All G = Hq / Hk query heads of a kv head share one pass
// over its keys: a row is (token, query head), r = i * G + g.  A CTA takes 8 NR * RT rows and a
// range of keys in tiles of 64; one warp copies the tiles of K and V codes, as they lie in the
// pages, into a ring in shared memory (bulk copies of a page's 2 to 8 KB, mbarriers); four warps
// per row group each take 32 keys of every second tile.  The keys of a row tile are split over a
// thread-block cluster, which joins its partial results through distributed shared memory (one
// launch, no workspace), or, for long tables, over as many CTAs as fill the SMs, joined by a second
// kernel through a workspace.
//
// Measured, 8 kv heads: one token (16 query heads) over 750 keys 7.5 us, the launch and a few rounds of
// latency; one token of 48 sequences of up to 8,192 keys (32 query heads), 452 MB of codes, 81 us
// (5.6 TB/s); one token of 16 sequences of 16,384 keys 93 us (5.8 TB/s); five tokens of two sequences
// of up to 100,001 keys, 379 MB, 83.5 us (4.5 TB/s: 10 rows take twice the matrix instructions for the
// same bytes; six key warps a CTA were slower, 155 against 140 us at 16 CTAs a unit).
//
// A warp's step on 32 keys, all in registers (mma.sync m16n8k16, fp32 accumulators), with the keys
// and V's channels on the 16-wide side of the MMAs and the query rows on the 8-wide one, so that a
// few rows waste little:
//   S^T = K Q^T: E4M3 codes become f16 exactly; Q is f16 too, each row times a power of two that
//     brings its largest value to [2^13, 2^14) (exact down to 2^-28 of that value).  The page's
//     K scale, the row's power and the softmax scale are one fp32 factor of the score.
//   softmax: running maximum m and sum l per row; p = 2^(t - m + 14), so that f16 keeps p's full
//     precision down to 2^-28 of the row's largest; l sums the unrounded p.  P^T's 8 x 8 blocks
//     are transposed across the warp (movmatrix) from accumulator to operand layout.
//   O^T += V^T P^T: the codes of V go in unscaled; O is held in units of 2^e_ref, the largest V
//     scale met so far.  Keys of a page with a smaller scale 2^e have P multiplied by
//     2^(e - e_ref), exactly; if that is below 2^-8, their product goes through accumulators of
//     its own, so that P's precision never depends on the scales.  (V scales more than 2^64 apart:
//     row_of_wide_scales.)
// The f16 conversions take one instruction per two codes (and one more for the upper half of a
// word), and only a byte permute stands between V's rows and the operand layout: the keys and
// channels of a step may be taken in any order as long as both operands agree.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "demon_host.h"
#include "kv_common.cuh"
#include "kv_host.h"

namespace demon {
namespace kv {

namespace small {

constexpr int kTile = 64;                  // keys per stage
constexpr int kWarpKeys = 32;              // keys per warp and step
constexpr int kHalf = kTile * kHeadDim;    // one stage's K (or V) codes, 8 KB
constexpr int kKeyWarps = 4;               // per row group: two per tile, on alternating tiles
constexpr float kPBias = 14.0f;            // p is scaled by 2^14 (see above)
constexpr int kFoldMin = -8;               // smallest V scale, relative to e_ref, folded into P
constexpr float kMaxFactor = 1.3e36f;      // of a score: a zero score stays zero (its page's scale may be a hidden key's)
constexpr int kSpread = 64;                // V exponents of a CTA's keys up to which its rows share e_ref

// NR: 8-row MMA tiles per warp; RT: row groups (of four warps) per CTA.
template <int NR, int RT>
struct Cfg {
  static constexpr int kRows = 8 * NR;                    // rows of a group
  static constexpr int kThreads = (kKeyWarps * RT + 1) * 32;
  // ring: what keeps the memory busy with the CTAs that registers allow on an SM
  static constexpr int kStages = RT == 1 ? 4 : 6;
  // The two warps of a tile see every second one: with an even number of stages they meet every
  // phase of the stages they use.  (With three, a warp one phase ahead took the phase before as its own.)
  static_assert(kStages % 2 == 0, "a stage must always belong to the same warps");
  static constexpr int kMinCtas = NR == 1 ? 3 : RT == 1 ? 2 : 1;
  // Registers: a scheduler's quarter of the file holds whole warps, so 128 let three CTAs of five
  // warps in, 168 two (200 would leave one), 168 one of nine.  16 rows with 128 spill 460 bytes: 92
  // against 82 us for five tokens over 100,000 keys.
  static constexpr int kRegs = NR == 1 ? 128 : 168;
  static constexpr bool kQShared = NR > 1;                // Q operands in shared memory, for those registers
  static constexpr int offScale = kStages * 2 * kHalf;    // [stage][piece][K, V] fp32
  static constexpr int offBar = offScale + kStages * 4 * 2 * 4;  // full[stage], empty[stage]
  static constexpr int offMisc = offBar + kStages * 2 * 8;       // abort flag, wide flag
  static constexpr int offQ = offMisc + 16;               // [row group][k-step][lane] Q operands
  static constexpr int kSmem = offQ + (kQShared ? RT * 8 * 32 * 16 : 0);
  // After the key loop the ring holds the partial results: per warp O [rows][128] fp32, then the
  // CTA's sum, and the rows' statistics.
  static constexpr int kWarpO = kRows * kHeadDim * 4;
  static constexpr int offSum = kKeyWarps * RT * kWarpO;
  static constexpr int offStat = offSum + RT * kWarpO;                  // per warp and row: m, l, e
  static constexpr int offRow = offStat + kKeyWarps * RT * kRows * 12;  // CTA, per row: M, L, E
  static_assert(offRow + RT * kRows * 12 <= offScale && offQ % 16 == 0, "partial results must fit into the ring");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// over the eight lanes that share lane % 4
__device__ __forceinline__ float oct_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
}
__device__ __forceinline__ float oct_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 4);
  x += __shfl_xor_sync(0xffffffffu, x, 8);
  return x + __shfl_xor_sync(0xffffffffu, x, 16);
}
__device__ __forceinline__ uint32_t map_rank(uint32_t a, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t a) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void bulk_load_s(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// Cluster barrier in the form that counts threads (the .aligned one needs every warp whole at it).
__device__ __forceinline__ void cluster_join() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// Factor that brings a partial result with maximum m (and V unit 2^e) to maximum M (unit 2^E).
__device__ __forceinline__ float join_factor(float m, float M) {
  return m == -INFINITY ? 0.0f : ex2(m - M);
}
__device__ __forceinline__ float unit_factor(int e, int E) { return e - E < -126 ? 0.0f : exp2i(imin(e - E, 0)); }

// Four channels of row `grow` of the kv head's rows from its joined sums.
__device__ __forceinline__ void store_row(const AttnParams& p, int b, int hk, int grow, int nq, int lane, float4 acc, float L,
                                          int E) {
  const int i = grow / p.G, gq = grow - i * p.G;
  // L == 0: the row sees no key (a NaN score makes L NaN, and stays)
  const float inv = (i < nq && L != 0.0f) ? 1.0f / L : 0.0f;
  const float un = exp2i(E);
  uint2 out = make_uint2(0u, 0u);
  if (inv != 0.0f)
    out = make_uint2(pack_bf16x2(acc.x * inv * un, acc.y * inv * un), pack_bf16x2(acc.z * inv * un, acc.w * inv * un));
  *reinterpret_cast<uint2*>(p.o + b * p.o_seq + (int64_t)i * p.o_row + (int64_t)(hk * p.G + gq) * p.o_head + 4 * lane) = out;
}

// One row over keys [from, to) by one warp, four channels a lane, on the codes where they lie: what a CTA
// falls back on when V's exponents lie more than kSpread apart among its keys.  The key loop holds O of all
// its rows in units of the largest exponent met; a row that does not see that one, and whose own lie far
// below, would leave fp32's range.  Here the unit is that of the keys that the row sees.  Statistics and
// biases as there.  (Units for each row in the key loop cost every call 2 to 5 %.)
__device__ __forceinline__ void row_of_wide_scales(const AttnParams& p, int b, int hk, int grow, int len, int nq, int from,
                                                   int to, int lane, float& m, float& l, int& unit, float4& acc) {
  const int i = grow / p.G, gq = grow - i * p.G;
  m = -INFINITY;
  l = 0.0f;
  unit = kMinExp;
  acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (i < nq) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p.q + b * p.q_seq + (int64_t)i * p.q_row +
                                                         (int64_t)(hk * p.G + gq) * p.q_head + 4 * lane));
    const float2 q0 = bf2_f2(w.x), q1 = bf2_f2(w.y);
    const uint32_t x = w.x & 0x7FFF7FFFu, y = w.y & 0x7FFF7FFFu;  // the largest finite magnitude, as in the key loop
    uint32_t mx = __vmaxu2(x & __vcmpltu2(x, 0x7F807F80u), y & __vcmpltu2(y, 0x7F807F80u));
    mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
    const int k = imax((int)(mx >> 7) - 127 - 13, -126);
    const float by = exp2i(-k), fac = exp2i(k) * p.scale_log2;
    const Keys see = visible(i, i, len, nq, p.causal != 0, p.window);
    const int lo = imax(see.lo, from), hi = imin(see.hi, to);
#pragma unroll 1
    for (int j0 = lo & ~15; j0 < hi; j0 += 16) {
      const int pid = page_id(p.table + b * p.ld_table, p.W, j0 / p.c.P, p.c.pages);
      if (pid < 0) continue;  // (reported by the copying warp)
      const int64_t ph = (int64_t)pid * p.c.heads + hk, at = (ph * p.c.P + j0 % p.c.P) * kHeadDim + 4 * lane;
      const float f = fminf(fac * fabsf(__ldg(p.c.scale[0] + ph)), kMaxFactor);
      const int ev = scale_exp(__ldg(p.c.scale[1] + ph));
      const int is = imax(unit, ev);
      const float vf = unit_factor(ev, is);
      float back = unit_factor(unit, is);
      unit = is;
#pragma unroll 1
      for (int j = imax(j0, lo); j < imin(j0 + 16, hi); ++j) {
        uint32_t a[2], c[2];
        e4m3x4_f16(__ldg(reinterpret_cast<const uint32_t*>(p.c.codes[0] + at + (j - j0) * kHeadDim)), a[0], a[1]);
        e4m3x4_f16(__ldg(reinterpret_cast<const uint32_t*>(p.c.codes[1] + at + (j - j0) * kHeadDim)), c[0], c[1]);
        const float2 k0 = f16x2_f32(a[0]), k1 = f16x2_f32(a[1]), v0 = f16x2_f32(c[0]), v1 = f16x2_f32(c[1]);
        float t = fmaf(q0.x * by, k0.x, fmaf(q0.y * by, k0.y, fmaf(q1.x * by, k1.x, q1.y * by * k1.y)));
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) t += __shfl_xor_sync(0xffffffffu, t, d);
        t *= f;
        const float n = fmaxf(m, t), s = n == -INFINITY ? 1.0f : ex2(m - n);
        const float e = ex2(t + (kPBias - (n == -INFINITY ? 0.0f : n)));
        m = n;
        l = fmaf(l, s, e);
        const float so = s * back, eo = e * vf;
        back = 1.0f;
        acc.x = fmaf(acc.x, so, v0.x * eo);
        acc.y = fmaf(acc.y, so, v0.y * eo);
        acc.z = fmaf(acc.z, so, v1.x * eo);
        acc.w = fmaf(acc.w, so, v1.y * eo);
      }
    }
  }
}

template <int NR, int RT>
__global__ void __launch_bounds__(Cfg<NR, RT>::kThreads) __maxnreg__((Cfg<NR, RT>::kRegs)) attention_small_kernel(const AttnParams p) {
  using C = Cfg<NR, RT>;
  constexpr int kStages = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::offBar);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::offMisc);
  volatile int* wide_flag = abort_flag + 1;  // V exponents more than kSpread apart
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t csize = (uint32_t)p.cluster, parts = (uint32_t)p.parts;  // clusters lie along x
  const uint32_t rank = blockIdx.x % parts;

  // unit: row tile fastest, then kv head, then sequence
  const uint32_t unit = blockIdx.x / parts;
  const int rt = (int)(unit % (uint32_t)p.n_rt);
  const uint32_t u1 = unit / (uint32_t)p.n_rt;
  const int hk = (int)(u1 % (uint32_t)p.c.heads), b = (int)(u1 / (uint32_t)p.c.heads);

  bool bad = false;
  const int len = clamp_len(p.lens[b], p.W * p.c.P, &bad);
  const int nq = p.q_lens ? clamp_len(p.q_lens[b], p.Sq, &bad) : p.Sq;
  if (bad && threadIdx.x == 0 && rank == 0 && rt == 0 && hk == 0) report(p.status, DEMON_DEV_BAD_ARG, 63);
  const int n_rows = p.Sq * p.G, row0 = rt * C::kRows * RT;  // below 2^31 (checked on the host)
  const int i0 = row0 / p.G, i1 = imin((row0 + C::kRows * RT - 1) / p.G, nq - 1);
  Keys ks;
  ks.lo = ks.hi = ks.lo_all = ks.hi_all = 0;
  if (i0 <= i1) ks = visible(i0, i1, len, nq, p.causal != 0, p.window);
  const int tile_lo = ks.lo / kTile, tile_hi = ks.hi > ks.lo ? (ks.hi + kTile - 1) / kTile : tile_lo;
  // this CTA's tiles: an even share
  const int n_all = tile_hi - tile_lo, share = n_all / (int)parts, extra = n_all - share * (int)parts;
  const int first = tile_lo + (int)rank * share + imin((int)rank, extra), n_tiles = share + ((int)rank < extra ? 1 : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2 * RT);
    }
    *abort_flag = 0;
    *wide_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  const int step = imin(p.c.P, kTile);  // keys per piece: what of a page lies in a tile
  const int pieces = kTile / step;

  // per-warp partial results: accumulator j of row tile r holds channels 16 g + 2 j (+ 1) of rows
  // 2 c, 2 c + 1 of the tile
  float o[NR][8][4];
  float m[NR][2], l[NR][2];
  int e_ref = kMinExp;
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r][0] = m[r][1] = -INFINITY;
    l[r][0] = l[r][1] = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[r][j][0] = o[r][j][1] = o[r][j][2] = o[r][j][3] = 0.0f;
  }

  if (warp == kKeyWarps * RT) {
    // ------------------------------------------------------------------------ copies
    // a lane per piece: 32 pieces' page ids and scales at a time, then their tiles in turn
    const int32_t* row = p.table + b * p.ld_table;
    const int n_pieces = n_tiles * pieces;
    bool ok = true;
    int issued = 0;  // tiles whose copies were started
    int e_lo = kMaxExp, e_hi = kMinExp;  // V exponents
    for (int base = 0; ok && base < n_pieces; base += 32) {
      const int pc = base + lane;
      int pid = -1, key = 0;
      float sk = -1.0f, sv = 0.0f;  // a negative K scale marks a piece without a page
      if (pc < n_pieces) {
        key = first * kTile + pc * step;
        if (key < ks.hi && key + step > ks.lo) {
          pid = page_id(row, p.W, key / p.c.P, p.c.pages);
          if (pid >= 0) {
            sk = fabsf(__ldg(p.c.scale[0] + (int64_t)pid * p.c.heads + hk));
            sv = __ldg(p.c.scale[1] + (int64_t)pid * p.c.heads + hk);
          } else {
            report(p.status, DEMON_DEV_BAD_ARG, 64);
          }
        }
      }
      if (pid >= 0) {
        e_lo = imin(e_lo, scale_exp(sv));
        e_hi = imax(e_hi, scale_exp(sv));
      }
      const int n_here = imin(32, n_pieces - base);
      for (int t = 0; t < n_here && ok; t += pieces) {
        const int tile = (base + t) / pieces, s = tile % kStages;
        ok = bounded_wait(&empty[s], ((uint32_t)(tile / kStages) & 1u) ^ 1u, abort_flag, p, 65);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool mine = lane >= t && lane < t + pieces;
        const uint32_t here = __ballot_sync(0xffffffffu, mine && pid >= 0);
        if (mine) {
          const uint32_t sc = sbase + C::offScale + (s * 4 + lane - t) * 8;
          st_shared_f32(sc, sk);
          st_shared_f32(sc + 4, sv);
        }
        __syncwarp();
        const uint32_t bytes = (uint32_t)(step * kHeadDim);
        if (lane == t) mbar_arrive_expect_tx(&full[s], 2 * bytes * __popc(here));
        __syncwarp();
        if (mine && pid >= 0) {
          const int64_t src = (((int64_t)pid * p.c.heads + hk) * p.c.P + key % p.c.P) * kHeadDim;
          const uint32_t dst = sbase + s * 2 * kHalf + (lane - t) * bytes;
          bulk_load_s(dst, p.c.codes[0] + src, bytes, &full[s]);
          bulk_load_s(dst + kHalf, p.c.codes[1] + src, bytes, &full[s]);
        }
        ++issued;
        __syncwarp();
      }
    }
    e_lo = __reduce_min_sync(0xffffffffu, e_lo);
    e_hi = __reduce_max_sync(0xffffffffu, e_hi);
    if (lane == 0 && e_hi - e_lo > kSpread) *wide_flag = 1;
    if (!ok) {  // gave up: no copy may be in flight when the CTA leaves
      volatile int never = 0;
      for (int t = imax(issued - kStages, 0); t < issued; ++t)
        mbar_wait(&full[t % kStages], (uint32_t)(t / kStages) & 1u, &never, globaltimer(), p.status, 66);
    }
  } else {
    // ------------------------------------------------------------------------ key loop
    const int kw = warp % kKeyWarps, wt = warp / kKeyWarps;  // part of the keys, row group
    // Q^T: row g of each row tile, k-step s, lane c: channels 16 c + 64 (s / 4) + 4 (s % 4) + 0..3, as
    // K's codes lie
    uint32_t qf[NR][8][2];  // (NR 2: read again from shared memory for every step)
    float fac[NR][2];  // score factors and positions of rows 2 c, 2 c + 1
    int pos[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int grow = row0 + wt * C::kRows + 8 * r + g;
      const int i = grow / p.G, gq = grow - i * p.G;
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = make_uint4(0, 0, 0, 0);
      if (grow < n_rows && i < nq) {
        const __nv_bfloat16* q = p.q + b * p.q_seq + (int64_t)i * p.q_row + (int64_t)(hk * p.G + gq) * p.q_head;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(q + 16 * c + 64 * (j >> 1) + 8 * (j & 1)));
      }
      uint32_t mx = 0;  // infinities and NaN do not count, and pass through
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
        for (int i2 = 0; i2 < 4; ++i2) {
          const uint32_t a = x[i2] & 0x7FFF7FFFu;
          mx = __vmaxu2(mx, a & __vcmpltu2(a, 0x7F807F80u));
        }
      }
      mx = max(mx & 0xFFFFu, mx >> 16);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int k = imax((int)(mx >> 7) - 127 - 13, -126);  // |q| 2^-k < 2^14
      const float2 mul = make_float2(exp2i(-k), exp2i(-k));
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const uint4& ww = w[2 * (s >> 2) + ((s & 3) >> 1)];
        const float2 f0 = mul_f2(bf2_f2((s & 1) ? ww.z : ww.x), mul), f1 = mul_f2(bf2_f2((s & 1) ? ww.w : ww.y), mul);
        qf[r][s][0] = pack_f16x2(f0.x, f0.y);
        qf[r][s][1] = pack_f16x2(f1.x, f1.y);
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        fac[r][x] = exp2i(__shfl_sync(0xffffffffu, k, 4 * (2 * c + x))) * p.scale_log2;
        pos[r][x] = len - nq + __shfl_sync(0xffffffffu, i, 4 * (2 * c + x));
      }
    }
    if (C::kQShared) {
      if (kw == 0) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          st_shared_v4(sbase + C::offQ + ((wt * 8 + s) * 32 + lane) * 16, qf[0][s][0], qf[0][s][1], qf[NR - 1][s][0],
                       qf[NR - 1][s][1]);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kKeyWarps * RT * 32) : "memory");  // the key warps
    }
    // keys of a 16-key block: A row x is key 4 (x % 8 / 2) + 2 (x / 8) + x % 2, so that the P operand's
    // columns of lane c are keys 4 c .. 4 c + 3
    const int kkey = 4 * (g >> 1) + (g & 1);
    const uint32_t k_off = (uint32_t)((kw & 1) * kWarpKeys + kkey) * kHeadDim + 16 * c;
    const uint32_t v_off = (uint32_t)kHalf + (uint32_t)((kw & 1) * kWarpKeys + 4 * c) * kHeadDim + 16 * g;

    bool ok = true;
    for (int t = kw >> 1; t < n_tiles; t += 2) {
      const int s = t % kStages;
      ok = bounded_wait(&full[s], (uint32_t)(t / kStages) & 1u, abort_flag, p, 67);
      ok = __all_sync(0xffffffffu, ok);
      __syncwarp();  // together for the MMAs
      if (!ok) break;
      const int j0 = (first + t) * kTile + (kw & 1) * kWarpKeys;
      if (j0 < ks.hi && j0 + kWarpKeys > ks.lo) {
        const uint32_t st = sbase + s * 2 * kHalf;
        float sk[2];
        int ev[2];
        bool there[2];  // keys 16 z .. of the step: a page, and some row that sees them
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t sc = sbase + C::offScale + (s * 4 + ((kw & 1) * kWarpKeys + 16 * z) / step) * 8;
          sk[z] = ld_shared_f32(sc);
          ev[z] = scale_exp(ld_shared_f32(sc + 4));
          there[z] = !(sk[z] < 0.0f) && j0 + 16 * z < ks.hi && j0 + 16 * z + 16 > ks.lo;
        }
        float sa[2][NR][4];
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int r = 0; r < NR; ++r) sa[z][r][0] = sa[z][r][1] = sa[z][r][2] = sa[z][r][3] = 0.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint4 kx[2], ky[2];
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            kx[z] = ld_shared_v4(st + k_off + 16 * z * kHeadDim + 64 * half);
            ky[z] = ld_shared_v4(st + k_off + (16 * z + 2) * kHeadDim + 64 * half);
          }
#pragma unroll
          for (int q4 = 0; q4 < 4; ++q4) {
            uint32_t qb[NR][2];
            if (C::kQShared) {
              const uint4 q = ld_shared_v4(sbase + C::offQ + ((wt * 8 + 4 * half + q4) * 32 + lane) * 16);
              qb[0][0] = q.x;
              qb[0][1] = q.y;
              qb[NR - 1][0] = q.z;
              qb[NR - 1][1] = q.w;
            } else {
              qb[0][0] = qf[0][4 * half + q4][0];
              qb[0][1] = qf[0][4 * half + q4][1];
            }
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t xs[4] = {kx[z].x, kx[z].y, kx[z].z, kx[z].w}, ys[4] = {ky[z].x, ky[z].y, ky[z].z, ky[z].w};
              uint32_t a[4];  // keys (x, y), channels 0, 1 and 2, 3 of the word
              e4m3x4_f16(xs[q4], a[0], a[2]);
              e4m3x4_f16(ys[q4], a[1], a[3]);
#pragma unroll
              for (int r = 0; r < NR; ++r) mma_f16(sa[z][r], a, qb[r][0], qb[r][1]);
            }
          }
        }
        // scores; accumulator i of block z is key kkey + 2 (i / 2) + 16 z of row 2 c + i % 2
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float f0 = fminf(fac[r][0] * sk[z], kMaxFactor), f1 = fminf(fac[r][1] * sk[z], kMaxFactor);
            sa[z][r][0] *= f0;
            sa[z][r][1] *= f1;
            sa[z][r][2] *= f0;
            sa[z][r][3] *= f1;
          }
        const bool whole = there[0] && there[1] && j0 >= ks.lo_all && j0 + kWarpKeys <= ks.hi_all;
        if (!whole) {
#pragma unroll
          for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int r = 0; r < NR; ++r)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int j = j0 + 16 * z + kkey + 2 * (i >> 1), at = pos[r][i & 1];
                const bool sees = there[z] && j < len && (!p.causal || j <= at) &&
                                  (p.window < 0 || (j <= at + p.window && j >= at - p.window));
                if (!sees) sa[z][r][i] = -INFINITY;
              }
        }
        // running maximum and unit
        const int eu = imax(e_ref, imax(there[0] ? ev[0] : kMinExp, there[1] ? ev[1] : kMinExp));
        float mx[NR][2];
        bool up = eu != e_ref;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mx[r][x] = oct_max(fmaxf(fmaxf(sa[0][r][x], sa[0][r][2 + x]), fmaxf(sa[1][r][x], sa[1][r][2 + x])));
            up = up || mx[r][x] > m[r][x];
          }
        if (__any_sync(0xffffffffu, up)) {
          const float uf = unit_factor(e_ref, eu);
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float f[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float n = fmaxf(m[r][x], mx[r][x]);
              const float a = n == -INFINITY ? 1.0f : ex2(m[r][x] - n);
              l[r][x] *= a;
              m[r][x] = n;
              f[x] = a * uf;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[r][j][0] *= f[0];
              o[r][j][1] *= f[1];
              o[r][j][2] *= f[0];
              o[r][j][3] *= f[1];
            }
          }
          e_ref = eu;
        }
        uint32_t pb[2][NR][2];  // P^T operands
        bool apart = false;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int de = there[z] ? ev[z] - eu : 0;  // <= 0
          apart = apart || de < kFoldMin;
          const float fold = de < kFoldMin ? 1.0f : exp2i(de);
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float mm = m[r][i & 1];
              e[i] = ex2(sa[z][r][i] + (kPBias - (mm == -INFINITY ? 0.0f : mm)));
              l[r][i & 1] += e[i];
              e[i] *= fold;
            }
            pb[z][r][0] = transpose_8x8(pack_f16x2(e[0], e[1]));
            pb[z][r][1] = transpose_8x8(pack_f16x2(e[2], e[3]));
          }
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint4 w[4];  // V: channels 16 g .. 16 g + 15 of keys 4 c .. 4 c + 3
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = ld_shared_v4(st + v_off + (16 * z + i) * kHeadDim);
          if (!whole) {
            if (!there[z]) continue;  // (uniform) nothing of the block counts, and it may not have been copied
            // a NaN of V in a key that some row does not see: it must not reach that row as 0 * NaN
            uint32_t nn = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) nn |= nan_bytes(w[i].x) | nan_bytes(w[i].y) | nan_bytes(w[i].z) | nan_bytes(w[i].w);
            if (__any_sync(0xffffffffu, nn != 0)) {
              uint32_t x[4][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w},
                                  {w[2].x, w[2].y, w[2].z, w[2].w}, {w[3].x, w[3].y, w[3].z, w[3].w}};
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                uint32_t see = 0;  // bit i: row g of the tile sees key 4 c + i
                const int at = len - nq + (row0 + wt * C::kRows + 8 * r + g) / p.G;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int j = j0 + 16 * z + 4 * c + i;
                  see |= (uint32_t)(j < len && (!p.causal || j <= at) &&
                                    (p.window < 0 || (j <= at + p.window && j >= at - p.window)))
                         << i;
                }
                const uint32_t one = 0x3C00u;
                const uint32_t b0 = ((see & 1u) ? one : 0u) | ((see & 2u) ? one << 16 : 0u);
                const uint32_t b1 = ((see & 4u) ? one : 0u) | ((see & 8u) ? one << 16 : 0u);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  uint32_t a[4];
#pragma unroll
                  for (int q = 0; q < 4; ++q) {  // channel 2 j + q % 2, keys 2 (q / 2) and the next
                    const int sh = 8 * ((2 * j + (q & 1)) & 3);
                    const uint32_t n0 = (nan_bytes(x[2 * (q >> 1)][j >> 1]) >> sh) & 0x80u;
                    const uint32_t n1 = (nan_bytes(x[2 * (q >> 1) + 1][j >> 1]) >> sh) & 0x80u;
                    a[q] = (n0 ? one : 0u) | (n1 ? one << 16 : 0u);
                  }
                  float cnt[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  mma_f16(cnt, a, b0, b1);
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    if (cnt[i] > 0.0f) o[r][j][i] = __int_as_float(0x7FFFFFFF);
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {  // and out of the product
                w[i].x &= ~((nan_bytes(w[i].x) >> 7) * 255u);
                w[i].y &= ~((nan_bytes(w[i].y) >> 7) * 255u);
                w[i].z &= ~((nan_bytes(w[i].z) >> 7) * 255u);
                w[i].w &= ~((nan_bytes(w[i].w) >> 7) * 255u);
              }
            }
          }
          const uint32_t x[4][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w},
                                    {w[2].x, w[2].y, w[2].z, w[2].w}, {w[3].x, w[3].y, w[3].z, w[3].w}};
          // bytes (key 4c, key 4c+1) of channels 2 j, 2 j + 1, and of the other two keys
          auto v_operand = [&](int j, uint32_t (&a)[4]) {
            const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
            e4m3x4_f16(__byte_perm(x[0][j >> 1], x[1][j >> 1], sel), a[0], a[1]);
            e4m3x4_f16(__byte_perm(x[2][j >> 1], x[3][j >> 1], sel), a[2], a[3]);
          };
          if (!__any_sync(0xffffffffu, apart && ev[z] - eu < kFoldMin)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t a[4];
              v_operand(j, a);
#pragma unroll
              for (int r = 0; r < NR; ++r) mma_f16(o[r][j], a, pb[z][r][0], pb[z][r][1]);
            }
          } else {  // (a block of its own: as a choice inside the loop it was predicated, twice the instructions)
            const float back = unit_factor(ev[z], eu);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t a[4];
              v_operand(j, a);
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma_f16(y, a, pb[z][r][0], pb[z][r][1]);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][j][i] = fmaf(y[i], back, o[r][j][i]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int x = 0; x < 2; ++x) l[r][x] = oct_sum(l[r][x]);
  }

  // -------------------------------------------------------------------------- join
  __syncthreads();  // every tile consumed: the ring is free (every copy was waited for)
  if (warp < kKeyWarps * RT) {
    const uint32_t wo = sbase + warp * C::kWarpO, ws = sbase + C::offStat + warp * C::kRows * 12;
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int row = 8 * r + 2 * c + x;
        if (g == 0) {
          st_shared_f32(ws + row * 12, m[r][x]);
          st_shared_f32(ws + row * 12 + 4, l[r][x]);
          // (a unit that others of the warp need must not count for a row that has seen nothing)
          st_shared_f32(ws + row * 12 + 8, __int_as_float(m[r][x] == -INFINITY ? kMinExp : e_ref));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          st_shared_f32x4(wo + (row * kHeadDim + 16 * g + 4 * q) * 4, o[r][2 * q][x], o[r][2 * q][2 + x], o[r][2 * q + 1][x],
                          o[r][2 * q + 1][2 + x]);
      }
  }
  __syncthreads();
  // the CTA's four partial results of each row into one: a warp per row, four channels a lane
  constexpr int n_warps = kKeyWarps * RT + 1;
  const int rows_here = imin(C::kRows * RT, n_rows - row0);
  const auto put_row = [&](int r, float M, float L, int E, const float4& acc) {
    if (p.ws) {
      float* w = p.ws + (((int64_t)unit * (C::kRows * RT) + r) * parts + rank) * kPartFloats;
      *reinterpret_cast<float4*>(w + 4 * lane) = acc;
      if (lane == 0) *reinterpret_cast<float4*>(w + kHeadDim) = make_float4(M, L, __int_as_float(E), 1.0f);
      return;
    }
    st_shared_f32x4(sbase + C::offSum + (r * kHeadDim + 4 * lane) * 4, acc.x, acc.y, acc.z, acc.w);
    if (lane == 0) {
      const uint32_t wr = sbase + C::offRow + r * 12;
      st_shared_f32(wr, M);
      st_shared_f32(wr + 4, L);
      st_shared_f32(wr + 8, __int_as_float(E));
    }
  };
  if (__builtin_expect(*wide_flag == 0, 1)) {
    for (int r = warp; r < rows_here; r += n_warps) {
      const int wt = r / C::kRows, rr = r % C::kRows;
      float mm[kKeyWarps], M = -INFINITY, L = 0.0f;
      int ee[kKeyWarps], E = kMinExp;
#pragma unroll
      for (int k = 0; k < kKeyWarps; ++k) {
        const uint32_t ws = sbase + C::offStat + ((wt * kKeyWarps + k) * C::kRows + rr) * 12;
        mm[k] = ld_shared_f32(ws);
        ee[k] = __float_as_int(ld_shared_f32(ws + 8));
        M = fmaxf(M, mm[k]);
        E = imax(E, ee[k]);
      }
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < kKeyWarps; ++k) {
        const uint32_t ws = sbase + C::offStat + ((wt * kKeyWarps + k) * C::kRows + rr) * 12;
        const float f = join_factor(mm[k], M);
        L = fmaf(ld_shared_f32(ws + 4), f, L);
        const float fo = f * unit_factor(ee[k], E);
        const float4 v = ld_shared_f32x4(sbase + (wt * kKeyWarps + k) * C::kWarpO + (rr * kHeadDim + 4 * lane) * 4);
        acc.x = fmaf(v.x, fo, acc.x);
        acc.y = fmaf(v.y, fo, acc.y);
        acc.z = fmaf(v.z, fo, acc.z);
        acc.w = fmaf(v.w, fo, acc.w);
      }
      put_row(r, M, L, E, acc);
    }
  } else {
    for (int r = warp; r < rows_here; r += n_warps) {
      float M, L;
      int E;
      float4 acc;
      row_of_wide_scales(p, b, hk, row0 + r, len, nq, first * kTile, (first + n_tiles) * kTile, lane, M, L, E, acc);
      put_row(r, M, L, E, acc);
    }
  }
  if (p.ws) return;  // attention_join_kernel does the rest
  if (csize > 1)
    cluster_join();
  else
    __syncwarp();  // a row's result is read by the warp that wrote it
  // rows of the cluster's results shared out over its CTAs
  for (int r = (int)rank * n_warps + warp; r < rows_here; r += (int)csize * n_warps) {
    const int grow = row0 + r;
    float M = -INFINITY, L = 0.0f;
    int E = kMinExp;
    for (uint32_t k = 0; k < csize; ++k) {
      const uint32_t wr = map_rank(sbase + C::offRow + r * 12, k);
      M = fmaxf(M, ld_cluster_f32(wr));
      E = imax(E, __float_as_int(ld_cluster_f32(wr + 8)));
    }
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t k = 0; k < csize; ++k) {
      const uint32_t wr = map_rank(sbase + C::offRow + r * 12, k);
      const float f = join_factor(ld_cluster_f32(wr), M);
      L = fmaf(ld_cluster_f32(wr + 4), f, L);
      const float fo = f * unit_factor(__float_as_int(ld_cluster_f32(wr + 8)), E);
      const float4 v = ld_cluster_f32x4(map_rank(sbase + C::offSum + (r * kHeadDim + 4 * lane) * 4, k));
      acc.x = fmaf(v.x, fo, acc.x);
      acc.y = fmaf(v.y, fo, acc.y);
      acc.z = fmaf(v.z, fo, acc.z);
      acc.w = fmaf(v.w, fo, acc.w);
    }
    store_row(p, b, hk, grow, nq, lane, acc, L, E);
  }
  if (csize > 1) cluster_join();  // no CTA leaves while another still reads its results
}

// The partial results of a row from the workspace: a CTA per row, its warps share the parts.  A part of
// the tensor-core kernel is the row's output over its keys and may be as large as V's largest value, next
// to fp32's: the parts' weights are summed first, and each is multiplied by its share of them.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const AttnParams p, const int tile_rows) {
  __shared__ float4 sums[kJoinWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t unit = blockIdx.x / (uint32_t)tile_rows, rt = unit % (uint32_t)p.n_rt, u1 = unit / (uint32_t)p.n_rt;
  const int hk = (int)(u1 % (uint32_t)p.c.heads), b = (int)(u1 / (uint32_t)p.c.heads);
  const int grow = (int)(rt * (uint32_t)tile_rows + blockIdx.x % (uint32_t)tile_rows);
  if (grow >= p.Sq * p.G) return;
  const float* w = p.ws + (int64_t)blockIdx.x * p.parts * kPartFloats;
  // maximum, unit and sum of weights: every warp the same
  float M = -INFINITY, L = 0.0f;
  int E = kMinExp;
  for (int k0 = 0; k0 < p.parts; k0 += 128) {
    float4 st[4];  // (loads first: in a chain with the sums they took a microsecond of 30)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = k0 + 32 * i + lane;
      st[i] = k < p.parts ? *reinterpret_cast<const float4*>(w + (int64_t)k * kPartFloats + kHeadDim)
                          : make_float4(-INFINITY, 0.0f, __int_as_float(kMinExp), 0.0f);
    }
    const float n = fmaxf(fmaxf(fmaxf(M, st[0].x), fmaxf(st[1].x, st[2].x)), st[3].x);
    L *= join_factor(M, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      L = fmaf(st[i].y, join_factor(st[i].x, n), L);
      E = imax(E, __float_as_int(st[i].z));
    }
    M = n;
  }
  float top = M;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  L *= join_factor(M, top);
  M = top;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) L += __shfl_xor_sync(0xffffffffu, L, d);
  E = __reduce_max_sync(0xffffffffu, E);
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = warp; k < p.parts; k += kJoinWarps) {
    const float* wk = w + (int64_t)k * kPartFloats;
    const float4 st = *reinterpret_cast<const float4*>(wk + kHeadDim);
    if (st.x == -INFINITY) continue;  // no key seen (and O perhaps not written)
    const float fo = join_factor(st.x, M) * st.w * inv * unit_factor(__float_as_int(st.z), E);
    const float4 v = *reinterpret_cast<const float4*>(wk + 4 * lane);
    acc.x = fmaf(v.x, fo, acc.x);
    acc.y = fmaf(v.y, fo, acc.y);
    acc.z = fmaf(v.z, fo, acc.z);
    acc.w = fmaf(v.w, fo, acc.w);
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp > 0) return;
  for (int k = 1; k < kJoinWarps; ++k) {
    const float4 v = sums[k][lane];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
  }
  if (L == L && L != 0.0f) L = 1.0f;  // (divided by already; a NaN stays)
  bool bad = false;  // (reported by the other kernel)
  store_row(p, b, hk, grow, p.q_lens ? clamp_len(p.q_lens[b], p.Sq, &bad) : p.Sq, lane, acc, L, E);
}

}  // namespace small
}  // namespace kv

namespace {

int kv_attn_check(const DemonKvAttnArgs* a) {
  DEMON_CHECK_ARG(a != nullptr, "kv_attention: null argument block");
  int rc = kv_cache_check(&a->cache, "kv_attention");
  if (rc == DEMON_OK) rc = kv_table_check(a->table, a->ld_table, a->B, a->W, a->cache.page_size, "kv_attention");
  if (rc != DEMON_OK) return rc;
  DEMON_CHECK_ARG(a->Sq >= 0 && a->Sq <= kv::kMaxTokens && a->Hq >= 1, "kv_attention: bad sizes Sq=%d Hq=%d", a->Sq, a->Hq);
  DEMON_CHECK_ARG(a->Hq % a->cache.heads == 0, "kv_attention: Hq must be a multiple of the kv heads (Hq=%d, Hk=%d)", a->Hq,
                  a->cache.heads);
  DEMON_CHECK_ARG(a->window >= -1 && a->window <= kv::kMaxTokens, "kv_attention: window must be -1 (none) or 0 .. 2^30 (got %d)",
                  a->window);
  DEMON_CHECK_ARG(a->scale > 0.0f && a->scale < INFINITY, "kv_attention: scale must be positive and finite");
  if (a->B == 0 || a->Sq == 0) return DEMON_OK;
  DEMON_CHECK_ARG(a->q && a->o && a->lens, "kv_attention: null q / o / lens");
  DEMON_CHECK_ARG(((uintptr_t)a->q & 15) == 0 && ((uintptr_t)a->o & 15) == 0, "kv_attention: q and o must be 16-byte aligned");
  DEMON_CHECK_ARG(a->q_seq % 8 == 0 && a->q_row % 8 == 0 && a->q_head % 8 == 0 && a->o_seq % 8 == 0 && a->o_row % 8 == 0 &&
                      a->o_head % 8 == 0,
                  "kv_attention: q / o strides must be multiples of 8 elements");
  return DEMON_OK;
}

// How the small kernel splits a call: `units` row tiles, the keys of each over `parts` CTAs.
struct SmallPlan {
  int64_t n_rt, units;
  int cluster, parts;
  int64_t ws_bytes;  // for partial results, 0 with a cluster
};

template <int NR, int RT>
SmallPlan plan_small(const DemonKvAttnArgs* a, bool workspace) {
  using C = kv::small::Cfg<NR, RT>;
  constexpr int kRows = C::kRows * RT;
  SmallPlan s{};
  s.n_rt = ((int64_t)a->Sq * (a->Hq / a->cache.heads) + kRows - 1) / kRows;
  s.units = (int64_t)a->B * a->cache.heads * s.n_rt;
  int64_t keys = (int64_t)a->W * a->cache.page_size;
  if (a->window >= 0)  // the band of a row tile's tokens
    keys = std::min<int64_t>(keys, kRows / (a->Hq / a->cache.heads) + 2 + (a->causal ? 1LL : 2LL) * a->window);
  const int64_t tiles = (keys + kv::small::kTile - 1) / kv::small::kTile;
  // Keys split over a cluster as far as all CTAs are resident at once (twice over with 32 rows a CTA and
  // 8,192 keys: 24 rows of 8 ragged sequences 103 us, once 117), two tiles or more each: with up to
  // twice as many CTAs, 32 units of 4,096 keys take 22.3 us against 12.8.  Where nothing more fits,
  // halves all the same: they even out sequences of different lengths (256 units of 800 to 8,192 keys
  // 56 us, whole 82; all of 4,096 keys 65 us, whole 52).
  const int kCtas = 148 * (RT == 1 || tiles < 128 ? C::kMinCtas : 2);
  s.cluster = 1;
  while (s.cluster < 16 && s.units * s.cluster * 2 <= kCtas && tiles >= 4 * s.cluster) s.cluster *= 2;
  if (s.cluster == 1 && s.units < kCtas && tiles >= 4) s.cluster = 2;
  s.parts = s.cluster;
  // Longer tables: as many parts as fill the SMs, any number, joined by a second kernel through a
  // workspace (the cluster's power of two up to 16 against it: 64 units of 16,384 keys 64.6 and 51 us,
  // 16 units of 100,000 keys 143 and 82 us, 4 of them 61 and 29 us; below 8,192 keys the second launch
  // and the workspace cost what they gain).
  const int64_t parts = s.units > 0 ? std::min<int64_t>(kCtas / s.units, tiles / 6) : 0;
  if (workspace && tiles >= 128 && parts > s.cluster) {
    s.cluster = 1;
    s.parts = (int)parts;
    s.ws_bytes = s.units * kRows * parts * kv::kPartFloats * 4;
  }
  return s;
}

int launch_join(const kv::AttnParams& p, int64_t units, int tile_rows, cudaStream_t st) {
  kv::small::attention_join_kernel<<<(unsigned)(units * tile_rows), kv::small::kJoinWarps * 32, 0, st>>>(p, tile_rows);
  DEMON_CUDA(cudaGetLastError());
  return DEMON_OK;
}

int check_workspace(const DemonKvAttnArgs* a, int64_t bytes) {
  DEMON_CHECK_ARG(((uintptr_t)a->workspace & 15) == 0, "kv_attention: workspace must be 16-byte aligned");
  DEMON_CHECK_ARG(a->workspace_bytes >= bytes, "kv_attention: workspace of %lld bytes, %lld needed",
                  (long long)a->workspace_bytes, (long long)bytes);
  return DEMON_OK;
}

template <int NR, int RT>
int launch_small(kv::AttnParams p, const DemonKvAttnArgs* a, cudaStream_t st) {
  using C = kv::small::Cfg<NR, RT>;
  static std::atomic<uint64_t> attr_done{0};
  const auto kernel = kv::small::attention_small_kernel<NR, RT>;
  if (device_pending(attr_done)) {
    DEMON_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    DEMON_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    mark_device_done(attr_done);
  }
  const int64_t rows = (int64_t)a->Sq * p.G;
  DEMON_CHECK_ARG(rows < ((int64_t)1 << 31) - 64, "kv_attention: too many query rows (%lld)", (long long)rows);
  const SmallPlan s = plan_small<NR, RT>(a, a->workspace != nullptr);
  if (s.ws_bytes > 0) {
    const int rc = check_workspace(a, s.ws_bytes);
    if (rc != DEMON_OK) return rc;
  }
  p.n_rt = (int)s.n_rt;
  const int64_t units = s.units;
  const int cluster = s.cluster;
  p.parts = s.parts;
  p.ws = s.ws_bytes > 0 ? (float*)a->workspace : nullptr;
  DEMON_CHECK_ARG(units * s.parts < ((int64_t)1 << 31), "kv_attention: too many work units (%lld)", (long long)units);
  p.cluster = cluster;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * s.parts), 1, 1);
  cfg.blockDim = dim3(C::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  DEMON_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return p.ws ? launch_join(p, units, C::kRows * RT, st) : DEMON_OK;
}


// The tensor-core kernel's split: blocks of 2 Tt tokens, the keys of each over `parts` units.
struct TcPlan {
  int64_t blocks;
  int parts;
  double us;         // estimate
  int64_t ws_bytes;  // 0 with one part
};

TcPlan plan_tc(const DemonKvAttnArgs* a, bool workspace) {
  const int G = a->Hq / a->cache.heads, tokens = 2 * (128 / G);
  double keys = (double)a->W * a->cache.page_size;
  if (a->window >= 0) keys = std::min(keys, (double)tokens + a->window * (a->causal ? 1.0 : 2.0));
  const double tiles = std::ceil(keys / 128.0);
  TcPlan s{};
  s.blocks = (int64_t)a->B * a->cache.heads * ((a->Sq + tokens - 1) / tokens);
  s.parts = 1;
  // 2.7 us per tile of 128 keys for 256 rows on one SM, 2 for a unit's start and output
  s.us = std::ceil(s.blocks / 148.0) * (tiles * 2.7 + 2.0);
  // Few blocks: their keys in parts of four tiles or more (512 tokens of 4 heads over 2, 20,000 keys:
  // 151 us whole, 50 in parts), where that takes a fifth off the estimate
  // with 4 us for the second kernel and the partial results' way through memory.
  if (workspace && s.blocks < 148) {
    const double whole = s.us, rows = (double)s.blocks * tokens * G;
    const int64_t most = std::max<int64_t>(148 / s.blocks, 8);  // (8: 80 blocks of 76 tiles 265 us whole, 180 in parts)
    for (int parts = 2; parts <= most && parts * 4 <= tiles; ++parts) {
      const double us = std::ceil(s.blocks * parts / 148.0) * (std::ceil(tiles / parts) * 2.7 + 2.0) + 4.0 +
                        rows * parts * (2 * kv::kPartFloats * 4) / 4e6;
      if (us < 0.8 * whole && us < s.us) s.us = us, s.parts = parts;
    }
    if (s.parts > 1) s.ws_bytes = s.blocks * tokens * G * s.parts * kv::kPartFloats * 4;
  }
  return s;
}

int launch_tc(kv::AttnParams p, const DemonKvAttnArgs* a, cudaStream_t st) {
  const TcPlan s = plan_tc(a, a->workspace != nullptr);
  p.parts = s.parts;
  if (s.ws_bytes > 0) {
    const int rc = check_workspace(a, s.ws_bytes);
    if (rc != DEMON_OK) return rc;
    p.ws = (float*)a->workspace;
  }
  int rc = kv::attention_tc(p, st);
  if (rc != DEMON_OK || !p.ws) return rc;
  const int tokens = 2 * (128 / p.G);
  p.n_rt = (p.Sq + tokens - 1) / tokens;
  return launch_join(p, s.blocks, tokens * p.G, st);
}

enum class Kernel { kRows8, kRows16, kRows32, kTc };

// `workspace`: there is one (its size is checked when the kernel that takes it is launched).
Kernel kernel_for(const DemonKvAttnArgs* a, bool workspace) {
  const int G = a->Hq / a->cache.heads;
  const int64_t rows = (int64_t)a->Sq * G;
  // DEMON_KV_ATTENTION=small / tc takes one of the two kernels for every call (tests, measurements)
  const char* force = std::getenv("DEMON_KV_ATTENTION");
  if (force && std::strcmp(force, "tc") == 0 && G <= 128) return Kernel::kTc;
  if (rows <= 8) return Kernel::kRows8;
  if (rows <= 16) return Kernel::kRows16;
  if (G > 128 || (force && std::strcmp(force, "small") == 0)) return Kernel::kRows32;
  // More rows: the lesser of two estimates, with the keys that the table covers, or those of the
  // window.  The small kernel reads the keys once per 32 rows, at about 2 TB/s; the tensor-core kernel
  // see above (without a workspace it takes whole key ranges: 64 tokens of 8 heads over one kv head and
  // 20,000 keys 387 us, the small kernel 82, parts 41).  8 kv heads, both measured: 24 rows over 16,384
  // keys small 32 us, tc 39; 128 rows over 20,000 keys 81 and 45; 60 rows over 4 x 20,000 keys 130 and
  // 122, 1,500 rows over 16 x 256 keys 597 and 64; 2 heads, 600 rows over 4,096 keys 37 and 38; 1 head,
  // 240 rows over 2,000 keys 22 and 32.
  double keys = (double)a->W * a->cache.page_size;
  if (a->window >= 0) keys = std::min(keys, 256.0 / G + a->window * (a->causal ? 1.0 : 2.0));
  const double us_small = (double)a->B * a->cache.heads * (double)((rows + 31) / 32) * keys * 256.0 / 2.0e6;
  return plan_tc(a, workspace).us < us_small ? Kernel::kTc : Kernel::kRows32;
}

}  // namespace
}  // namespace demon

using namespace demon;

extern "C" int demon_kv_attention(const DemonKvAttnArgs* a, void* stream) {
  DEMON_API_BEGIN();
  const int rc = kv_attn_check(a);
  if (rc != DEMON_OK) return rc;
  if (a->B == 0 || a->Sq == 0) return DEMON_OK;
  kv::AttnParams p{};
  p.c = kv_cache(&a->cache);
  p.q = (const __nv_bfloat16*)a->q;
  p.q_seq = a->q_seq, p.q_row = a->q_row, p.q_head = a->q_head;
  p.o = (__nv_bfloat16*)a->o;
  p.o_seq = a->o_seq, p.o_row = a->o_row, p.o_head = a->o_head;
  p.table = a->table, p.lens = a->lens, p.q_lens = a->q_lens, p.ld_table = a->ld_table;
  p.B = a->B, p.Sq = a->Sq, p.Hq = a->Hq, p.G = a->Hq / a->cache.heads, p.W = a->W;
  p.causal = a->causal != 0, p.window = std::min(a->window, kv::kMaxTokens - 2);
  p.scale_log2 = (float)((double)a->scale * 1.4426950408889634);
  p.status = status_word();
  switch (kernel_for(a, a->workspace != nullptr)) {
    case Kernel::kTc: return launch_tc(p, a, (cudaStream_t)stream);
    case Kernel::kRows8: return launch_small<1, 1>(p, a, (cudaStream_t)stream);
    case Kernel::kRows16: return launch_small<2, 1>(p, a, (cudaStream_t)stream);
    default: return launch_small<2, 2>(p, a, (cudaStream_t)stream);
  }
}

extern "C" int64_t demon_kv_attention_workspace(const DemonKvAttnArgs* a) {
  if (kv_attn_check(a) != DEMON_OK || a->B == 0 || a->Sq == 0) return 0;  // (the call itself says why)
  switch (kernel_for(a, true)) {
    case Kernel::kTc: return plan_tc(a, true).ws_bytes;
    case Kernel::kRows8: return plan_small<1, 1>(a, true).ws_bytes;
    case Kernel::kRows16: return plan_small<2, 1>(a, true).ws_bytes;
    default: return plan_small<2, 2>(a, true).ws_bytes;
  }
}
