// kv_attention.cu -- attention of new queries over a paged E4M3 K/V cache:
//   o[i] = sum_j softmax_j(scale q[i] . k[j]) v[j]   over the keys j that query i sees
// (j < length, causal and band limits; a query that sees no key gives zeros).
//
// Small kernel (few query rows per kv head: single tokens, short chunks).  Bound by reading the
// codes, 256 bytes per key and kv head.  All G = Hq / Hk query heads of a kv head and up to 16
// query tokens share one pass over its keys: a row is (token, query head), row r = i * G + g.
// A CTA takes 16 * RT rows and a range of keys in tiles of 64; one warp copies the tiles of K
// and V codes, as they lie in the pages, into a ring in shared memory (bulk copies of a page's
// 2 to 8 KB, mbarriers); four warps per 16 rows each take 16 keys of a tile.  The keys of a row
// tile are split over a thread-block cluster, which joins its partial results through
// distributed shared memory: one launch, no workspace.
//
// A warp's step on 16 keys, all in registers (mma.sync m16n8k16, fp32 accumulators):
//   S = Q K^T: E4M3 codes become f16 exactly; Q is f16 too, each row times a power of two that
//     brings its largest value to [2^13, 2^14) (exact down to 2^-28 of that value).  The page's
//     K scale, the row's power and the softmax scale are one fp32 factor of the score.
//   softmax: running maximum m and sum l per row; p = 2^(t - m + 14), so that f16 keeps p's full
//     precision down to 2^-28 of the row's largest; l sums the unrounded p.
//   O += P V: the codes of V go in unscaled; O is held in units of 2^e_ref, the largest V scale
//     met so far.  A page with a smaller scale 2^e has P multiplied by 2^(e - e_ref), exactly;
//     if that is below 2^-8, its product goes through accumulators of its own, so that P's
//     precision never depends on the scales.
// The f16 conversions take one instruction per two codes, and only a byte permute stands
// between V's rows and the operand layout (the keys and channels of a step may be taken in any
// order as long as both operands agree).
#include <algorithm>

#include "demon_host.h"
#include "kv_common.cuh"
#include "kv_host.h"

namespace demon {
namespace kv {

namespace small {

constexpr int kTile = 64;                  // keys per stage
constexpr int kWarpKeys = 16;              // keys per warp and stage
constexpr int kHalf = kTile * kHeadDim;    // one stage's K (or V) codes, 8 KB
constexpr int kStages = 6;
constexpr int kKeyWarps = kTile / kWarpKeys;
constexpr float kPBias = 14.0f;            // p is scaled by 2^14 (see above)
constexpr int kFoldMin = -8;               // smallest V scale, relative to e_ref, folded into P

constexpr int offScale = kStages * 2 * kHalf;           // [stage][piece][K, V] fp32
constexpr int offBar = offScale + kStages * 4 * 2 * 4;  // full[stage], empty[stage]
constexpr int offMisc = offBar + 2 * kStages * 8;       // abort flag
constexpr int kSmem = offMisc + 16;

// After the key loop the ring holds the partial results: per warp O [16][128] fp32, then the
// CTA's sum [16 RT][128], and the rows' statistics.
constexpr int kWarpO = 16 * kHeadDim * 4;
template <int RT>
struct Join {
  static constexpr int offSum = kKeyWarps * RT * kWarpO;
  static constexpr int offStat = offSum + RT * kWarpO;               // per warp and row: m, l, e
  static constexpr int offRow = offStat + kKeyWarps * RT * 16 * 12;  // CTA, per row: M, L, E
  static constexpr int kEnd = offRow + RT * 16 * 12;
  static_assert(kEnd <= offScale, "partial results must fit into the ring");
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
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

// Factor that brings a partial result with maximum m (and V unit 2^e) to maximum M (unit 2^E).
__device__ __forceinline__ float join_factor(float m, float M) {
  return m == -INFINITY ? 0.0f : ex2(m - M);
}
__device__ __forceinline__ float unit_factor(int e, int E) { return e - E < -126 ? 0.0f : exp2i(imin(e - E, 0)); }

template <int RT>
__global__ void __launch_bounds__(kKeyWarps* RT * 32 + 32, 2 / RT) attention_small_kernel(const AttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sbase = smem_u32(smem);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + offBar);
  uint64_t* empty = full + kStages;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + offMisc);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t t0 = globaltimer();
  uint32_t rank, csize;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));

  // unit: row tile fastest, then kv head, then sequence
  const uint32_t unit = blockIdx.x / csize;
  const int rt = (int)(unit % (uint32_t)p.n_rt);
  const uint32_t u1 = unit / (uint32_t)p.n_rt;
  const int hk = (int)(u1 % (uint32_t)p.c.heads), b = (int)(u1 / (uint32_t)p.c.heads);

  bool bad = false;
  const int len = clamp_len(p.lens[b], p.W * p.c.P, &bad);
  const int nq = p.q_lens ? clamp_len(p.q_lens[b], p.Sq, &bad) : p.Sq;
  if (bad && threadIdx.x == 0 && rank == 0 && rt == 0 && hk == 0) report(p.status, DEMON_DEV_BAD_ARG, 63);
  const int64_t n_rows = (int64_t)p.Sq * p.G, row0 = (int64_t)rt * 16 * RT;
  const int i0 = (int)(row0 / p.G), i1 = imin((int)((row0 + 16 * RT - 1) / p.G), nq - 1);
  Keys ks;
  ks.lo = ks.hi = ks.lo_all = ks.hi_all = 0;
  if (i0 <= i1) ks = visible(i0, i1, len, nq, p.causal != 0, p.window);
  const int tile_lo = ks.lo / kTile, tile_hi = ks.hi > ks.lo ? (ks.hi + kTile - 1) / kTile : tile_lo;
  // this CTA's tiles: an even share of the cluster's
  const int n_all = tile_hi - tile_lo, share = n_all / (int)csize, extra = n_all - share * (int)csize;
  const int first = tile_lo + (int)rank * share + imin((int)rank, extra), n_tiles = share + ((int)rank < extra ? 1 : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kKeyWarps * RT);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();

  const int step = imin(p.c.P, kTile);  // keys per piece: what of a page lies in a tile
  const int pieces = kTile / step;

  // per-warp partial results (warps of the key loop)
  float o[16][4];
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  int e_ref = kMinExp;
  const int g = lane >> 2, c = lane & 3;
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

  if (warp == kKeyWarps * RT) {
    // ------------------------------------------------------------------------ copies
    // a lane per piece: 32 pieces' page ids and scales at a time, then their tiles in turn
    const int32_t* row = p.table + b * p.ld_table;
    const int n_pieces = n_tiles * pieces;
    bool ok = true;
    int issued = 0;  // tiles whose copies were started
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
      const int n_here = imin(32, n_pieces - base);
      for (int t = 0; t < n_here && ok; t += pieces) {
        const int tile = (base + t) / pieces, s = tile % kStages;
        ok = mbar_wait(&empty[s], ((uint32_t)(tile / kStages) & 1u) ^ 1u, abort_flag, t0, p.status, 65);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const bool mine = lane >= t && lane < t + pieces;
        const uint32_t here = __ballot_sync(0xffffffffu, mine && pid >= 0);
        if (mine) {
          const uint32_t sc = sbase + offScale + (s * 4 + lane - t) * 8;
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
    if (!ok) {  // gave up: no copy may be in flight when the CTA leaves
      volatile int never = 0;
      for (int t = imax(issued - kStages, 0); t < issued; ++t)
        mbar_wait(&full[t % kStages], (uint32_t)(t / kStages) & 1u, &never, globaltimer(), p.status, 66);
    }
  } else {
    // ------------------------------------------------------------------------ key loop
    const int kw = warp % kKeyWarps, wt = warp / kKeyWarps;  // 16-key part of a tile, row tile
    // this lane's two rows of Q: rows g and g + 8 of the warp's sixteen
    uint32_t qf[8][4];
    float fac[2];
    int pos[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t r = row0 + wt * 16 + g + 8 * half;
      const int i = (int)(r / p.G), gq = (int)(r - (int64_t)i * p.G);
      const bool valid = r < n_rows && i < nq;
      pos[half] = len - nq + i;
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = make_uint4(0, 0, 0, 0);
      if (valid) {
        const __nv_bfloat16* q = p.q + b * p.q_seq + (int64_t)i * p.q_row + (int64_t)(hk * p.G + gq) * p.q_head;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __ldg(reinterpret_cast<const uint4*>(q + 16 * c + 64 * (j >> 1) + 8 * (j & 1)));
      }
      uint32_t mx = 0;
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
      fac[half] = exp2i(k);
      // k-step s, lane c: channels 16 c + 64 (s / 4) + 4 (s % 4) + 0..3, as K's codes lie
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        const uint4& ww = w[2 * (s >> 2) + ((s & 3) >> 1)];
        const uint32_t x0 = (s & 1) ? ww.z : ww.x, x1 = (s & 1) ? ww.w : ww.y;
        const float2 f0 = mul_f2(bf2_f2(x0), mul), f1 = mul_f2(bf2_f2(x1), mul);
        qf[s][half] = pack_f16x2(f0.x, f0.y);
        qf[s][2 + half] = pack_f16x2(f1.x, f1.y);
      }
    }
    // keys of a step: S column n of 8-column tile nt is key 4 (n / 2) + 2 nt + n % 2, so that the
    // P operand's columns of lane c are keys 4 c .. 4 c + 3
    const int kkey = 4 * (g >> 1) + (g & 1);
    const uint32_t k_off = (uint32_t)(kw * kWarpKeys + kkey) * kHeadDim + 16 * c;
    const uint32_t v_off = (uint32_t)kHalf + (uint32_t)(kw * kWarpKeys + 4 * c) * kHeadDim + 16 * g;
    const int piece = kw * kWarpKeys / step;

    bool ok = true;
    for (int t = 0; t < n_tiles; ++t) {
      const int s = t % kStages;
      ok = mbar_wait(&full[s], (uint32_t)(t / kStages) & 1u, abort_flag, t0, p.status, 67);
      ok = __all_sync(0xffffffffu, ok && *abort_flag == 0);
      if (!ok) break;
      const int j0 = (first + t) * kTile + kw * kWarpKeys;
      const uint32_t sc = sbase + offScale + (s * 4 + piece) * 8;
      const float sk = ld_shared_f32(sc), sv = ld_shared_f32(sc + 4);
      if (!(sk < 0.0f) && j0 < ks.hi && j0 + kWarpKeys > ks.lo) {
        const uint32_t st = sbase + s * 2 * kHalf;
        float sa[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          sa[nt][0] = sa[nt][1] = sa[nt][2] = sa[nt][3] = 0.0f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 w = ld_shared_v4(st + k_off + nt * 2 * kHeadDim + 64 * half);
            uint32_t x0, x1;
            e4m3x4_f16(w.x, x0, x1);
            mma_f16(sa[nt], qf[4 * half + 0], x0, x1);
            e4m3x4_f16(w.y, x0, x1);
            mma_f16(sa[nt], qf[4 * half + 1], x0, x1);
            e4m3x4_f16(w.z, x0, x1);
            mma_f16(sa[nt], qf[4 * half + 2], x0, x1);
            e4m3x4_f16(w.w, x0, x1);
            mma_f16(sa[nt], qf[4 * half + 3], x0, x1);
          }
        }
        const float f0 = fac[0] * sk * p.scale_log2, f1 = fac[1] * sk * p.scale_log2;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          sa[nt][0] *= f0;
          sa[nt][1] *= f0;
          sa[nt][2] *= f1;
          sa[nt][3] *= f1;
        }
        uint4 w[4];  // V: channels 16 g .. 16 g + 15 of keys 4 c .. 4 c + 3
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = ld_shared_v4(st + v_off + i * kHeadDim);
        const bool whole = j0 >= ks.lo_all && j0 + kWarpKeys <= ks.hi_all;
        uint32_t see = 0xFFu;  // bit 4 half + i: row `half` sees key 4 c + i
        if (!whole) {
          see = 0;
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = j0 + 4 * c + i;
              const bool v = j < len && (!p.causal || j <= pos[half]) &&
                             (p.window < 0 || (j <= pos[half] + p.window && j >= pos[half] - p.window));
              see |= (uint32_t)v << (4 * half + i);
            }
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!((see >> (4 * (i >> 1) + 2 * nt + (i & 1))) & 1u)) sa[nt][i] = -INFINITY;
          // a NaN of V in a key that some row does not see: it must not reach that row as 0 * NaN
          uint32_t nn = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) nn |= nan_bytes(w[i].x) | nan_bytes(w[i].y) | nan_bytes(w[i].z) | nan_bytes(w[i].w);
          if (__any_sync(0xffffffffu, nn != 0)) {
            uint32_t a[4];  // who sees what, as a 0 / 1 operand
            const uint32_t one = 0x3C00u;
#pragma unroll
            for (int r = 0; r < 4; ++r) {  // a[0]: row g, keys 4c, 4c+1; a[1]: row g+8; a[2], a[3]: keys 4c+2, 4c+3
              const uint32_t bits = see >> (4 * (r & 1) + 2 * (r >> 1));
              a[r] = ((bits & 1u) ? one : 0u) | ((bits & 2u) ? one << 16 : 0u);
            }
            uint32_t x[4][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w},
                                {w[2].x, w[2].y, w[2].z, w[2].w}, {w[3].x, w[3].y, w[3].z, w[3].w}};
#pragma unroll
            for (int nt = 0; nt < 16; ++nt) {
              const int sh = 8 * (nt & 3);
              const uint32_t n0 = (nan_bytes(x[0][nt >> 2]) >> sh) & 0x80u, n1 = (nan_bytes(x[1][nt >> 2]) >> sh) & 0x80u;
              const uint32_t n2 = (nan_bytes(x[2][nt >> 2]) >> sh) & 0x80u, n3 = (nan_bytes(x[3][nt >> 2]) >> sh) & 0x80u;
              float cnt[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_f16(cnt, a, (n0 ? one : 0u) | (n1 ? one << 16 : 0u), (n2 ? one : 0u) | (n3 ? one << 16 : 0u));
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (cnt[i] > 0.0f) o[nt][i] = __int_as_float(0x7FFFFFFF);
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
        // running maximum
        const float x0 = quad_max(fmaxf(fmaxf(sa[0][0], sa[0][1]), fmaxf(sa[1][0], sa[1][1])));
        const float x1 = quad_max(fmaxf(fmaxf(sa[0][2], sa[0][3]), fmaxf(sa[1][2], sa[1][3])));
        const int ev = scale_exp(sv);
        const int eu = imax(e_ref, ev);  // O's unit from here on
        if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1) || eu != e_ref) {
          const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
          const float a0 = n0 == -INFINITY ? 1.0f : ex2(m0 - n0), a1 = n1 == -INFINITY ? 1.0f : ex2(m1 - n1);
          l0 *= a0;
          l1 *= a1;
          const float uf = unit_factor(e_ref, eu);
          const float b0 = a0 * uf, b1 = a1 * uf;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            o[i][0] *= b0;
            o[i][1] *= b0;
            o[i][2] *= b1;
            o[i][3] *= b1;
          }
          m0 = n0;
          m1 = n1;
          e_ref = eu;
        }
        const float d0 = kPBias - (m0 == -INFINITY ? 0.0f : m0), d1 = kPBias - (m1 == -INFINITY ? 0.0f : m1);
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          sa[nt][0] = ex2(sa[nt][0] + d0);
          sa[nt][1] = ex2(sa[nt][1] + d0);
          sa[nt][2] = ex2(sa[nt][2] + d1);
          sa[nt][3] = ex2(sa[nt][3] + d1);
          l0 += sa[nt][0] + sa[nt][1];
          l1 += sa[nt][2] + sa[nt][3];
        }
        const int de = ev - eu;  // <= 0
        const bool apart = de < kFoldMin;
        const float fold = apart ? 1.0f : exp2i(de);
        const uint32_t pa[4] = {pack_f16x2(sa[0][0] * fold, sa[0][1] * fold), pack_f16x2(sa[0][2] * fold, sa[0][3] * fold),
                                pack_f16x2(sa[1][0] * fold, sa[1][1] * fold), pack_f16x2(sa[1][2] * fold, sa[1][3] * fold)};
        const uint32_t x[4][4] = {{w[0].x, w[0].y, w[0].z, w[0].w}, {w[1].x, w[1].y, w[1].z, w[1].w},
                                  {w[2].x, w[2].y, w[2].z, w[2].w}, {w[3].x, w[3].y, w[3].z, w[3].w}};
        const float back = unit_factor(ev, eu);
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            // bytes (key 4c, key 4c+1) of two channels, and of the other two keys
            const uint32_t sel = hf ? 0x7362u : 0x5140u;
            uint32_t b00, b01, b10, b11;
            e4m3x4_f16(__byte_perm(x[0][q4], x[1][q4], sel), b00, b01);
            e4m3x4_f16(__byte_perm(x[2][q4], x[3][q4], sel), b10, b11);
            const int nt = 4 * q4 + 2 * hf;
            if (!apart) {
              mma_f16(o[nt], pa, b00, b10);
              mma_f16(o[nt + 1], pa, b01, b11);
            } else {
              float y0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma_f16(y0, pa, b00, b10);
              mma_f16(y1, pa, b01, b11);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[nt][i] = fmaf(y0[i], back, o[nt][i]);
                o[nt + 1][i] = fmaf(y1[i], back, o[nt + 1][i]);
              }
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    l0 = quad_sum(l0);
    l1 = quad_sum(l1);
  }

  // -------------------------------------------------------------------------- join
  using J = Join<RT>;
  __syncthreads();  // every tile consumed: the ring is free (every copy was waited for)
  if (warp < kKeyWarps * RT) {
    const uint32_t wo = sbase + warp * kWarpO, ws = sbase + J::offStat + warp * 16 * 12;
    if (c == 0) {
      st_shared_f32(ws + g * 12, m0);
      st_shared_f32(ws + g * 12 + 4, l0);
      st_shared_f32(ws + g * 12 + 8, __int_as_float(e_ref));
      st_shared_f32(ws + (g + 8) * 12, m1);
      st_shared_f32(ws + (g + 8) * 12 + 4, l1);
      st_shared_f32(ws + (g + 8) * 12 + 8, __int_as_float(e_ref));
    }
    // O column n of 8-column tile nt is channel 16 n + nt
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      st_shared_f32x4(wo + (g * kHeadDim + 32 * c + 4 * q4) * 4, o[4 * q4][0], o[4 * q4 + 1][0], o[4 * q4 + 2][0], o[4 * q4 + 3][0]);
      st_shared_f32x4(wo + (g * kHeadDim + 32 * c + 16 + 4 * q4) * 4, o[4 * q4][1], o[4 * q4 + 1][1], o[4 * q4 + 2][1], o[4 * q4 + 3][1]);
      st_shared_f32x4(wo + ((g + 8) * kHeadDim + 32 * c + 4 * q4) * 4, o[4 * q4][2], o[4 * q4 + 1][2], o[4 * q4 + 2][2], o[4 * q4 + 3][2]);
      st_shared_f32x4(wo + ((g + 8) * kHeadDim + 32 * c + 16 + 4 * q4) * 4, o[4 * q4][3], o[4 * q4 + 1][3], o[4 * q4 + 2][3], o[4 * q4 + 3][3]);
    }
  }
  __syncthreads();
  // the CTA's four partial results of each row into one: a warp per row, four channels a lane
  const int n_warps = kKeyWarps * RT + 1;
  for (int r = warp; r < 16 * RT; r += n_warps) {
    const int wt = r >> 4, rr = r & 15;
    float mm[kKeyWarps], M = -INFINITY, L = 0.0f;
    int ee[kKeyWarps], E = kMinExp;
#pragma unroll
    for (int k = 0; k < kKeyWarps; ++k) {
      const uint32_t ws = sbase + J::offStat + ((wt * kKeyWarps + k) * 16 + rr) * 12;
      mm[k] = ld_shared_f32(ws);
      ee[k] = __float_as_int(ld_shared_f32(ws + 8));
      M = fmaxf(M, mm[k]);
      E = imax(E, ee[k]);
    }
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < kKeyWarps; ++k) {
      const uint32_t ws = sbase + J::offStat + ((wt * kKeyWarps + k) * 16 + rr) * 12;
      const float f = join_factor(mm[k], M);
      L = fmaf(ld_shared_f32(ws + 4), f, L);
      const float fo = f * unit_factor(ee[k], E);
      const float4 v = ld_shared_f32x4(sbase + (wt * kKeyWarps + k) * kWarpO + (rr * kHeadDim + 4 * lane) * 4);
      acc.x = fmaf(v.x, fo, acc.x);
      acc.y = fmaf(v.y, fo, acc.y);
      acc.z = fmaf(v.z, fo, acc.z);
      acc.w = fmaf(v.w, fo, acc.w);
    }
    st_shared_f32x4(sbase + J::offSum + (r * kHeadDim + 4 * lane) * 4, acc.x, acc.y, acc.z, acc.w);
    if (lane == 0) {
      const uint32_t wr = sbase + J::offRow + r * 12;
      st_shared_f32(wr, M);
      st_shared_f32(wr + 4, L);
      st_shared_f32(wr + 8, __int_as_float(E));
    }
  }
  cluster_sync();
  // rows of the cluster's results shared out over its CTAs
  for (int r = (int)rank * n_warps + warp; r < 16 * RT; r += (int)csize * n_warps) {
    const int64_t grow = row0 + r;
    if (grow >= n_rows) continue;
    float M = -INFINITY, L = 0.0f;
    int E = kMinExp;
    for (uint32_t k = 0; k < csize; ++k) {
      const uint32_t wr = map_rank(sbase + J::offRow + r * 12, k);
      M = fmaxf(M, ld_cluster_f32(wr));
      E = imax(E, __float_as_int(ld_cluster_f32(wr + 8)));
    }
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t k = 0; k < csize; ++k) {
      const uint32_t wr = map_rank(sbase + J::offRow + r * 12, k);
      const float f = join_factor(ld_cluster_f32(wr), M);
      L = fmaf(ld_cluster_f32(wr + 4), f, L);
      const float fo = f * unit_factor(__float_as_int(ld_cluster_f32(wr + 8)), E);
      const float4 v = ld_cluster_f32x4(map_rank(sbase + J::offSum + (r * kHeadDim + 4 * lane) * 4, k));
      acc.x = fmaf(v.x, fo, acc.x);
      acc.y = fmaf(v.y, fo, acc.y);
      acc.z = fmaf(v.z, fo, acc.z);
      acc.w = fmaf(v.w, fo, acc.w);
    }
    const int i = (int)(grow / p.G), gq = (int)(grow - (int64_t)i * p.G);
    // L == 0: the row sees no key (a NaN score makes L NaN, and stays)
    const float inv = (i < nq && L != 0.0f) ? 1.0f / L : 0.0f;
    const float un = exp2i(E);
    uint2 out = make_uint2(0u, 0u);
    if (inv != 0.0f)
      out = make_uint2(pack_bf16x2(acc.x * inv * un, acc.y * inv * un), pack_bf16x2(acc.z * inv * un, acc.w * inv * un));
    *reinterpret_cast<uint2*>(p.o + b * p.o_seq + (int64_t)i * p.o_row + (int64_t)(hk * p.G + gq) * p.o_head + 4 * lane) = out;
  }
  cluster_sync();  // no CTA leaves while another still reads its results
}

}  // namespace small
}  // namespace kv

namespace {

std::atomic<uint64_t> g_kv_small_attr{0};

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

template <int RT>
int launch_small(const kv::AttnParams& p, int64_t units, int cluster, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * cluster), 1, 1);
  cfg.blockDim = dim3(kv::small::kKeyWarps * RT * 32 + 32, 1, 1);
  cfg.dynamicSmemBytes = kv::small::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  DEMON_CUDA(cudaLaunchKernelEx(&cfg, kv::small::attention_small_kernel<RT>, p));
  return DEMON_OK;
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
  if (device_pending(g_kv_small_attr)) {
    DEMON_CUDA(cudaFuncSetAttribute(kv::small::attention_small_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv::small::kSmem));
    DEMON_CUDA(cudaFuncSetAttribute(kv::small::attention_small_kernel<2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kv::small::kSmem));
    DEMON_CUDA(cudaFuncSetAttribute(kv::small::attention_small_kernel<1>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    DEMON_CUDA(cudaFuncSetAttribute(kv::small::attention_small_kernel<2>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    mark_device_done(g_kv_small_attr);
  }
  const int64_t rows = (int64_t)a->Sq * p.G;
  if (rows > 64 && p.G <= 128) return kv::attention_tc(p, (cudaStream_t)stream);
  const int rt = rows > 16 ? 2 : 1;
  p.n_rt = (int)((rows + 16 * rt - 1) / (16 * rt));
  const int64_t units = (int64_t)a->B * a->cache.heads * p.n_rt;
  // Keys split over a cluster until some four waves of CTAs exist, at least two tiles per CTA.
  const int64_t tiles = ((int64_t)a->W * a->cache.page_size + kv::small::kTile - 1) / kv::small::kTile;
  int cluster = 1;
  while (cluster < 16 && units * cluster < 4 * 148 * (rt == 1 ? 2 : 1) && tiles >= 4 * cluster) cluster *= 2;
  DEMON_CHECK_ARG(units * cluster < ((int64_t)1 << 31), "kv_attention: too many work units (%lld)", (long long)units);
  return rt == 1 ? launch_small<1>(p, units, cluster, (cudaStream_t)stream)
                 : launch_small<2>(p, units, cluster, (cudaStream_t)stream);
}
