// kv_attention_tc.cu -- attention over the paged E4M3 K/V cache for many query rows (prompts,
// chunks, the DiT's cross attention) on the 5th-generation tensor cores.
//
// The same function as the small kernel in kv_attention.cu (rows, masks, empty rows, NaN).  Work
// unit: one (sequence, kv head, block of 256 query rows), a row being (token, query head) with
// the G query heads of the kv head next to each other, so that any G fills the tiles.  The two
// halves of 128 rows share every K / V tile of 128 keys.  Persistent CTAs (one per SM), blocks
// with the most keys (the last of a causal prompt) first.
//
// Operands.  The codes go from their pages through registers into shared memory as f16, which
// holds every E4M3 value: one conversion instruction per two codes, so that the scales stay out
// of the tiles.  Q is f16 too, each row times a power of two (exact down to 2^-28 of the row's
// largest).  Score of row r, key j: t = S[r][j] * (row's power * page's K scale * softmax scale),
// in log2 units.  V's scale 2^ev joins the exponent of the probability: with M a running offset
// of max_j (t_j + ev_j),
//   P_j = 2^(t_j + ev_j - M + 6)   (f16; the largest value lies in [2^6, 2^14])
// is what each key's codes weigh in the row's output, whatever the pages' scales, and
//   l = sum_j 2^(t_j - m) = sum_groups 2^(M - m - ev_g - 6) sum_{j in g} P_j
// is summed in fp32 from the unrounded P_j with an offset m of its own (the running max of t_j).
// When some |M - m - ev_g| > 60 (V scales that differ by 2^60 within a call), P_j could underflow
// where 2^(t_j - m) does not; the tile's sum then takes a second exponential per key.
// Output: O * 2^(M - m - 6) / l.  Both offsets are raised only when exceeded by more than 8.
//
// Warp roles (512 threads; setmaxnreg as in attention.cu):
//   warpgroup 0 / 1   softmax of row half 0 / 1, one query row per thread,
//   warpgroup 2       Q (cp.async into its slot, converted in place) and the output rows,
//   warp 12           MMA issue (one thread) and tensor-memory allocation,
//   warps 13 - 15     K / V codes: loads of the next half tile stay in flight in registers while
//                     the ring slot is awaited, then convert, store swizzled, signal.
// Tensor memory as in attention.cu: S_h at 128 h, P_h over its upper half, O_h at 256 + 128 h.
//
// Bound by the exponentials (one per row and key, 16 per clock and SM) and the MMAs, which take
// as long; short key ranges (256 keys of a condition are two tiles) by the units' Q and output.
#include <algorithm>

#include "demon_host.h"
#include "kv_common.cuh"
#include "kv_host.h"

namespace demon {
namespace kv {
namespace tc {

constexpr int kBlk = 128;                // rows per half, keys per tile
constexpr int kRows = 2 * kBlk;          // rows per unit
constexpr int kBox = 128 * 128;          // 64 f16 columns x 128 rows (16 KB)
constexpr int kTile = 2 * kBox;          // 128 x 128 f16
constexpr int kSlots = 3;                // K / V ring
constexpr int kQSlots = 3;               // Q ring (one half of 128 rows each)
constexpr int kScSlots = 8;              // tiles whose scales are kept (see the ring comment)
constexpr int kNanSlots = 4;             // tiles whose NaN maps are kept
constexpr int kConvWarps = 3;
constexpr int kItems = 11;               // ceil(32 / kConvWarps) 16-byte loads per lane and half tile
constexpr int kThreads = 512;
constexpr float kBias = 6.0f;            // P = 2^(.. + 6)
constexpr float kRaise = 8.0f;           // offsets are raised when exceeded by more than this
constexpr float kFast = 60.0f;           // |M - m - ev| up to which l comes from P

constexpr int kLaunchRegs = 128, kSoftmaxRegs = 176, kQRegs = 80, kIssueRegs = 80;
static_assert(256 * kSoftmaxRegs + 128 * kQRegs + 128 * kIssueRegs <= kThreads * kLaunchRegs,
              "register split exceeds the launch's registers (setmaxnreg.inc would wait for good)");

// scales of a tile, per 16-key group: K scale, V exponent, 2^(ev_0 - ev_g); then the smallest and
// largest V exponent and the groups without a page
constexpr int kScWords = 32;
constexpr int scK = 0, scEv = 8, scInv = 16, scMin = 24, scMax = 25, scBad = 26;

constexpr int offQ = 0;
constexpr int offKV = offQ + kQSlots * kTile;
constexpr int offNan = offKV + kSlots * kTile;                 // [slot][128 keys] 128-bit maps
constexpr int offNanRow = offNan + kNanSlots * kBlk * 16;      // [2][128] 128-bit maps
constexpr int offL = offNanRow + 2 * kBlk * 16;                // [2][128] output factors
constexpr int offRow = offL + 2 * kBlk * 16;                   // [8][128] rows' powers of two
constexpr int offSc = offRow + 8 * kBlk * 4;
constexpr int offNanW = offSc + kScSlots * kScWords * 4;       // [slot][warp] any NaN
constexpr int offBar = offNanW + kScSlots * 4 * 4;
constexpr int kNumBars = 2 * kQSlots + 2 * kSlots + 14 + 1 + 2 * kScSlots + 8;
constexpr int offMisc = offBar + kNumBars * 8;
constexpr int kSmem = offMisc + 16 + 1024;
static_assert(kSmem <= 232448, "shared memory exceeds the sm_100 per-block limit");

constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColP = 64, kColO = 256;

// kind::f16, F16 x F16 -> F32, K-major A and B
constexpr uint32_t idesc_f16(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t tile, int kk) {
  return smem_desc(tile + (uint32_t)(kk >> 2) * kBox + (uint32_t)(kk & 3) * 32, 16, 1024, 2);
}
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t tile, int kk) {
  return smem_desc(tile + (uint32_t)kk * 2048, kBox, 1024, 2);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t t0,
                                          unsigned int* status, unsigned int where) {
  const bool ok = mbar_wait(bar, parity, abort, t0, status, where);
  return __all_sync(0xffffffffu, ok && *abort == 0);
}
template <int N>
__device__ __forceinline__ void setmaxnreg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void st_shared_u16(uint32_t a, uint32_t x) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((unsigned short)x) : "memory");
}
__device__ __forceinline__ void st_shared_b32(uint32_t a, uint32_t x) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(x) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_b32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

struct Unit {
  int b, hk, len, nq;
  int64_t row0;     // first row (token * G + head) of the block
  Keys ks;          // keys that some / every row of the block sees
  int tile0, nt;    // key tiles
};

// The j-th unit of this CTA: rounds go over the CTAs in turn, back and forth, since the units
// come in order of falling work.
__device__ __forceinline__ uint32_t unit_index(uint32_t j) {
  return j * gridDim.x + ((j & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}
__device__ __forceinline__ Unit decode(const AttnParams& p, uint32_t u, bool* bad) {
  Unit w;
  const uint32_t bh = (uint32_t)p.B * (uint32_t)p.c.heads;
  const uint32_t q = u / bh, r = u - q * bh;
  w.b = (int)(r / (uint32_t)p.c.heads);
  w.hk = (int)(r - (uint32_t)w.b * (uint32_t)p.c.heads);
  w.row0 = (int64_t)(p.n_rt - 1 - (int)q) * kRows;
  w.len = clamp_len(__ldg(p.lens + w.b), p.W * p.c.P, bad);
  w.nq = p.q_lens ? clamp_len(__ldg(p.q_lens + w.b), p.Sq, bad) : p.Sq;
  const int i0 = (int)((uint32_t)w.row0 / (uint32_t)p.G);
  const int i1 = imin((int)((uint32_t)(w.row0 + kRows - 1) / (uint32_t)p.G), w.nq - 1);
  w.ks.lo = w.ks.hi = w.ks.lo_all = w.ks.hi_all = 0;
  if (i0 <= i1) w.ks = visible(i0, i1, w.len, w.nq, p.causal != 0, p.window);
  w.tile0 = w.ks.lo / kBlk;
  w.nt = w.ks.hi > w.ks.lo ? (w.ks.hi + kBlk - 1) / kBlk - w.tile0 : 0;
  return w;
}
// Advances *j to the next unit with keys; false when there is none.
__device__ __forceinline__ bool next_unit(const AttnParams& p, uint32_t units, uint32_t* j, Unit* w) {
  bool bad = false;
  for (;; ++*j) {
    if ((uint64_t)*j * gridDim.x >= units) return false;
    const uint32_t u = unit_index(*j);
    if (u >= units) continue;
    *w = decode(p, u, &bad);
    if (w->nt > 0) {
      ++*j;
      return true;
    }
  }
}

template <int NG>  // 16-key-or-larger groups of a tile with a scale of their own: 128 / min(P, 128)
__global__ void __launch_bounds__(kThreads, 1) attention_tc_kernel(const AttnParams p, const uint32_t units, const int wide) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + offBar);
  uint64_t* q_full = bars;                      // [3] Q half converted
  uint64_t* q_empty = q_full + kQSlots;         // [3] its last S computed
  uint64_t* kv_full = q_empty + kQSlots;        // [3] K or V tile converted
  uint64_t* kv_empty = kv_full + kSlots;        // [3] its MMAs done
  uint64_t* s_full = kv_empty + kSlots;         // [2] S_h computed
  uint64_t* pa_full = s_full + 2;               // [2] P_h of keys 0-63 in tensor memory
  uint64_t* pb_full = s_full + 4;               // [2] P_h of keys 64-127
  uint64_t* o_full = s_full + 6;                // [2] the unit's last P V done
  uint64_t* o_empty = s_full + 8;               // [2] O_h read out
  uint64_t* l_full = s_full + 10;               // [2] output factors written
  uint64_t* l_empty = s_full + 12;              // [2] output factors read
  uint64_t* mma_done = s_full + 14;
  // The scales, NaN maps and row powers have rings longer than any lag between their writers and
  // readers: K tile t + 2 waits for the slot of a tile whose Q K^T was issued after the softmax of
  // tile t - 1 published its P, and Q of unit i + 4 for a Q slot of unit i + 2.
  uint64_t* sc_full = mma_done + 1;             // [8] scales of a tile
  uint64_t* nan_full = sc_full + kScSlots;      // [8] NaN map of a tile
  uint64_t* row_full = nan_full + kScSlots;     // [8] rows' powers of a Q half
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + offMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + offMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t t0 = globaltimer();

  if (threadIdx.x == 0) {
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(&q_full[s], 4);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&kv_full[s], kConvWarps);
      mbar_init(&kv_empty[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&s_full[h], 1);
      mbar_init(&pa_full[h], 4);
      mbar_init(&pb_full[h], 4);
      mbar_init(&o_full[h], 1);
      mbar_init(&o_empty[h], 4);
      mbar_init(&l_full[h], 4);
      mbar_init(&l_empty[h], 4);
    }
    mbar_init(mma_done, 1);
    for (int s = 0; s < kScSlots; ++s) {
      mbar_init(&sc_full[s], 1);
      mbar_init(&nan_full[s], kConvWarps);
      mbar_init(&row_full[s], 4);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_holder, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int wg = warp >> 2;

  if (wg == 3) {
    setmaxnreg_dec<kIssueRegs>();
    if (warp == 12) {
      // ------------------------------------------------------------------ MMA issue
      if (elect_one()) {
        const uint32_t idesc_qk = idesc_f16(kBlk, kBlk);
        const uint32_t idesc_pv = idesc_f16(kBlk, kHeadDim) | (1u << 16);  // B (V) MN-major
        uint32_t g = 0, it = 0, tiles = 0;  // half tiles consumed, units, key tiles (all units)
        bool ok = true;
        auto qk = [&](int h, uint32_t kslot) {
          const uint32_t qa = sbase + offQ + ((2 * it + h) % kQSlots) * kTile, kb = sbase + offKV + kslot * kTile;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_bf16(tmem + kColS + 128 * h, kmajor_desc(qa, kk), kmajor_desc(kb, kk), idesc_qk, kk > 0);
          tc_commit(&s_full[h]);
        };
        auto pv = [&](int h, uint32_t vslot, int half, bool acc) {
          const uint32_t vb = sbase + offKV + vslot * kTile;
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const int kk = 4 * half + k4;
            mma_bf16_ts(tmem + kColO + 128 * h, tmem + kColS + 128 * h + kColP + 8 * kk, mnmajor_desc(vb, kk), idesc_pv,
                        (acc || kk > 0) ? 1u : 0u);
          }
        };
        auto wait_on = [&](uint64_t* bar, uint32_t parity, unsigned int where) {
          ok = mbar_wait(bar, parity, abort_flag, t0, p.status, where);
          if (ok) tc_fence_after();
          return ok;
        };
        auto wait_kv = [&](uint32_t gi) { return wait_on(&kv_full[gi % kSlots], (gi / kSlots) & 1u, 71); };
        auto pv_tile = [&](int h, uint32_t vslot, uint32_t t, bool acc) {
          if (!wait_on(&pa_full[h], t & 1u, 72)) return false;
          pv(h, vslot, 0, acc);
          if (!wait_on(&pb_full[h], t & 1u, 73)) return false;
          pv(h, vslot, 1, true);
          return true;
        };
        auto wait_oe = [&](int h) { return wait_on(&o_empty[h], (it & 1u) ^ 1u, 74); };
        auto wait_q = [&](int h) { return wait_on(&q_full[(2 * it + h) % kQSlots], ((2 * it + h) / kQSlots) & 1u, 75); };
        auto free_q = [&](int h) { tc_commit(&q_empty[(2 * it + h) % kQSlots]); };
        // as in attention.cu: a unit's last P_1 V goes after the next unit's first S_0
        bool pend = false, pend_acc = false;
        uint32_t pend_v = 0, pend_t = 0;
        auto flush = [&]() {
          if (!pend) return true;
          if (!pv_tile(1, pend_v % kSlots, pend_t, pend_acc)) return false;
          tc_commit(&kv_empty[pend_v % kSlots]);
          tc_commit(&o_full[1]);
          pend = false;
          return true;
        };
        uint32_t j = 0;
        Unit w;
        while (ok && next_unit(p, units, &j, &w)) {
          const int n = w.nt;
          uint32_t gk = g, gv = g + 1;
          if (!wait_q(0) || !wait_kv(gk)) break;
          qk(0, gk % kSlots);
          if (n == 1) free_q(0);
          if (!flush() || !wait_q(1)) break;
          qk(1, gk % kSlots);
          tc_commit(&kv_empty[gk % kSlots]);
          if (n == 1) free_q(1);
          if (!wait_kv(gv) || !wait_oe(0) || !pv_tile(0, gv % kSlots, tiles, false)) break;
          uint32_t prev_v = gv;
          g += 2;
          for (int i = 1; i < n; ++i) {
            gk = g;
            gv = g + 1;
            if (!wait_kv(gk)) break;
            qk(0, gk % kSlots);
            if (i == n - 1) free_q(0);
            if (i == 1 && !wait_oe(1)) break;
            if (!pv_tile(1, prev_v % kSlots, tiles + i - 1, i - 1 > 0)) break;
            tc_commit(&kv_empty[prev_v % kSlots]);
            qk(1, gk % kSlots);
            tc_commit(&kv_empty[gk % kSlots]);
            if (i == n - 1) free_q(1);
            if (!wait_kv(gv) || !pv_tile(0, gv % kSlots, tiles + i, true)) break;
            prev_v = gv;
            g += 2;
          }
          if (!ok) break;
          tc_commit(&o_full[0]);
          if (n == 1 && !wait_oe(1)) break;  // this unit's only P_1 V overwrites O_1
          pend = true;
          pend_v = prev_v;
          pend_t = tiles + n - 1;
          pend_acc = n > 1;
          tiles += n;
          ++it;
        }
        if (ok) flush();
        tc_commit(mma_done);
      }
      __syncwarp();
      {
        volatile int never = 0;
        mbar_wait(mma_done, 0, &never, globaltimer(), p.status, 76);
      }
      __syncwarp();
    } else {
      // ------------------------------------------------------------------ K / V codes
      const int cw = warp - 13, c = lane & 3, rl = lane >> 2;
      uint4 r[kItems];
      uint32_t g = 0, tiles = 0, j = 0;
      Unit w, nw;         // the unit being converted, the one of the next tile
      int tile = 0;       // key tile of w within its range
      int pid = -1;       // lanes 0 .. 7: page of their 16 keys of the current tile, -1: none seen
      int npid = -1;      // and of the next tile
      float sk = 0.0f, sv = 0.0f, nsk = 0.0f, nsv = 0.0f;
      bool absent = false, nabsent = false;  // a seen group without a page
      auto look_up = [&](const Unit& u, int t, int& pg, float& k, float& v, bool& gone) {
        pg = -1;
        k = v = 0.0f;
        gone = false;
        const int key = (u.tile0 + t) * kBlk + 16 * lane, gw = kBlk / NG;
        const int gk = key & ~(gw - 1);  // first key of the group that has one scale
        if (lane < 8 && gk < u.ks.hi && gk + gw > u.ks.lo) {
          pg = page_id(p.table + u.b * p.ld_table, p.W, key / p.c.P, p.c.pages);
          if (pg >= 0) {
            k = __ldg(p.c.scale[0] + (int64_t)pg * p.c.heads + u.hk);
            v = __ldg(p.c.scale[1] + (int64_t)pg * p.c.heads + u.hk);
          } else {
            gone = true;
            if (cw == 0) report(p.status, DEMON_DEV_BAD_ARG, 64);
          }
        }
      };
      // item n = cw + 3 i: rows 8 (n / 2) .. + 7 of the tile, 64-code half n % 2
      auto load = [&](const Unit& u, int t, int pg, int kv) {
        const int k0 = (u.tile0 + t) * kBlk;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          const int n = cw + kConvWarps * i;
          r[i] = make_uint4(0, 0, 0, 0);
          const int pgi = __shfl_sync(0xffffffffu, pg, (n >> 2) & 7);
          if (n < 32 && pgi >= 0) {
            const int key = k0 + 8 * (n >> 1) + rl;
            const int64_t at = (((int64_t)pgi * p.c.heads + u.hk) * p.c.P + (key & (p.c.P - 1))) * kHeadDim + 64 * (n & 1) + 16 * c;
            r[i] = __ldg(reinterpret_cast<const uint4*>(p.c.codes[kv] + at));
          }
        }
      };
      auto store = [&](uint32_t dst, int i, int n) {
        const int row = 8 * (n >> 1) + rl;
        uint32_t x[8];
        e4m3x4_f16(r[i].x, x[0], x[1]);
        e4m3x4_f16(r[i].y, x[2], x[3]);
        e4m3x4_f16(r[i].z, x[4], x[5]);
        e4m3x4_f16(r[i].w, x[6], x[7]);
        const uint32_t a = dst + (n & 1) * kBox + row * 128;
        st_shared_v4(a + (((2 * c) ^ rl) << 4), x[0], x[1], x[2], x[3]);
        st_shared_v4(a + (((2 * c + 1) ^ rl) << 4), x[4], x[5], x[6], x[7]);
      };
      bool have = next_unit(p, units, &j, &w);
      if (have) {
        look_up(w, 0, pid, sk, sv, absent);
        load(w, 0, pid, 0);
      }
      bool ok = true;
      while (have && ok) {
        // the tile after this one
        bool more = true;
        int ntile = tile + 1;
        if (ntile < w.nt) {
          nw = w;
        } else {
          more = next_unit(p, units, &j, &nw);
          ntile = 0;
        }
        if (more) look_up(nw, ntile, npid, nsk, nsv, nabsent);
        // K
        if (!(ok = warp_wait(&kv_empty[g % kSlots], ((g / kSlots) & 1u) ^ 1u, abort_flag, t0, p.status, 77))) break;
        uint32_t dst = sbase + offKV + (g % kSlots) * kTile;
#pragma unroll
        for (int i = 0; i < kItems; ++i)
          if (cw + kConvWarps * i < 32) store(dst, i, cw + kConvWarps * i);
        if (cw == 0) {
          const uint32_t sc = sbase + offSc + (tiles % kScSlots) * kScWords * 4;
          const uint32_t held = __ballot_sync(0xffffffffu, lane < 8 && pid >= 0);
          const uint32_t gone = __ballot_sync(0xffffffffu, absent);
          // groups without a page take another group's V exponent: they weigh nothing
          const int any = held ? __ffs(held) - 1 : 0;
          int ev = scale_exp(sv);
          const int ev_any = __shfl_sync(0xffffffffu, ev, any);
          if (pid < 0) ev = ev_any;
          const int ev0 = __shfl_sync(0xffffffffu, ev, 0);
          if (lane >= 8) ev = ev0;
          const int lo = __reduce_min_sync(0xffffffffu, ev), hi = __reduce_max_sync(0xffffffffu, ev);
          if (lane < 8) {
            st_shared_f32(sc + 4 * (scK + lane), fabsf(sk));
            st_shared_f32(sc + 4 * (scEv + lane), (float)ev);
            st_shared_f32(sc + 4 * (scInv + lane), exp2i(imin(imax(ev0 - ev, -126), 126)));
          }
          if (lane == 0) {
            st_shared_f32(sc + 4 * scMin, (float)lo);
            st_shared_f32(sc + 4 * scMax, (float)hi);
            st_shared_b32(sc + 4 * scBad, gone);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&kv_full[g % kSlots]);
          if (cw == 0) mbar_arrive(&sc_full[tiles % kScSlots]);
        }
        ++g;
        load(w, tile, pid, 1);
        // V
        if (!(ok = warp_wait(&kv_empty[g % kSlots], ((g / kSlots) & 1u) ^ 1u, abort_flag, t0, p.status, 78))) break;
        dst = sbase + offKV + (g % kSlots) * kTile;
        const int k0 = (w.tile0 + tile) * kBlk;
        if (k0 < w.ks.lo_all || k0 + kBlk > w.ks.hi_all) {
          // Some row does not see some key: NaN codes go into a map instead of the product.  (Where
          // every row sees every key they may run through it.)
          uint32_t any = 0;
          const uint32_t map = sbase + offNan + (tiles % kNanSlots) * kBlk * 16;
#pragma unroll
          for (int i = 0; i < kItems; ++i) {
            const int n = cw + kConvWarps * i;
            if (n >= 32) continue;
            uint32_t y[4] = {nan_bytes(r[i].x) >> 7, nan_bytes(r[i].y) >> 7, nan_bytes(r[i].z) >> 7, nan_bytes(r[i].w) >> 7};
            r[i].x &= ~(y[0] * 255u);
            r[i].y &= ~(y[1] * 255u);
            r[i].z &= ~(y[2] * 255u);
            r[i].w &= ~(y[3] * 255u);
            uint32_t bits = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) bits |= ((y[q] | (y[q] >> 7) | (y[q] >> 14) | (y[q] >> 21)) & 15u) << (4 * q);
            any |= bits;
            st_shared_u16(map + (8 * (n >> 1) + rl) * 16 + ((n & 1) * 4 + c) * 2, bits);
          }
          any = __reduce_or_sync(0xffffffffu, any);
          if (lane == 0) st_shared_b32(sbase + offNanW + ((tiles % kScSlots) * 4 + cw) * 4, any);
        }
#pragma unroll
        for (int i = 0; i < kItems; ++i)
          if (cw + kConvWarps * i < 32) store(dst, i, cw + kConvWarps * i);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&kv_full[g % kSlots]);
          mbar_arrive(&nan_full[tiles % kScSlots]);
        }
        ++g;
        ++tiles;
        have = more;
        if (more) {
          w = nw;
          tile = ntile;
          pid = npid;
          sk = nsk;
          sv = nsv;
          absent = nabsent;
          load(w, tile, pid, 0);
        }
      }
    }
  } else if (wg < 2) {
    setmaxnreg_inc<kSoftmaxRegs>();
    // -------------------------------------------------------------------- softmax
    constexpr int GW = kBlk / NG, CH = 8 / NG;  // columns and maximum chains per group
    constexpr int SG = 8 / NG;                  // 16-key scale entries per group
    const int h = wg, quad = warp & 3, rr = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + kColS + 128 * h;
    const uint32_t o_addr = tmem + lane_addr + kColO + 128 * h;
    uint32_t t = 0, it = 0, j = 0;
    Unit w;
    while (next_unit(p, units, &j, &w)) {
      const int64_t row = w.row0 + h * kBlk + rr;
      const int qi = (int)((uint32_t)row / (uint32_t)p.G);
      const bool live = row < (int64_t)p.Sq * p.G && qi < w.nq;
      int jlo = 0, jhi = w.len;  // keys that this row sees: [jlo, jhi)
      if (live) {
        const Keys k = visible(qi, qi, w.len, w.nq, p.causal != 0, p.window);
        jlo = k.lo;
        jhi = k.hi;
      }
      bool ok = warp_wait(&row_full[(2 * it + h) % 8], ((2 * it + h) / 8) & 1u, abort_flag, t0, p.status, 80);
      if (!ok) break;
      const float fr = ld_shared_f32(sbase + offRow + (((2 * it + h) % 8) * kBlk + rr) * 4);
      float M = -INFINITY, m = -INFINITY, l = 0.0f;
      bool nan_row = false;
      for (int i = 0; i < w.nt; ++i, ++t) {
        if (!(ok = warp_wait(&s_full[h], t & 1u, abort_flag, t0, p.status, 81))) break;
        tc_fence_after();
        if (!(ok = warp_wait(&sc_full[t % kScSlots], (t / kScSlots) & 1u, abort_flag, t0, p.status, 82))) break;
        uint32_t sr[128];
        tmem_ld_32x32b_x32(s_addr + 0, *reinterpret_cast<uint32_t(*)[32]>(sr + 0));
        tmem_ld_32x32b_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(sr + 32));
        tmem_ld_32x32b_x32(s_addr + 64, *reinterpret_cast<uint32_t(*)[32]>(sr + 64));
        tmem_ld_32x32b_x32(s_addr + 96, *reinterpret_cast<uint32_t(*)[32]>(sr + 96));
        tmem_ld_wait();
        float* s = reinterpret_cast<float*>(sr);
        const uint32_t sc = sbase + offSc + (t % kScSlots) * kScWords * 4;
        const int k0 = (w.tile0 + i) * kBlk;
        const int lo = jlo - k0, hi = jhi - 1 - k0;
        if (__any_sync(0xffffffffu, lo > 0)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c < lo ? -INFINITY : s[c];
        }
        if (__any_sync(0xffffffffu, hi < kBlk - 1)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c > hi ? -INFINITY : s[c];
        }
        const uint32_t gone = ld_shared_b32(sc + 4 * scBad);
        if (gone) {  // pages that do not exist: seen by no row
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = (gone >> (c >> 4)) & 1u ? -INFINITY : s[c];
        }
        // maxima per group, in score units and with V's exponent
        float mt = -INFINITY, Mt = -INFINITY;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          float mc[CH];
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            mc[c] = fmaxf(s[gi * GW + c], s[gi * GW + c + CH]);
#pragma unroll
            for (int q = 2; q < 16; q += 2) mc[c] = max3(mc[c], s[gi * GW + c + CH * q], s[gi * GW + c + CH * (q + 1)]);
          }
          float gm = mc[0];
#pragma unroll
          for (int c = 1; c < CH; ++c) gm = fmaxf(gm, mc[c]);
          // kept within 2^+-120: a masked score times 0 would be NaN
          const float f = fminf(fmaxf(fr * ld_shared_f32(sc + 4 * (scK + gi * SG)) * p.scale_log2, 7.5e-37f), 1.3e36f);
          const float x = gm * f;
          mt = fmaxf(mt, x);
          Mt = fmaxf(Mt, x + ld_shared_f32(sc + 4 * (scEv + gi * SG)));
        }
        if (mt > m + kRaise || (m == -INFINITY && mt > -INFINITY)) {
          l *= ex2(m - mt);
          m = mt;
        }
        float factor = 1.0f;
        bool rescale = false;
        if (Mt > M + kRaise || (M == -INFINITY && Mt > -INFINITY)) {
          factor = ex2(M - Mt);
          rescale = i > 0;
          M = Mt;
        }
        const float mo = M == -INFINITY ? 0.0f : M, ml = m == -INFINITY ? 0.0f : m;
        const float D = mo - ml;
        const bool far = D - ld_shared_f32(sc + 4 * scMin) > kFast || ld_shared_f32(sc + 4 * scMax) - D > kFast;
        float lw = ex2(D - kBias - ld_shared_f32(sc + 4 * scEv));  // weight of group 0's sum in l
        if (__any_sync(0xffffffffu, far)) {
#pragma unroll
          for (int c = 0; c < 128; ++c) {
            const float f = fminf(fmaxf(fr * ld_shared_f32(sc + 4 * (scK + (c / GW) * SG)) * p.scale_log2, 7.5e-37f), 1.3e36f);
            l += ex2(fmaf(s[c], f, -ml));
          }
          lw = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c == 2) {
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
              for (int oc = 0; oc < 4; ++oc) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(o_addr + 32 * oc, o);
                tmem_ld_wait();
#pragma unroll
                for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * factor);
                tmem_st_32x32b_x32(o_addr + 32 * oc, o);
              }
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pa_full[h]);
          }
          uint32_t pk[16];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int gi = (32 * c + 16 * half) / GW;
            const float f = fminf(fmaxf(fr * ld_shared_f32(sc + 4 * (scK + gi * SG)) * p.scale_log2, 7.5e-37f), 1.3e36f);
            const float n = ld_shared_f32(sc + 4 * (scEv + gi * SG)) - mo + kBias;
            const float2 f2 = make_float2(f, f), n2 = make_float2(n, n);
            float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int at = 32 * c + 16 * half + 2 * q;
              const float2 x = fma_f2(make_float2(s[at], s[at + 1]), f2, n2);
              const float2 e = make_float2(ex2(x.x), ex2(x.y));
              acc = add_f2(acc, e);
              pk[8 * half + q] = pack_f16x2(e.x, e.y);
            }
            l = fmaf(lw * ld_shared_f32(sc + 4 * (scInv + gi * SG)), acc.x + acc.y, l);
          }
          tmem_st_32x32b_x16(s_addr + kColP + 16 * c, pk);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pb_full[h]);
        if (k0 < w.ks.lo_all || k0 + kBlk > w.ks.hi_all) {  // the converters left NaN codes of V out
          if (!(ok = warp_wait(&nan_full[t % kScSlots], (t / kScSlots) & 1u, abort_flag, t0, p.status, 83))) break;
          const uint32_t nw = sbase + offNanW + (t % kScSlots) * 16;
          if (ld_shared_b32(nw) | ld_shared_b32(nw + 4) | ld_shared_b32(nw + 8)) {
            uint4 seen = make_uint4(0, 0, 0, 0);
            const uint32_t map = sbase + offNan + (t % kNanSlots) * kBlk * 16;
            for (int c = imax(lo, 0); c <= imin(hi, kBlk - 1); ++c) {
              const uint4 x = ld_shared_v4(map + c * 16);
              seen.x |= x.x;
              seen.y |= x.y;
              seen.z |= x.z;
              seen.w |= x.w;
            }
            // the row's map is handed over with its output factors: the last unit's must be read
            if (!(ok = warp_wait(&l_empty[h], (it & 1u) ^ 1u, abort_flag, t0, p.status, 84))) break;
            const uint32_t a = sbase + offNanRow + (h * kBlk + rr) * 16;
            if (nan_row) {
              const uint4 x = ld_shared_v4(a);
              seen.x |= x.x;
              seen.y |= x.y;
              seen.z |= x.z;
              seen.w |= x.w;
            }
            st_shared_v4(a, seen.x, seen.y, seen.z, seen.w);
            nan_row = true;
          }
        }
      }
      if (!ok) break;
      if (!warp_wait(&l_empty[h], (it & 1u) ^ 1u, abort_flag, t0, p.status, 85)) break;
      // output factor 2^(M - m - 6) / l, in two parts that both stay normal
      float fa = 0.0f, fb = 0.0f;
      if (live && l != 0.0f) {
        fa = ex2(0.5f * (M - m - kBias));
        fb = fa / l;
      }
      st_shared_f32x4(sbase + offL + (h * kBlk + rr) * 16, fa, fb, nan_row ? 1.0f : 0.0f, 0.0f);
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_full[h]);
      ++it;
    }
  } else {
    setmaxnreg_dec<kQRegs>();
    // -------------------------------------------------------------------- Q in, output rows out
    const int quad = warp & 3, rr = quad * 32 + lane, sub = lane & 15;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t n_rows = (uint32_t)p.Sq * (uint32_t)p.G;
    // rows quad * 32 + 2 k + (lane / 16) of half h: 16 bytes per lane
    auto q_load = [&](const Unit& w, uint32_t slot, int h) {
      uint32_t row = (uint32_t)w.row0 + h * kBlk + quad * 32 + (lane >> 4);
      int i = (int)(row / (uint32_t)p.G), g = (int)(row - (uint32_t)i * (uint32_t)p.G);
      const __nv_bfloat16* q = p.q + w.b * p.q_seq + (int64_t)(w.hk * p.G) * p.q_head + sub * 8;
#pragma unroll 4
      for (int k = 0; k < 16; ++k) {
        const int rt = quad * 32 + 2 * k + (lane >> 4);
        const uint32_t dst = sbase + offQ + slot * kTile + (sub >> 3) * kBox + rt * 128 + (((sub & 7) ^ (rt & 7)) << 4);
        if (row < n_rows && i < w.nq)
          cp_async_16(dst, q + (int64_t)i * p.q_row + (int64_t)g * p.q_head);
        else
          st_shared_v4(dst, 0, 0, 0, 0);
        row += 2;
        g += 2;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (g >= p.G) {
            g -= p.G;
            ++i;
          }
      }
    };
    auto q_convert = [&](uint32_t qi, int h) {
      cp_async_wait_all();
      const uint32_t slot = qi % kQSlots;
#pragma unroll 4
      for (int k = 0; k < 16; ++k) {
        const int rt = quad * 32 + 2 * k + (lane >> 4);
        const uint32_t a = sbase + offQ + slot * kTile + (sub >> 3) * kBox + rt * 128 + (((sub & 7) ^ (rt & 7)) << 4);
        const uint4 x = ld_shared_v4(a);
        uint32_t mx = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
        mx = max(mx & 0xFFFFu, mx >> 16);
        if (mx >= 0x7F80u) mx = 0;  // infinities and NaN pass through at any power
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const int e = imax((int)(mx >> 7) - 127 - 13, -126);  // |q| 2^-e < 2^14
        const float2 mul = make_float2(exp2i(-e), exp2i(-e));
        const float2 f0 = mul_f2(bf2_f2(x.x), mul), f1 = mul_f2(bf2_f2(x.y), mul), f2 = mul_f2(bf2_f2(x.z), mul),
                     f3 = mul_f2(bf2_f2(x.w), mul);
        st_shared_v4(a, pack_f16x2(f0.x, f0.y), pack_f16x2(f1.x, f1.y), pack_f16x2(f2.x, f2.y), pack_f16x2(f3.x, f3.y));
        if (sub == 0) st_shared_f32(sbase + offRow + ((qi % 8) * kBlk + rt) * 4, exp2i(e));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&q_full[slot]);
        mbar_arrive(&row_full[qi % 8]);
      }
      (void)h;
    };
    auto wait_slot = [&](uint32_t qi) {
      return warp_wait(&q_empty[qi % kQSlots], ((qi / kQSlots) & 1u) ^ 1u, abort_flag, t0, p.status, 90);
    };
    auto out_row = [&](const Unit& w, int h, bool* inside) {
      const uint32_t row = (uint32_t)w.row0 + h * kBlk + rr;
      *inside = row < n_rows;
      const uint32_t i = row / (uint32_t)p.G, g = row - i * (uint32_t)p.G;
      return p.o + w.b * p.o_seq + (int64_t)i * p.o_row + (int64_t)(w.hk * p.G + (int)g) * p.o_head;
    };
    auto put = [&](__nv_bfloat16* o, const uint32_t (&x)[16]) {  // 32 columns
      if (wide) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o + 16 * q), "r"(x[8 * q]),
                       "r"(x[8 * q + 1]), "r"(x[8 * q + 2]), "r"(x[8 * q + 3]), "r"(x[8 * q + 4]), "r"(x[8 * q + 5]),
                       "r"(x[8 * q + 6]), "r"(x[8 * q + 7])
                       : "memory");
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) st_global_v4(o + 8 * q, make_uint4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]));
      }
    };
    // this CTA's next unit; rows of units without keys are zeroed on the way
    uint32_t j = 0;
    auto advance = [&](Unit* w) {
      for (;; ++j) {
        if ((uint64_t)j * gridDim.x >= units) return false;
        const uint32_t u = unit_index(j);
        if (u >= units) continue;
        bool bad = false;
        *w = decode(p, u, &bad);
        if (bad && w->hk == 0 && w->row0 == 0 && threadIdx.x == 256) report(p.status, DEMON_DEV_BAD_ARG, 63);
        if (w->nt > 0) {
          ++j;
          return true;
        }
        const uint32_t zero[16] = {};
        for (int h = 0; h < 2; ++h) {
          bool inside;
          __nv_bfloat16* o = out_row(*w, h, &inside);
          if (inside)
            for (int c = 0; c < 4; ++c) put(o + 32 * c, zero);
        }
      }
    };
    auto epilogue = [&](const Unit& w, uint32_t it, int h) {
      if (!warp_wait(&l_full[h], it & 1u, abort_flag, t0, p.status, 91)) return false;
      const float4 f = ld_shared_f32x4(sbase + offL + (h * kBlk + rr) * 16);
      uint4 nan = make_uint4(0, 0, 0, 0);
      if (f.z != 0.0f) nan = ld_shared_v4(sbase + offNanRow + (h * kBlk + rr) * 16);
      __syncwarp();
      if (lane == 0) mbar_arrive(&l_empty[h]);
      bool inside;
      __nv_bfloat16* out = out_row(w, h, &inside);
      if (!warp_wait(&o_full[h], it & 1u, abort_flag, t0, p.status, 92)) return false;
      tc_fence_after();
      const float2 fa = make_float2(f.x, f.x), fb = make_float2(f.y, f.y);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(tmem + lane_addr + kColO + 128 * h + 32 * c, o);
        tmem_ld_wait();
        if (c == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_empty[h]);
        }
        if (f.z != 0.0f) {
          const uint32_t bits = c == 0 ? nan.x : c == 1 ? nan.y : c == 2 ? nan.z : nan.w;
#pragma unroll
          for (int q = 0; q < 32; ++q)
            if ((bits >> q) & 1u) o[q] = 0x7FFFFFFFu;
        }
        uint32_t x[16];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float2 v = mul_f2(mul_f2(make_float2(__uint_as_float(o[2 * q]), __uint_as_float(o[2 * q + 1])), fa), fb);
          x[q] = f.y == 0.0f ? 0u : pack_bf16x2(v.x, v.y);  // rows that see nothing: zeros, never 0 * NaN
        }
        if (inside) put(out + 32 * c, x);
      }
      return true;
    };

    Unit w, nw;
    uint32_t it = 0;
    bool have = advance(&w);
    if (have) {
      q_load(w, 0, 0);
      q_load(w, 1, 1);
      q_convert(0, 0);
      q_convert(1, 1);
    }
    while (have) {
      const bool more = advance(&nw);
      const uint32_t n0 = 2 * it + 2, n1 = 2 * it + 3;
      if (more) {
        if (!wait_slot(n0)) break;
        q_load(nw, n0 % kQSlots, 0);
        q_convert(n0, 0);
        if (!wait_slot(n1)) break;
        q_load(nw, n1 % kQSlots, 1);
      }
      if (!epilogue(w, it, 0)) break;
      if (more) q_convert(n1, 1);
      if (!epilogue(w, it, 1)) break;
      w = nw;
      have = more;
      ++it;
    }
    cp_async_wait_all();  // no copy in flight when the CTA leaves
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, kTmemCols);
}

std::atomic<uint64_t> g_attr{0};

template <int NG>
int prepare() {
  cudaFuncAttributes fa;
  DEMON_CUDA(cudaFuncGetAttributes(&fa, attention_tc_kernel<NG>));
  if (fa.numRegs != kLaunchRegs) {
    set_error("kv_attention: kernel built with %d registers per thread, the register split needs %d", fa.numRegs, kLaunchRegs);
    return DEMON_ERR_CUDA;
  }
  DEMON_CUDA(cudaFuncSetAttribute(attention_tc_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  return DEMON_OK;
}

}  // namespace tc

int attention_tc(AttnParams p, cudaStream_t st) {
  using namespace tc;
  const int64_t rows = (int64_t)p.Sq * p.G;
  p.n_rt = (int)((rows + kRows - 1) / kRows);
  const int64_t units = (int64_t)p.n_rt * p.B * p.c.heads;
  DEMON_CHECK_ARG(rows < ((int64_t)1 << 31) - kRows && units < ((int64_t)1 << 31), "kv_attention: too many query rows (%lld)",
                  (long long)rows);
  if (device_pending(g_attr)) {
    int rc = prepare<1>();
    if (rc == DEMON_OK) rc = prepare<2>();
    if (rc == DEMON_OK) rc = prepare<4>();
    if (rc == DEMON_OK) rc = prepare<8>();
    if (rc != DEMON_OK) return rc;
    mark_device_done(g_attr);
  }
  int dev = 0, sms = 148;
  DEMON_CUDA(cudaGetDevice(&dev));
  DEMON_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const unsigned grid = (unsigned)std::min<int64_t>(units, sms);
  const int wide = ((uintptr_t)p.o & 31) == 0 && p.o_seq % 16 == 0 && p.o_row % 16 == 0 && p.o_head % 16 == 0;
  switch (p.c.P) {
    case 16: attention_tc_kernel<8><<<grid, kThreads, kSmem, st>>>(p, (uint32_t)units, wide); break;
    case 32: attention_tc_kernel<4><<<grid, kThreads, kSmem, st>>>(p, (uint32_t)units, wide); break;
    case 64: attention_tc_kernel<2><<<grid, kThreads, kSmem, st>>>(p, (uint32_t)units, wide); break;
    default: attention_tc_kernel<1><<<grid, kThreads, kSmem, st>>>(p, (uint32_t)units, wide); break;
  }
  DEMON_CUDA(cudaGetLastError());
  return DEMON_OK;
}

}  // namespace kv
}  // namespace demon
