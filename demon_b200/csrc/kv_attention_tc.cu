// kv_attention_tc.cu -- attention over the paged E4M3 K/V cache for many query rows (prompts,
// chunks, the DiT's cross attention) on the 5th-generation tensor cores.
//
// The same function as the small kernel in kv_attention.cu (rows, masks, empty rows, NaN).  Work
// unit: one (sequence, kv head, block of 2 Tt query tokens), Tt = floor(128 / G): each half of the
// block is Tt tokens times the G query heads of the kv head, up to 128 rows of a tile.  The two
// halves share every K / V tile of 128 keys.  Few blocks over long keys: a block's keys are several
// units, whose partial results the join kernel of kv_attention.cu puts together.  Persistent CTAs (one
// per SM), blocks with the most keys (the last of a causal prompt) first.
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
// Warp roles (512 threads):
//   warpgroup 0 / 1   row half 0 / 1, one query row per thread: its Q row in place (before the last
//                     unit's output, so that Q K^T runs meanwhile), the softmax of every key tile, the
//                     output row,
//   warpgroup 2       codes -> f16, swizzled, into a ring of three K / V tiles,
//   warp 12           MMA issue (one thread) and tensor-memory allocation,
//   warp 13           page look-ups, scales, bulk copies of K / V codes into a ring of half tiles,
//   warp 14           the next unit's Q by TMA, each half as soon as the last Q K^T has read the slot,
//   warp 15           the list of units: lengths and masks into a ring of records that every role reads.
// Tensor memory as in attention.cu: S_h at 128 h, P_h over its upper half, O_h at 256 + 128 h.
//
// Bound by the softmax warps' path from S to P (2,830 clocks per tile and half, of which the
// exponentials' rate asks for 1,024) and, for short key ranges (256 keys of a condition are two
// tiles), by the units' Q conversion and output (Q converted by warpgroup 2 after the unit's first
// tile: 69 us for 16 x 750 over 256 keys against 64).  Measured, 16 query heads over 8: 6,016 x 6,016
// 333 us (0.89 PFLOP/s; the bf16 kernel of attention.cu 267 us), 16 x 750 over 256 keys 64.5 us (bf16
// 34.5 us), 6,001 causal 180 us.  Slower, not kept: steps of 64 keys with two score
// buffers (Q K^T 64 wide takes the tensor core longer, and the overheads of a step double: 396 us at
// 6,016 x 6,016); two threads per row (466 us); the next scores loaded ahead of the exponentials
// (509 us, they come late).
#include <algorithm>

#include "demon_host.h"
#include "kv_common.cuh"
#include "kv_host.h"

namespace demon {
namespace kv {
namespace tc {

constexpr int kBlk = 128;                // rows per half, keys per tile
constexpr int kBox = 128 * 128;          // 64 f16 columns x 128 rows (16 KB)
constexpr int kTile = 2 * kBox;          // 128 x 128 f16
constexpr int kSlots = 3;                // K / V tiles as f16
constexpr int kRawSlots = 3;             // ring of half tiles (K or V) as codes
constexpr int kRaw = kBlk * kHeadDim;    // 16 KB
constexpr int kScSlots = 8;              // tiles whose scales are kept (see the ring comment)
constexpr int kNanSlots = 4;             // tiles whose NaN maps are kept
constexpr int kConvWarps = 4;
constexpr int kUnitSlots = 4;            // unit records in flight
constexpr int kUnitReaders = 8 + kConvWarps + 3;  // warps that read each record
constexpr int kThreads = 512;
constexpr float kBias = 6.0f;            // P = 2^(.. + 6)
constexpr float kRaise = 8.0f;           // offsets are raised when exceeded by more than this
constexpr float kFast = 60.0f;           // |M - m - ev| up to which l comes from P

// Registers per thread after the split (setmaxnreg): the launch gives 512 x 128.  6,016 x 6,016 keys
// 334 us; 176 / 80 / 80 341 us, 184 / 72 / 72 339, 160 / 96 / 96 372, 168 / 96 / 80 354.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 168, kConvRegs = 88, kIssueRegs = 88;
static_assert(256 * kSoftmaxRegs + 128 * kConvRegs + 128 * kIssueRegs <= kThreads * kLaunchRegs,
              "register split exceeds the launch's registers (setmaxnreg.inc would wait for good)");

// Scales of a tile: per 16 keys {K scale, V exponent ev, 2^(ev_0 - ev), 0}, and {., -inf, ., -inf}
// for keys without a page, which so weigh nothing; then {smallest ev, largest ev, ev_0, 0}.
constexpr int kScWords = 36;
constexpr int kScTail = 32;

constexpr int offQ = 0;                                        // [2 halves]
constexpr int offKV = offQ + 2 * kTile;
constexpr int offRaw = offKV + kSlots * kTile;
constexpr int offNan = offRaw + kRawSlots * kRaw;              // [slot][128 keys] 128-bit maps
constexpr int offNanRow = offNan + kNanSlots * kBlk * 16;      // [2][128] 128-bit maps
constexpr int offSc = offNanRow + 2 * kBlk * 16;
constexpr int offNanW = offSc + kScSlots * kScWords * 4;       // [slot][warp] any NaN
constexpr int offUnit = offNanW + kScSlots * 4 * 4;            // [slot] 12 words
constexpr int offRawMask = offUnit + kUnitSlots * 48;          // [slot] 16-key groups copied
constexpr int offBar = offRawMask + 4 * 4;
constexpr int kNumBars = 4 + 2 * kSlots + 8 + 1 + 2 * kScSlots + 2 * kRawSlots + 2 + 2 * kUnitSlots;
constexpr int offMisc = offBar + kNumBars * 8;
constexpr int kSmem = offMisc + 16 + 1024;
static_assert(kSmem <= 232448, "shared memory exceeds the sm_100 per-block limit");

constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColP = 64, kColO = 256;  // P over the upper half of S

// kind::f16, F16 x F16 -> F32, K-major A and B
constexpr uint32_t idesc_f16(int M, int N) {
  return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Shared-memory descriptors of 128-byte-swizzled tiles (see attention.cu): the low word holds the
// address (>> 4) and the leading byte offset, the high word the stride and layout, so a k-step is an
// addition to the low word.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride 1024 B, version 1, swizzle 128 B
__device__ __forceinline__ uint32_t kmajor_lo(uint32_t tile) { return (tile >> 4) | ((16u >> 4) << 16); }
__device__ __forceinline__ uint32_t mnmajor_lo(uint32_t tile) { return (tile >> 4) | ((uint32_t)(kBox >> 4) << 16); }
__host__ __device__ constexpr uint32_t kmajor_step(int kk) { return (uint32_t)((kk >> 2) * kBox + (kk & 3) * 32) >> 4; }
__host__ __device__ constexpr uint32_t mnmajor_step(int kk) { return (uint32_t)(kk * 2048) >> 4; }
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) { return (uint64_t)lo | ((uint64_t)kDescHi << 32); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A warp-uniform bounded wait.  Most find their phase complete, and the cost of a completed wait
// counts on the MMA warp's path (175 clocks each with the abort flag read every time: 439 us against
// 402 us for 16 heads over 6,016 queries and keys), so only a wait that goes on looks at the flag.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, const AttnParams& p,
                                          unsigned int where) {
  if (__all_sync(0xffffffffu, mbar_try_wait(smem_u32(bar), parity))) return true;
  return __all_sync(0xffffffffu, bounded_wait(bar, parity, abort, p, where));
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
// 4-D tiled load.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, uint64_t* bar, int32_t x, int32_t y, int32_t z,
                                            int32_t u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}

// 32 lanes x 16 consecutive 32-bit columns -> 16 registers per thread.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

struct Unit {
  int b, hk, len, nq;
  int i0;           // first token of the block
  Keys ks;          // keys that some / every row of the block sees
  int tile0, nt;    // key tiles; nt 0: no keys (warp 15 writes its zeros, no record), nt -1: no more units
  int part;         // of the parts that share the block's keys
};

// The j-th unit of this CTA: rounds go over the CTAs in turn, back and forth, since the units
// come in order of falling work.
__device__ __forceinline__ uint32_t unit_index(uint32_t j) {
  return j * gridDim.x + ((j & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}
__device__ __forceinline__ Unit decode(const AttnParams& p, uint32_t u, bool* bad) {
  Unit w;
  const uint32_t bh = (uint32_t)p.B * (uint32_t)p.c.heads, block = u / (uint32_t)p.parts;
  const uint32_t q = block / bh, r = block - q * bh;
  w.part = (int)(u - block * (uint32_t)p.parts);
  w.b = (int)(r / (uint32_t)p.c.heads);
  w.hk = (int)(r - (uint32_t)w.b * (uint32_t)p.c.heads);
  w.i0 = (p.n_rt - 1 - (int)q) * 2 * p.Tt;
  w.len = clamp_len(__ldg(p.lens + w.b), p.W * p.c.P, bad);
  w.nq = p.q_lens ? clamp_len(__ldg(p.q_lens + w.b), p.Sq, bad) : p.Sq;
  const int i1 = imin(w.i0 + 2 * p.Tt, w.nq) - 1;
  w.ks.lo = w.ks.hi = w.ks.lo_all = w.ks.hi_all = 0;
  if (w.i0 <= i1) w.ks = visible(w.i0, i1, w.len, w.nq, p.causal != 0, p.window);
  w.tile0 = w.ks.lo / kBlk;
  w.nt = w.ks.hi > w.ks.lo ? (w.ks.hi + kBlk - 1) / kBlk - w.tile0 : 0;
  if (p.parts > 1) {  // an even share of the tiles
    const int share = w.nt / p.parts, extra = w.nt - share * p.parts;
    w.tile0 += w.part * share + imin(w.part, extra);
    w.nt = share + (w.part < extra ? 1 : 0);
  }
  return w;
}
// A unit's record in shared memory.
__device__ __forceinline__ void put_unit(uint32_t a, const Unit& w) {
  st_shared_v4(a, w.b, w.hk, w.len, w.nq);
  st_shared_v4(a + 16, w.i0, w.ks.lo, w.ks.hi, w.ks.lo_all);
  st_shared_v4(a + 32, w.ks.hi_all, w.tile0, w.nt, w.part);
}
__device__ __forceinline__ Unit get_unit(uint32_t a) {
  const uint4 x = ld_shared_v4(a), y = ld_shared_v4(a + 16), z = ld_shared_v4(a + 32);
  Unit w;
  w.b = (int)x.x, w.hk = (int)x.y, w.len = (int)x.z, w.nq = (int)x.w;
  w.i0 = (int)y.x, w.ks.lo = (int)y.y, w.ks.hi = (int)y.z, w.ks.lo_all = (int)y.w;
  w.ks.hi_all = (int)z.x, w.tile0 = (int)z.y, w.nt = (int)z.z, w.part = (int)z.w;
  return w;
}

// NG: 16-key-or-larger groups of a tile with a scale of their own, 128 / min(P, 128).  Split: partial
// results to the workspace (a variant of its own: the branch costs the other 5 % in registers).
template <int NG, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1) attention_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const AttnParams p,
                                                                    const uint32_t units, const int wide) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + offBar);
  uint64_t* q_full = bars;                      // [2] Q half converted
  uint64_t* q_empty = q_full + 2;               // [2] the unit's last Q K^T done
  uint64_t* kv_full = q_empty + 2;              // [3] K or V tile converted
  uint64_t* kv_empty = kv_full + kSlots;        // [3] its MMAs done
  uint64_t* s_full = kv_empty + kSlots;         // [2] S_h computed
  uint64_t* pa_full = s_full + 2;               // [2] P_h of keys 0-63 in tensor memory
  uint64_t* pb_full = s_full + 4;               // [2] P_h of keys 64-127
  uint64_t* o_full = s_full + 6;                // [2] the unit's last P_h V done
  uint64_t* mma_done = s_full + 8;
  // The scales and NaN maps have rings longer than any lag between their writers and readers: V of
  // tile t takes the slot of K of tile t - 1, whose last Q K^T was issued after both softmax
  // warpgroups had published, and so were done with, tile t - 2; the codes of tile t are copied at
  // most two tiles before that.
  uint64_t* sc_full = mma_done + 1;             // [8] scales of a tile
  uint64_t* nan_full = sc_full + kScSlots;      // [8] NaN map of a tile
  uint64_t* raw_full = nan_full + kScSlots;     // [3] codes of a half tile copied
  uint64_t* raw_empty = raw_full + kRawSlots;   // [3] and converted
  uint64_t* q_raw = raw_empty + kRawSlots;      // [2] Q half copied
  uint64_t* unit_full = q_raw + 2;              // [4] unit record written
  uint64_t* unit_empty = unit_full + kUnitSlots;  // [4] and read by every role
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + offMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + offMisc + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&kv_full[s], kConvWarps);
      mbar_init(&kv_empty[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&q_full[h], 4);
      mbar_init(&q_empty[h], 1);
      mbar_init(&q_raw[h], 1);
      mbar_init(&s_full[h], 1);
      mbar_init(&pa_full[h], 4);
      mbar_init(&pb_full[h], 4);
      mbar_init(&o_full[h], 1);
    }
    mbar_init(mma_done, 1);
    for (int s = 0; s < kUnitSlots; ++s) {
      mbar_init(&unit_full[s], 1);
      mbar_init(&unit_empty[s], kUnitReaders);
    }
    for (int s = 0; s < kRawSlots; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], kConvWarps);
    }
    for (int s = 0; s < kScSlots; ++s) {
      mbar_init(&sc_full[s], 1);
      mbar_init(&nan_full[s], kConvWarps);
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
  // The next unit for this warp (*j counts records); false at the end.  Records are of units with keys
  // alone: warp 13 waits for the next unit's before it copies the last tile of its own, and the softmax
  // warps read on only after that tile, so a run of empty records longer than the ring would stop both.
  auto next_unit = [&](uint32_t* j, Unit* w) {
    const uint32_t s = *j % kUnitSlots;
    if (!warp_wait(&unit_full[s], (*j / kUnitSlots) & 1u, abort_flag, p, 70)) return false;
    *w = get_unit(sbase + offUnit + s * 48);
    __syncwarp();
    if (lane == 0) mbar_arrive(&unit_empty[s]);
    ++*j;
    return w->nt >= 0;
  };

  if (wg == 3) {
    setmaxnreg_dec<kIssueRegs>();
    if (warp == 12) {
      // ------------------------------------------------------------------ MMA issue (one thread)
      if (elect_one()) {
        const uint32_t idesc_qk = idesc_f16(kBlk, kBlk);
        const uint32_t idesc_pv = idesc_f16(kBlk, kHeadDim) | (1u << 16);  // B (V) MN-major
        uint32_t g = 0, it = 0, tiles = 0;  // half tiles, units, key tiles (all units)
        auto qk = [&](int h, uint32_t kslot) {
          const uint32_t qa = kmajor_lo(sbase + offQ + h * kTile), kb = kmajor_lo(sbase + offKV + kslot * kTile);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            mma_bf16(tmem + kColS + 128 * h, desc_of(qa + kmajor_step(kk)), desc_of(kb + kmajor_step(kk)), idesc_qk, kk > 0);
          tc_commit(&s_full[h]);
        };
        auto pv = [&](int h, uint32_t vslot, int half, bool acc) {
          const uint32_t vb = mnmajor_lo(sbase + offKV + vslot * kTile);
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) {
            const int kk = 4 * half + k4;
            mma_bf16_ts(tmem + kColO + 128 * h, tmem + kColS + 128 * h + kColP + 8 * kk, desc_of(vb + mnmajor_step(kk)),
                        idesc_pv, (acc || kk > 0) ? 1u : 0u);
          }
        };
        auto wait_on = [&](uint64_t* bar, uint32_t parity, unsigned int where) {
          const bool ok = bounded_wait(bar, parity, abort_flag, p, where);
          tc_fence_after();
          return ok;
        };
        // The key tiles of all units form one stream; per tile: S_0, the last tile's P_1 V, S_1, P_0 V
        // (one half's softmax runs while the other half's products do, across units too; P_1 V of a
        // unit's last tile before the next unit's Q: 66.8 us against 64 for 16 x 750 over 256 keys, the
        // halves then store their rows at the same time).  A unit's first P_h V may overwrite O_h: its
        // P_h comes from threads that have stored the last unit's rows.
        bool ok = true, pend = false, pend_acc = false, pend_last = false;
        uint32_t pend_v = 0;
        auto flush = [&]() {  // P_1 V of the last tile
          if (!pend) return true;
          if (!wait_on(&pa_full[1], (tiles - 1) & 1u, 72)) return false;
          pv(1, pend_v, 0, pend_acc);
          if (!wait_on(&pb_full[1], (tiles - 1) & 1u, 73)) return false;
          pv(1, pend_v, 1, true);
          tc_commit(&kv_empty[pend_v]);
          if (pend_last) tc_commit(&o_full[1]);
          pend = false;
          return true;
        };
        for (uint32_t j = 0; ok; ++j) {
          const uint32_t us = j % kUnitSlots;
          if (!wait_on(&unit_full[us], (j / kUnitSlots) & 1u, 70)) break;
          const int nt = (int)ld_shared_b32(sbase + offUnit + us * 48 + 40);
          mbar_arrive(&unit_empty[us]);
          if (nt < 0) {
            flush();
            break;
          }
          if (!(ok = wait_on(&q_full[0], it & 1u, 75) && wait_on(&kv_full[g % kSlots], (g / kSlots) & 1u, 71))) break;
#pragma unroll 1
          for (int i = 0; i < nt; ++i) {
            const uint32_t ks = g % kSlots, vs = (g + 1) % kSlots, vp = ((g + 1) / kSlots) & 1u;  // K has been waited for
            g += 2;
            const bool last = i == nt - 1;
            qk(0, ks);
            if (last) tc_commit(&q_empty[0]);
            if (!(ok = flush() && (i > 0 || wait_on(&q_full[1], it & 1u, 75)))) break;
            qk(1, ks);
            tc_commit(&kv_empty[ks]);
            if (last) tc_commit(&q_empty[1]);
            if (!(ok = wait_on(&kv_full[vs], vp, 71) && wait_on(&pa_full[0], tiles & 1u, 72))) break;
            pv(0, vs, 0, i > 0);
            // the next K before the last wait of this tile
            if (!last && !(ok = wait_on(&kv_full[g % kSlots], (g / kSlots) & 1u, 71))) break;
            if (!(ok = wait_on(&pb_full[0], tiles & 1u, 73))) break;
            pv(0, vs, 1, true);
            if (last) tc_commit(&o_full[0]);
            pend = true;
            pend_v = vs;
            pend_acc = i > 0;
            pend_last = last;
            ++tiles;
          }
          ++it;
        }
        tc_commit(mma_done);
      }
      __syncwarp();
      {
        volatile int never = 0;
        mbar_wait(mma_done, 0, &never, globaltimer(), p.status, 76);
      }
      __syncwarp();
    } else if (warp == 13) {
      // ------------------------------------------------------------------ pages, scales, copies
      uint32_t n = 0, tiles = 0, j = 0;  // half tiles, tiles
      Unit w;
      int tile = 0;
      int pid = -1;  // lanes 0 .. 7: page of their 16 keys of the tile, -1: none seen
      float sk = 0.0f, sv = 0.0f;
      bool absent = false;  // seen keys without a page
      constexpr int gw = kBlk / NG;  // keys that share a page within a tile
      auto look_up = [&](const Unit& u, int t, int& pg, float& k, float& v, bool& gone) {
        pg = -1;
        k = v = 0.0f;
        gone = false;
        const int key = (u.tile0 + t) * kBlk + 16 * lane, gk = key & ~(gw - 1);
        if (lane < 8 && gk < u.ks.hi && gk + gw > u.ks.lo) {
          pg = page_id(p.table + u.b * p.ld_table, p.W, key / p.c.P, p.c.pages);
          if (pg >= 0) {
            k = __ldg(p.c.scale[0] + (int64_t)pg * p.c.heads + u.hk);
            v = __ldg(p.c.scale[1] + (int64_t)pg * p.c.heads + u.hk);
          } else {
            gone = true;
            report(p.status, DEMON_DEV_BAD_ARG, 64);
          }
        }
      };
      bool ok = true, have = next_unit(&j, &w);
      if (have) look_up(w, 0, pid, sk, sv, absent);
      while (have && ok) {
        // the next tile's pages and scales are on their way while this one's copies wait for room
        Unit nw = w;
        bool more = true, nabsent = false;
        int ntile = tile + 1, npid = -1;
        float nsk = 0.0f, nsv = 0.0f;
        if (ntile >= w.nt) {
          more = next_unit(&j, &nw);
          ntile = 0;
        }
        if (more) look_up(nw, ntile, npid, nsk, nsv, nabsent);
        const uint32_t held = __ballot_sync(0xffffffffu, pid >= 0);
        const uint32_t sc = sbase + offSc + (tiles % kScSlots) * kScWords * 4;
        // keys without a page take another group's V exponent: they weigh nothing
        int ev = scale_exp(sv);
        const int ev_any = __shfl_sync(0xffffffffu, ev, held ? __ffs(held) - 1 : 0);
        if (pid < 0) ev = ev_any;
        const int ev0 = __shfl_sync(0xffffffffu, ev, 0);
        if (lane >= 8) ev = ev0;
        const int elo = __reduce_min_sync(0xffffffffu, ev), ehi = __reduce_max_sync(0xffffffffu, ev);
        if (lane < 8)
          st_shared_f32x4(sc + 16 * lane, fabsf(sk), absent ? -INFINITY : (float)ev, exp2i(imin(imax(ev0 - ev, -126), 126)),
                          absent ? -INFINITY : 0.0f);
        if (lane == 8) st_shared_f32x4(sc + 4 * kScTail, (float)elo, (float)ehi, (float)ev0, 0.0f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_full[tiles % kScSlots]);
        const bool copies = pid >= 0 && (16 * lane) % gw == 0;
        const uint32_t n_copies = __popc(__ballot_sync(0xffffffffu, copies));
        const int key = (w.tile0 + tile) * kBlk + 16 * lane;
        const int64_t src = (((int64_t)imax(pid, 0) * p.c.heads + w.hk) * p.c.P + (key & (p.c.P - 1))) * kHeadDim;
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t s = n % kRawSlots;
          if (!(ok = warp_wait(&raw_empty[s], ((n / kRawSlots) & 1u) ^ 1u, abort_flag, p, 77))) break;
          if (lane == 0) {
            st_shared_b32(sbase + offRawMask + s * 4, held);
            mbar_arrive_expect_tx(&raw_full[s], n_copies * gw * kHeadDim);
          }
          __syncwarp();
          if (copies) bulk_load(smem + offRaw + s * kRaw + lane * 16 * kHeadDim, p.c.codes[kv] + src, gw * kHeadDim, &raw_full[s]);
        }
        w = nw;
        tile = ntile;
        pid = npid;
        sk = nsk;
        sv = nsv;
        absent = nabsent;
        have = more;
        ++tiles;
      }
      // no copy may still be in flight when the CTA leaves (immediate on the normal path)
      volatile int never = 0;
      for (uint32_t i = n > (uint32_t)kRawSlots ? n - kRawSlots : 0; i < n; ++i)
        mbar_wait(&raw_full[i % kRawSlots], (i / kRawSlots) & 1u, &never, globaltimer(), p.status, 79);
      __syncwarp();
    } else if (warp == 14) {
      // ------------------------------------------------------------------ Q
      uint32_t j = 0, it = 0;
      uint32_t issued = 0;  // halves
      Unit w;
      bool ok = true;
      const int q_rows = p.Tt * p.G;
      const uint32_t bytes = (uint32_t)q_rows * kHeadDim * 2;
      // Rows behind the last whole token: no copy writes them.  Zeros, since what shared memory held could
      // vote for the softmax's second exponential, which rounds the sums of the warp's other rows
      // differently.  (Zeroed by all threads at the start: 6,016 x 6,016 keys 333 -> 347 us, by the softmax
      // warps 341: the compiler's choices in their loop.)
      for (int i = lane; i < (kBlk - q_rows) * 32; i += 32)
        st_shared_v4(sbase + offQ + ((i >> 4) & 1) * kTile + ((i >> 3) & 1) * kBox + (q_rows + (i >> 5)) * 128 + (i & 7) * 16, 0, 0, 0, 0);
      __syncwarp();
      for (; ok && next_unit(&j, &w); ++it)
        for (int h = 0; h < 2; ++h) {
          if (!(ok = warp_wait(&q_empty[h], (it & 1u) ^ 1u, abort_flag, p, 91))) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_raw[h], bytes);
            for (int box = 0; box < 2; ++box)
              tma_load_4d(sbase + offQ + h * kTile + box * kBox, &tmQ, &q_raw[h], 64 * box, w.hk * p.G, w.i0 + h * p.Tt, w.b);
          }
          __syncwarp();
          ++issued;
        }
      // no copy may still be in flight when the CTA leaves (immediate on the normal path)
      volatile int never = 0;
      for (uint32_t i = issued > 2 ? issued - 2 : 0; i < issued; ++i)
        mbar_wait(&q_raw[i & 1], (i >> 1) & 1u, &never, globaltimer(), p.status, 93);
      __syncwarp();
    } else {
      // ------------------------------------------------------------------ units
      // a unit without keys: its rows are zeros, or partial results that weigh nothing
      auto empty_unit = [&](const Unit& u) {
        const int rows = 2 * p.Tt * p.G;
        if constexpr (kSplit) {
          const int64_t block = ((int64_t)u.b * p.c.heads + u.hk) * p.n_rt + u.i0 / (2 * p.Tt);
          for (int r = lane; r < rows && u.i0 + r / p.G < p.Sq; r += 32)
            *reinterpret_cast<float4*>(p.ws + ((block * rows + r) * p.parts + u.part) * kPartFloats + kHeadDim) =
                make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        } else {
          for (int r = lane >> 4; r < rows; r += 2) {
            const int i = u.i0 + r / p.G;
            if (i >= p.Sq) break;
            st_global_v4(p.o + u.b * p.o_seq + (int64_t)i * p.o_row + (int64_t)(u.hk * p.G + r % p.G) * p.o_head + (lane & 15) * 8,
                         make_uint4(0, 0, 0, 0));
          }
        }
        __syncwarp();
      };
      for (uint32_t j = 0, n = 0;; ++j) {
        bool bad = false;
        Unit w;
        w.nt = -1;
        if ((uint64_t)j * gridDim.x < units) {
          const uint32_t u = unit_index(j);
          if (u >= units) continue;
          w = decode(p, u, &bad);
          if (bad && w.hk == 0 && w.i0 == 0 && lane == 0) report(p.status, DEMON_DEV_BAD_ARG, 63);
          if (w.nt == 0) {
            empty_unit(w);
            continue;
          }
        }
        const uint32_t s = n % kUnitSlots;
        if (!warp_wait(&unit_empty[s], ((n / kUnitSlots) & 1u) ^ 1u, abort_flag, p, 69)) break;
        if (lane == 0) {
          put_unit(sbase + offUnit + s * 48, w);
          mbar_arrive(&unit_full[s]);
        }
        __syncwarp();
        ++n;
        if (w.nt < 0) break;
      }
    }
  } else if (wg == 2) {
    setmaxnreg_dec<kConvRegs>();
    // -------------------------------------------------------------------- codes -> f16
    // Warp cw takes keys 32 cw .. 32 cw + 31: chunk i is 16 codes of row 8 (i / 2) + lane / 4, and
    // neighbouring rows take opposite halves of their 128 codes (no bank conflicts either way).
    const int cw = warp & 3, c = lane & 3, rl = lane >> 2;
    const uint32_t a0 = (uint32_t)rl * 128 + (((2 * c) ^ rl) << 4), a1 = (uint32_t)rl * 128 + (((2 * c + 1) ^ rl) << 4);
    uint32_t n = 0, tiles = 0, j = 0;
    bool ok = true;
    Unit w;
    while (ok && next_unit(&j, &w)) {
      for (int t = 0; ok && t < w.nt; ++t, ++tiles) {
        const int k0 = (w.tile0 + t) * kBlk;
        const bool whole = k0 >= w.ks.lo_all && k0 + kBlk <= w.ks.hi_all;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const uint32_t s = n % kRawSlots;
          if (!(ok = warp_wait(&raw_full[s], (n / kRawSlots) & 1u, abort_flag, p, 78))) break;
          const uint32_t held = (ld_shared_b32(sbase + offRawMask + s * 4) >> (2 * cw)) & 3u;
          const uint32_t src = sbase + offRaw + s * kRaw + (cw * 32 + rl) * kHeadDim + 16 * c;
          uint4 r[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) r[i] = ld_shared_v4(src + (i >> 1) * 8 * kHeadDim + 64 * ((i & 1) ^ (rl & 1)));
          if (held != 3u) {  // keys that were not copied: zeros
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!((held >> (i >> 2)) & 1u)) r[i] = make_uint4(0, 0, 0, 0);
          }
          if (!(ok = warp_wait(&kv_empty[n % kSlots], ((n / kSlots) & 1u) ^ 1u, abort_flag, p, 86))) break;
          if (kv && !whole) {
            // Some row does not see some key: NaN codes go into a map instead of the product.
            // (Where every row sees every key they may run through it.)
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) any |= nan_bytes(r[i].x) | nan_bytes(r[i].y) | nan_bytes(r[i].z) | nan_bytes(r[i].w);
            any = __reduce_or_sync(0xffffffffu, any);
            if (lane == 0) st_shared_b32(sbase + offNanW + ((tiles % kScSlots) * 4 + cw) * 4, any);
            const uint32_t map = sbase + offNan + ((tiles % kNanSlots) * kBlk + cw * 32 + rl) * 16;
            if (any) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                uint32_t y[4] = {r[i].x, r[i].y, r[i].z, r[i].w}, bits = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  const uint32_t x = nan_bytes(y[q]) >> 7;
                  y[q] &= ~(x * 255u);
                  bits |= ((x | (x >> 7) | (x >> 14) | (x >> 21)) & 15u) << (4 * q);
                }
                r[i] = make_uint4(y[0], y[1], y[2], y[3]);
                st_shared_u16(map + (i >> 1) * 8 * 16 + (((i & 1) ^ (rl & 1)) * 4 + c) * 2, bits);
              }
            } else {
              st_shared_v4(sbase + offNan + ((tiles % kNanSlots) * kBlk + cw * 32 + lane) * 16, 0, 0, 0, 0);
            }
          }
          const uint32_t dst = sbase + offKV + (n % kSlots) * kTile + cw * 32 * 128;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t x[8];
            e4m3x4_f16(r[i].x, x[0], x[1]);
            e4m3x4_f16(r[i].y, x[2], x[3]);
            e4m3x4_f16(r[i].z, x[4], x[5]);
            e4m3x4_f16(r[i].w, x[6], x[7]);
            const uint32_t a = dst + ((i & 1) ^ (rl & 1)) * kBox + (i >> 1) * 8 * 128;
            st_shared_v4(a + a0, x[0], x[1], x[2], x[3]);
            st_shared_v4(a + a1, x[4], x[5], x[6], x[7]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&raw_empty[s]);
            mbar_arrive(&kv_full[n % kSlots]);
            if (kv) mbar_arrive(&nan_full[tiles % kScSlots]);
          }
        }
      }
    }
  } else {
    setmaxnreg_inc<kSoftmaxRegs>();
    // -------------------------------------------------------------------- query rows
    constexpr int GW = kBlk / NG, CH = 8 / NG;  // columns and maximum chains per scale group
    constexpr int SG = 8 / NG;                  // 16-key scale entries per group
    const int h = wg, quad = warp & 3, rr = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t o_addr = tmem + lane_addr + kColO + 128 * h;
    const int ri = rr / p.G, rg = rr - ri * p.G;  // token and head of this row within the half
    auto token_of = [&](const Unit& w) { return w.i0 + h * p.Tt + ri; };
    auto out_row = [&](const Unit& w, bool* inside) {
      const int i = token_of(w);
      *inside = ri < p.Tt && i < p.Sq;
      return p.o + w.b * p.o_seq + (int64_t)i * p.o_row + (int64_t)(w.hk * p.G + rg) * p.o_head;
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
    // the same row's place in the workspace, when several parts share a block's keys
    auto part_row = [&](const Unit& w, bool* inside) {
      const int rows = p.Tt * p.G;  // of a half
      *inside = ri < p.Tt && token_of(w) < p.Sq;
      const int64_t block = ((int64_t)w.b * p.c.heads + w.hk) * p.n_rt + w.i0 / (2 * p.Tt);
      return p.ws + ((block * 2 * rows + h * rows + rr) * p.parts + w.part) * kPartFloats;
    };
    uint32_t j = 0;
    const uint32_t s_addr = tmem + lane_addr + kColS + 128 * h;
    // This thread's row of the unit's Q in place, bf16 -> f16 times 2^-e, once the copy has landed;
    // the score factor of the row in *f
    auto q_convert = [&](uint32_t unit, float* f) {
      if (!warp_wait(&q_raw[h], unit & 1u, abort_flag, p, 90)) return false;
      const uint32_t base = sbase + offQ + h * kTile + rr * 128;
      const uint32_t flip = (rr & 7) << 4;
      // read once and kept: the shared memory's bandwidth is what this costs
      uint4 x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = ld_shared_v4(base + (k >> 3) * kBox + ((k & 7) << 4 ^ flip));
      uint32_t mx = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        mx = __vmaxu2(mx, __vmaxu2(__vmaxu2(x[k].x & 0x7FFF7FFFu, x[k].y & 0x7FFF7FFFu), __vmaxu2(x[k].z & 0x7FFF7FFFu, x[k].w & 0x7FFF7FFFu)));
      if (__vcmpgeu2(mx, 0x7F807F80u)) {  // infinities and NaN do not count, and pass through
        mx = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint32_t y[4] = {x[k].x & 0x7FFF7FFFu, x[k].y & 0x7FFF7FFFu, x[k].z & 0x7FFF7FFFu, x[k].w & 0x7FFF7FFFu};
#pragma unroll
          for (int q = 0; q < 4; ++q) mx = __vmaxu2(mx, y[q] & __vcmpltu2(y[q], 0x7F807F80u));
        }
      }
      mx = max(mx & 0xFFFFu, mx >> 16);
      const int e = imax((int)(mx >> 7) - 127 - 13, -126);  // |q| 2^-e < 2^14
      const float2 mul = make_float2(exp2i(-e), exp2i(-e));
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float2 f0 = mul_f2(bf2_f2(x[k].x), mul), f1 = mul_f2(bf2_f2(x[k].y), mul), f2 = mul_f2(bf2_f2(x[k].z), mul),
                     f3 = mul_f2(bf2_f2(x[k].w), mul);
        st_shared_v4(base + (k >> 3) * kBox + ((k & 7) << 4 ^ flip), pack_f16x2(f0.x, f0.y), pack_f16x2(f1.x, f1.y),
                     pack_f16x2(f2.x, f2.y), pack_f16x2(f3.x, f3.y));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[h]);
      *f = exp2i(e) * p.scale_log2;
      return true;
    };

    uint32_t t = 0;  // tiles
    Unit w, nw;
    float fr = 0.0f, next_fr = 0.0f, M = -INFINITY, m = -INFINITY, l = 0.0f;
    bool live = false;
    const uint32_t nan_at = sbase + offNanRow + (h * kBlk + rr) * 16;
    for (uint32_t it = 0;; ++it) {  // units, and the output of the last one
      // the next unit's Q, so that its Q K^T runs during this one's output
      const bool more = next_unit(&j, &nw);
      if (more && !q_convert(it, &next_fr)) break;
      if (it > 0) {
        // the output row: O 2^(M - m - 6) / l, the factor in two parts that stay normal
        float fa = 0.0f, fb = 0.0f;
        if (live && l != 0.0f) {
          fa = ex2(0.5f * (M - m - kBias));
          fb = fa / l;
        }
        bool inside;
        __nv_bfloat16* out = out_row(w, &inside);
        float* part = kSplit ? part_row(w, &inside) : nullptr;
        if (!warp_wait(&o_full[h], (it - 1) & 1u, abort_flag, p, 92)) break;
        tc_fence_after();
        const float2 a2 = make_float2(fa, fa), b2 = make_float2(fb, fb);
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t o[64];
          tmem_ld_32x32b_x32(o_addr + 64 * c, *reinterpret_cast<uint32_t(*)[32]>(o));
          tmem_ld_32x32b_x32(o_addr + 64 * c + 32, *reinterpret_cast<uint32_t(*)[32]>(o + 32));
          tmem_ld_wait();
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            uint32_t x[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) {
              const float2 v = mul_f2(
                  mul_f2(make_float2(__uint_as_float(o[32 * d + 2 * q]), __uint_as_float(o[32 * d + 2 * q + 1])), a2), b2);
              x[q] = fb == 0.0f ? 0u : pack_bf16x2(v.x, v.y);  // rows that see nothing: zeros, never 0 * NaN
              if (kSplit) {
                if (inside)
                  *reinterpret_cast<float2*>(part + 64 * c + 32 * d + 2 * q) = fb == 0.0f ? make_float2(0.0f, 0.0f) : v;
              }
            }
            if (inside && !kSplit) put(out + 64 * c + 32 * d, x);
          }
        }
        const uint4 nan = ld_shared_v4(nan_at);
        if ((nan.x | nan.y | nan.z | nan.w) && live) {  // channels that met a NaN of V
#pragma unroll 1
          for (int d = 0; d < kHeadDim; ++d) {
            const uint32_t bits = d < 32 ? nan.x : d < 64 ? nan.y : d < 96 ? nan.z : nan.w;
            if ((bits >> (d & 31)) & 1u) {
              if (kSplit)
                part[d] = __int_as_float(0x7FFFFFFF);
              else
                reinterpret_cast<unsigned short*>(out)[d] = 0x7FFF;
            }
          }
        }
        if (kSplit && inside)  // the part's own output, and what it weighs: l 2^m
          *reinterpret_cast<float4*>(part + kHeadDim) = fb == 0.0f ? make_float4(-INFINITY, 0.0f, 0.0f, 0.0f) : make_float4(m, l, 0.0f, l);
        tc_fence_before();  // O_h is read before this warp publishes the next unit's P_h
      }
      if (!more) break;
      w = nw;
      fr = next_fr;
      int jlo = 0, jhi = w.len;  // keys that this row sees: [jlo, jhi)
      live = false;
      {
        const int qi = token_of(w);
        live = ri < p.Tt && qi < w.nq;
        if (live) {
          const Keys k = visible(qi, qi, w.len, w.nq, p.causal != 0, p.window);
          jlo = k.lo;
          jhi = k.hi;
        }
      }
      M = m = -INFINITY;
      l = 0.0f;
      st_shared_v4(nan_at, 0, 0, 0, 0);
      bool ok = true;
      // the keys that every row of the warp sees: tiles within them need no mask
      const int all_lo = __reduce_max_sync(0xffffffffu, jlo), all_hi = __reduce_min_sync(0xffffffffu, jhi);
#pragma unroll 1
      for (int i = 0; i < w.nt; ++i, ++t) {
        if (!(ok = warp_wait(&sc_full[t % kScSlots], (t / kScSlots) & 1u, abort_flag, p, 82))) break;
        const uint32_t sc = sbase + offSc + (t % kScSlots) * kScWords * 4;
        const float4 tail = ld_shared_f32x4(sc + 4 * kScTail);
        const int k0 = (w.tile0 + i) * kBlk;
        if (!(ok = warp_wait(&s_full[h], t & 1u, abort_flag, p, 81))) break;
        tc_fence_after();
        if (k0 < all_lo || k0 + kBlk > all_hi) {
          // Keys that some row does not see: -inf into its scores where they lie.  (On the loaded
          // registers the same choice cost every tile, 382 us against 337 for 16 heads, 6,016 x 6,016.)
          const int lo = jlo - k0, hi = jhi - 1 - k0;
#pragma unroll 1
          for (int c = 0; c < kBlk; c += 16) {
            uint32_t x[16];
            tmem_ld_32x32b_x16(s_addr + c, x);
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 16; ++q) x[q] = (c + q < lo || c + q > hi) ? 0xFF800000u : x[q];
            tmem_st_32x32b_x16(s_addr + c, x);
          }
          tmem_st_wait();
        }
        uint32_t sr[kBlk];
        tmem_ld_32x32b_x32(s_addr + 0, *reinterpret_cast<uint32_t(*)[32]>(sr + 0));
        tmem_ld_32x32b_x32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(sr + 32));
        tmem_ld_32x32b_x32(s_addr + 64, *reinterpret_cast<uint32_t(*)[32]>(sr + 64));
        tmem_ld_32x32b_x32(s_addr + 96, *reinterpret_cast<uint32_t(*)[32]>(sr + 96));
        tmem_ld_wait();
        float* s = reinterpret_cast<float*>(sr);
        // score factor of a group, kept within 2^+-120: a masked score times 0 would be NaN
        const auto factor_of = [&](float k) { return fminf(fmaxf(fr * k, 7.5e-37f), 1.3e36f); };
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
          const float4 g4 = ld_shared_f32x4(sc + 16 * gi * SG);
          const float x = gm * factor_of(g4.x);
          mt = fmaxf(mt, x + g4.w);
          Mt = fmaxf(Mt, x + g4.y);
        }
        const bool up = mt > m + kRaise || (m == -INFINITY && mt > -INFINITY);
        const bool UP = Mt > M + kRaise || (M == -INFINITY && Mt > -INFINITY);
        const float m1 = up ? mt : m, M1 = UP ? Mt : M;
        const float mo = M1 == -INFINITY ? 0.0f : M1, ml = m1 == -INFINITY ? 0.0f : m1;
        const float D = mo - ml;
        const bool far = D - tail.x > kFast || tail.y - D > kFast;
        float lw = D;
        if (__any_sync(0xffffffffu, up || UP || far)) {
          if (up) l *= ex2(m - m1);
          if (__any_sync(0xffffffffu, UP && i > 0)) {
            // O_h *= 2^(M - M1): O_h is idle until this tile's P is published
            const float f = UP ? ex2(M - M1) : 1.0f;
#pragma unroll 1
            for (int oc = 0; oc < 8; ++oc) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(o_addr + 16 * oc, o);
              tmem_ld_wait();
#pragma unroll
              for (int q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * f);
              tmem_st_32x32b_x16(o_addr + 16 * oc, o);
            }
          }
          if (__any_sync(0xffffffffu, far)) {  // l's terms by an exponential of their own
#pragma unroll 1
            for (int c = 0; c < kBlk; c += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(s_addr + c, x);
              tmem_ld_wait();
              const float4 g4 = ld_shared_f32x4(sc + c);
              const float f = factor_of(g4.x);
#pragma unroll
              for (int q = 0; q < 16; ++q) l += ex2(fmaf(__uint_as_float(x[q]), f, g4.w - ml));
            }
            lw = -INFINITY;
          }
          m = m1;
          M = M1;
        }
        lw = ex2(lw - kBias - tail.z);  // weight of a sum at ev_0 in l
        float gf = 0.0f, gn = 0.0f, gl = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (c == 2) {
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pa_full[h]);
          }
          uint32_t pk[16];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if ((32 * c + 16 * half) % GW == 0) {  // the next group
              const float4 g4 = ld_shared_f32x4(sc + 16 * ((32 * c + 16 * half) / GW) * SG);
              gf = factor_of(g4.x);
              gn = g4.y - mo + kBias;
              gl = lw * g4.z;
            }
            const float2 f2 = make_float2(gf, gf), n2 = make_float2(gn, gn);
            float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const int at = 32 * c + 16 * half + 2 * q;
              const float2 x = fma_f2(make_float2(s[at], s[at + 1]), f2, n2);
              const float2 e = make_float2(ex2(x.x), ex2(x.y));
              acc = add_f2(acc, e);
              pk[8 * half + q] = pack_f16x2(e.x, e.y);
            }
            l = fmaf(gl, acc.x + acc.y, l);
          }
          tmem_st_32x32b_x16(s_addr + kColP + 16 * c, pk);
        }
        if (k0 < w.ks.lo_all || k0 + kBlk > w.ks.hi_all) {  // the converters leave NaN codes of V out of such tiles
          if (!(ok = warp_wait(&nan_full[t % kScSlots], (t / kScSlots) & 1u, abort_flag, p, 83))) break;
          const uint4 any = ld_shared_v4(sbase + offNanW + (t % kScSlots) * 16);
          if (any.x | any.y | any.z | any.w) {
            uint4 seen = ld_shared_v4(nan_at);
            const uint32_t map = sbase + offNan + (t % kNanSlots) * kBlk * 16;
#pragma unroll 1
            for (int c = imax(jlo - k0, 0); c <= imin(jhi - 1 - k0, kBlk - 1); ++c) {
              const uint4 x = ld_shared_v4(map + c * 16);
              seen.x |= x.x;
              seen.y |= x.y;
              seen.z |= x.z;
              seen.w |= x.w;
            }
            st_shared_v4(nan_at, seen.x, seen.y, seen.z, seen.w);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pb_full[h]);
      }
      if (!ok) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, kTmemCols);
}

template <int NG, bool kSplit>
int launch(const CUtensorMap& tq, const AttnParams& p, uint32_t units, int wide, unsigned grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const auto kernel = attention_tc_kernel<NG, kSplit>;
  if (device_pending(done)) {
    cudaFuncAttributes fa;
    DEMON_CUDA(cudaFuncGetAttributes(&fa, kernel));
    if (fa.numRegs != kLaunchRegs) {  // with fewer at launch the setmaxnreg.inc would never return
      set_error("kv_attention: kernel built with %d registers per thread, the register split needs %d", fa.numRegs, kLaunchRegs);
      return DEMON_ERR_CUDA;
    }
    DEMON_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    mark_device_done(done);
  }
  kernel<<<grid, kThreads, kSmem, st>>>(tq, p, units, wide);
  DEMON_CUDA(cudaGetLastError());
  return DEMON_OK;
}

template <int NG>
int launch(const CUtensorMap& tq, const AttnParams& p, uint32_t units, int wide, unsigned grid, cudaStream_t st) {
  return p.ws ? launch<NG, true>(tq, p, units, wide, grid, st) : launch<NG, false>(tq, p, units, wide, grid, st);
}

}  // namespace tc

int attention_tc(AttnParams p, cudaStream_t st) {
  using namespace tc;
  p.Tt = kBlk / p.G;
  p.n_rt = (p.Sq + 2 * p.Tt - 1) / (2 * p.Tt);
  const int64_t units = (int64_t)p.n_rt * p.B * p.c.heads * p.parts;
  DEMON_CHECK_ARG(units < ((int64_t)1 << 31), "kv_attention: too many work units (%lld)", (long long)units);
  CUtensorMap tq;
  const int rc0 = make_tmap_4d_bf16(&tq, p.q, {kHeadDim, (uint64_t)p.Hq, (uint64_t)p.Sq, (uint64_t)p.B},
                                    {(uint64_t)p.q_head * 2, (uint64_t)p.q_row * 2, (uint64_t)p.q_seq * 2},
                                    {64, (uint32_t)p.G, (uint32_t)p.Tt, 1});
  if (rc0 != DEMON_OK) return rc0;
  int dev = 0, sms = 148;
  DEMON_CUDA(cudaGetDevice(&dev));
  DEMON_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  const unsigned grid = (unsigned)std::min<int64_t>(units, sms);
  const int wide = ((uintptr_t)p.o & 31) == 0 && p.o_seq % 16 == 0 && p.o_row % 16 == 0 && p.o_head % 16 == 0;
  const uint32_t n = (uint32_t)units;
  switch (p.c.P) {
    case 16: return launch<8>(tq, p, n, wide, grid, st);
    case 32: return launch<4>(tq, p, n, wide, grid, st);
    case 64: return launch<2>(tq, p, n, wide, grid, st);
    default: return launch<1>(tq, p, n, wide, grid, st);
  }
}

}  // namespace kv
}  // namespace demon
