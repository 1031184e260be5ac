// kv_common.cuh -- device helpers of the paged E4M3 K/V cache kernels.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "demon_common.cuh"
#include "kv_index.h"

namespace demon {
namespace kv {

// The cache as the kernels see it.  Page p, head h: P x 128 codes at ((p * heads + h) * P) * 128,
// one scale at p * heads + h.
struct Cache {
  uint8_t* codes[2];  // K, V
  float* scale[2];
  int64_t pages;
  int heads, P;
};

// Four E4M3 codes -> two packed f16 pairs (exact: E4M3 values are f16 values).
__device__ __forceinline__ void e4m3x4_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ float2 f16x2_f32(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Two fp32 values -> E4M3 codes, nearest even, saturating at +-448 (infinities too); NaN stays
// NaN.  `a` in the low byte.
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }
// Exponent of a power-of-two scale, brought into the range that the cache uses.
__device__ __forceinline__ int scale_exp(float s) {
  return imin(imax((int)((__float_as_uint(s) >> 23) & 255u) - 127, kMinExp), kMaxExp);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 0x80 in every byte of w that is E4M3's NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ float ld_shared_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_f32x4(uint32_t a, float x, float y, float z, float w) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}

// A partial result of a row in the workspace: O [128], then the maximum m (log2 units) and the sum l
// (in units of 2^m), the exponent that O is held in units of, and O's weight beside 2^m.
constexpr int kPartFloats = kHeadDim + 4;

// One attention call, as both attention kernels see it.
struct AttnParams {
  Cache c;
  const __nv_bfloat16* q;
  int64_t q_seq, q_row, q_head;
  __nv_bfloat16* o;
  int64_t o_seq, o_row, o_head;
  const int32_t *table, *lens, *q_lens;
  int64_t ld_table;
  int B, Sq, Hq, G, W;
  int causal, window;  // window < 0: no band
  float scale_log2;    // softmax scale * log2(e)
  int n_rt;            // row tiles (or blocks) per kv head
  int Tt;              // tokens per half block (tensor-core kernel)
  int cluster;         // CTAs per cluster (small kernel)
  int parts;           // parts that share the keys of a row tile (or block)
  float* ws;           // their partial results, joined by attention_join_kernel; null: none
  unsigned int* status;
};

// What a wait of a call may take: 2 s, and 1 us for every key of the table, some ten times what the
// attention kernels need for the units that a warp may wait for (a cache may hold 2^30 keys).
__device__ __forceinline__ uint64_t wait_limit(const AttnParams& p) {
  return DEMON_WAIT_LIMIT_NS + (uint64_t)(uint32_t)p.W * (uint32_t)p.c.P * 1000u;
}
// mbar_wait with the time counted from this wait's own start, not the kernel's: a long call (half a
// million tokens over as many keys take seconds) is no failure.
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, volatile int* abort, const AttnParams& p,
                                             unsigned int where) {
  const uint32_t a = smem_u32(bar);
  uint64_t since = 0;
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(a, parity)) return true;
    if ((i & 255u) == 255u) {
      if (*abort) return false;
      const uint64_t now = globaltimer();
      if (since == 0) since = now;
      if (now - since > wait_limit(p)) {
        *abort = 1;
        report(p.status, DEMON_DEV_TIMEOUT, where);
        return false;
      }
    }
  }
}

}  // namespace kv
}  // namespace demon
