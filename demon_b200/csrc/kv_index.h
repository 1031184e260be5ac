// kv_index.h -- index arithmetic of the paged 8-bit K/V cache, shared by its kernels and by
// host code (plain C++ without CUDA types, so the CPU tests compile it as it is).
//
// Everything a kernel reads from device memory before it forms an address (a page id, a
// length, a start) goes through one of these checks first: a value out of range gives an
// empty span or page -1, the kernel reports DEMON_DEV_BAD_ARG in the status word and touches
// nothing for it.
#pragma once
#include <cstdint>

#if defined(__CUDACC__)
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

namespace demon {
namespace kv {

constexpr int kHeadDim = 128;        // values per token and head
constexpr int kMaxTokens = 1 << 30;  // positions a table may cover, and the largest window
constexpr int kMinExp = -120, kMaxExp = 119;  // scale exponents: every code * 2^e is a bf16 value

KV_HD int imin(int a, int b) { return a < b ? a : b; }
KV_HD int imax(int a, int b) { return a > b ? a : b; }

// Tokens an append writes for one sequence: [start, start + count), empty and bad when it does
// not lie in [0, cap).
struct Span {
  int start, count;
  bool bad;
};
KV_HD Span append_span(int start, int count, int S, int cap) {
  const bool bad = start < 0 || count < 0 || count > S || start > cap || count > cap - start;
  Span s;
  s.start = bad ? 0 : start;
  s.count = bad ? 0 : count;
  s.bad = bad;
  return s;
}

// Pages an append of S tokens can touch (the last one may be empty).
KV_HD int append_pages(int S, int P) { return (int)(((int64_t)S + P - 2) / P) + 1; }

// A length held in device memory, brought into [0, cap].
KV_HD int clamp_len(int len, int cap, bool* bad) {
  if (len < 0 || len > cap) *bad = true;
  return imin(imax(len, 0), cap);
}

// Page id of entry i of a sequence's table row, or -1 when there is none.
KV_HD int page_id(const int32_t* row, int W, int i, int64_t pages) {
  if (i < 0 || i >= W) return -1;
  const int p = row[i];
  return p >= 0 && (int64_t)p < pages ? p : -1;
}

// Keys that queries i0 .. i1 of a sequence see: some query sees a key of [lo, hi) and none sees
// one outside; every query sees all of [lo_all, hi_all).  Query i stands at position
// len - nq + i; causal: j <= position; window >= 0: |j - position| <= window.
struct Keys {
  int lo, hi, lo_all, hi_all;
};
KV_HD Keys visible(int i0, int i1, int len, int nq, bool causal, int window) {
  const int p0 = len - nq + i0, p1 = len - nq + i1;
  Keys k;
  k.lo = k.lo_all = 0;
  k.hi = k.hi_all = len;
  if (window >= 0) {
    k.lo = imax(0, p0 - window);
    k.lo_all = imax(0, p1 - window);
    k.hi = imin(len, imax(0, p1 + window + 1));
    k.hi_all = imin(len, imax(0, p0 + window + 1));
  }
  if (causal) {
    k.hi = imin(k.hi, imax(0, p1 + 1));
    k.hi_all = imin(k.hi_all, imax(0, p0 + 1));
  }
  k.hi = imax(k.hi, k.lo);  // empty: hi == lo
  return k;
}

}  // namespace kv
}  // namespace demon
