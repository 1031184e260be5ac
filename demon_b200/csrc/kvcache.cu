// kvcache.cu -- writing tokens into a paged E4M3 K/V cache and reading them back.
//
// A page holds P tokens of every kv head; per page and head there is one power-of-two scale
// 2^e, and a value is code * 2^e.  A power of two costs E4M3 nothing in relative precision
// (the codes are floating point; only the subnormal end moves), makes every cached value
// exact in bf16, and lets a scale grow in place: code * 2^(e_old - e) is exact but for the
// codes that become subnormal.
//
// Append (one launch for K and V).  For a page and head with n_old tokens before `start`:
//   a = max |finite new values|,  e = min { e : a <= 448 2^e },  e = max(e, e_old) if n_old > 0,
//   code = rne_e4m3(x 2^-e);  when e > e_old the n_old codes are rounded again to 2^e.
// One pass: 16 tokens of a page and head are one warp's, 16 lanes x 16 bytes per token, all
// eight of a lane's loads in flight and kept in registers between the maximum and the
// rounding; P / 16 warps of a CTA share a page and join their maxima through shared memory.
// Bound by memory for prompts (22,000 tokens of 8 heads: 134 MB in 25.9 us, 5.2 TB/s; 36.9 us with
// 64-bit unit arithmetic, a finite mask on every word and the page looked up before the loads),
// by the launch for single tokens (3 us).  Four CTAs per SM: 28.2 us with three, 27.5 with five.
//
// Read.  Eight lanes take one token and head (128 codes, 16 per lane) and write its 256 bytes;
// consecutive rows are the heads of one token, so a warp's stores are contiguous.  Bound by memory,
// the writes above all: 32-byte stores and two rows per lane took 135.6 us to 106.5 us for 691 MB
// (6.5 TB/s, the measured copy rate; four rows or 16-byte stores keep fewer requests in flight).
#include "demon_host.h"
#include "kv_common.cuh"
#include "kv_host.h"

namespace demon {
namespace kv {

constexpr int kAppendThreads = 256;
constexpr int kTokWarp = 16;  // tokens of a page per warp

struct AppendParams {
  Cache c;
  const __nv_bfloat16* x[2];
  int64_t seq[2], row[2], head[2];  // element strides of x
  const int32_t *table, *start, *count;
  int64_t ld_table;
  int B, S, W, T;     // T: pages an append can touch
  int groups;         // page-head groups per CTA: 128 / P
  uint32_t units;     // B * T * 2 * heads groups in all
  unsigned int* status;
};

// max of packed bf16 magnitudes, and the same over the finite ones
__device__ __forceinline__ uint32_t mag_max(uint32_t m, uint32_t v) { return __vmaxu2(m, v & 0x7FFF7FFFu); }
__device__ __forceinline__ uint32_t finite_max(uint32_t m, uint32_t v) {
  const uint32_t a = v & 0x7FFF7FFFu;
  return __vmaxu2(m, a & __vcmpltu2(a, 0x7F807F80u));
}

__global__ void __launch_bounds__(kAppendThreads, 4) append_kernel(const AppendParams p) {
  __shared__ uint32_t warp_max[kAppendThreads / 32];
  const int P = p.c.P, nw = P / kTokWarp;  // warps per page
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = warp / nw, wip = warp - grp * nw;
  // unit order: heads fastest, then K / V, then the page, then the sequence, so that a CTA's
  // neighbours read the same token rows
  const uint32_t u = blockIdx.x * (uint32_t)p.groups + grp;  // below 2^31 (checked on the host)
  bool active = u < p.units;
  const uint32_t uu = active ? u : 0, heads = (uint32_t)p.c.heads;
  const uint32_t r1 = uu / heads, r2 = r1 >> 1;
  const int h = (int)(uu - r1 * heads), kv = (int)(r1 & 1);
  const int b = (int)(r2 / (uint32_t)p.T), t = (int)(r2 - (uint32_t)b * (uint32_t)p.T);

  const Span sp = append_span(p.start[b], p.count ? p.count[b] : p.S, p.S, p.W * P);
  if (sp.bad && active && t == 0 && h == 0 && lane == 0 && wip == 0) report(p.status, DEMON_DEV_BAD_ARG, 60);
  const int end = sp.start + sp.count;
  const int page = sp.start / P + t, tok0 = page * P;
  active = active && sp.count > 0 && tok0 < end;

  // the new tokens' loads first: their addresses do not wait for the page
  const int sub = lane & 15;
  uint4 v[8];
  bool mine[8];
  uint32_t mx = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int pos = tok0 + wip * kTokWarp + 2 * j + (lane >> 4);
    mine[j] = active && pos >= sp.start && pos < end;
    v[j] = make_uint4(0, 0, 0, 0);
    if (mine[j])
      v[j] = __ldg(reinterpret_cast<const uint4*>(p.x[kv] + b * p.seq[kv] + (int64_t)(pos - sp.start) * p.row[kv] +
                                                  h * p.head[kv] + sub * 8));
  }
  int pid = -1;
  if (active) {
    pid = page_id(p.table + b * p.ld_table, p.W, page, p.c.pages);
    if (pid < 0 && h == 0 && lane == 0 && wip == 0) report(p.status, DEMON_DEV_BAD_ARG, 61);
    active = pid >= 0;
  }
  const int64_t ph = active ? (int64_t)pid * p.c.heads + h : 0;
  const int n_old = imin(imax(sp.start - tok0, 0), P);
  const float s_old = active && n_old > 0 ? p.c.scale[kv][ph] : 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) mx = mag_max(mag_max(mag_max(mag_max(mx, v[j].x), v[j].y), v[j].z), v[j].w);
  if (__vcmpgeu2(mx, 0x7F807F80u)) {  // infinities or NaN: they do not count
    mx = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = finite_max(finite_max(finite_max(finite_max(mx, v[j].x), v[j].y), v[j].z), v[j].w);
  }
  uint32_t am = max(mx & 0xFFFFu, mx >> 16);
  am = __reduce_max_sync(0xffffffffu, am);
  if (nw > 1) {
    if (lane == 0) warp_max[warp] = am;
    __syncthreads();
    for (int w = 0; w < nw; ++w) am = max(am, warp_max[grp * nw + w]);
  }
  if (!active) return;

  // am: bits of a bf16 magnitude m7 / 128 * 2^(E - 127) with 128 <= m7 + 128 < 256; 448 = 7/8 2^9
  int e = (int)(am >> 7) - 135 + ((am & 127u) > 96u ? 1 : 0);
  e = imin(imax(e, kMinExp), kMaxExp);
  const int e_old = scale_exp(s_old);
  if (n_old > 0) e = imax(e, e_old);
  if (lane == 0 && wip == 0 && (n_old == 0 || e != e_old)) p.c.scale[kv][ph] = exp2i(e);
  const float inv = exp2i(-e);
  uint8_t* dst = p.c.codes[kv] + (ph * P + wip * kTokWarp) * kHeadDim + sub * 8;
  const float2 iv = make_float2(inv, inv);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (!mine[j]) continue;
    const float2 f0 = mul_f2(bf2_f2(v[j].x), iv), f1 = mul_f2(bf2_f2(v[j].y), iv), f2 = mul_f2(bf2_f2(v[j].z), iv),
                 f3 = mul_f2(bf2_f2(v[j].w), iv);
    *reinterpret_cast<uint2*>(dst + (2 * j + (lane >> 4)) * kHeadDim) =
        make_uint2(e4m3x4(f0.x, f0.y, f1.x, f1.y), e4m3x4(f2.x, f2.y, f3.x, f3.y));
  }
  if (n_old > 0 && e > e_old) {  // the scale grew: round the earlier tokens' codes to it
    const float f = exp2i(imax(e_old - e, -30));  // below 2^-30 every code rounds to zero
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      const int tok = wip * kTokWarp + 2 * j + (lane >> 4);
      if (tok >= n_old) continue;
      uint2* a = reinterpret_cast<uint2*>(dst + (2 * j + (lane >> 4)) * kHeadDim);
      uint2 w = *a;
      uint32_t q[4];
      e4m3x4_f16(w.x, q[0], q[1]);
      e4m3x4_f16(w.y, q[2], q[3]);
      const float2 f0 = f16x2_f32(q[0]), f1 = f16x2_f32(q[1]), f2 = f16x2_f32(q[2]), f3 = f16x2_f32(q[3]);
      w.x = e4m3x4(f0.x * f, f0.y * f, f1.x * f, f1.y * f);
      w.y = e4m3x4(f2.x * f, f2.y * f, f3.x * f, f3.y * f);
      *a = w;
    }
  }
}

// ---------------------------------------------------------------------------------- read

constexpr int kReadThreads = 256;
constexpr int kReadRows = 2;  // rows (token, head) per eight lanes

struct ReadParams {
  Cache c;
  __nv_bfloat16* out[2];
  int64_t seq[2], row[2];  // element strides of out; heads contiguous
  const int32_t *table, *lens;
  int64_t ld_table;
  uint32_t rows;  // rows of a sequence: max_len * heads
  int W;
  int wide;  // 32-byte stores: outputs and pitches aligned to 32 bytes
  unsigned int* status;
};

__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadParams p) {
  const int P = p.c.P, b = blockIdx.y, kv = blockIdx.z;
  const int sub = threadIdx.x & 7;
  bool bad = false;
  const int len = clamp_len(p.lens[b], p.W * P, &bad);
  const uint32_t r0 = (blockIdx.x * kReadRows) * (kReadThreads / 8) + (threadIdx.x >> 3), heads = (uint32_t)p.c.heads;
  const int32_t* row = p.table + b * p.ld_table;
  uint4 w[kReadRows];
  float s[kReadRows];
  int tok[kReadRows], h[kReadRows];
#pragma unroll
  for (int j = 0; j < kReadRows; ++j) {
    const uint32_t r = r0 + j * (kReadThreads / 8);
    tok[j] = r < p.rows ? (int)(r / heads) : -1;
    h[j] = (int)(r - (uint32_t)tok[j] * heads);
    w[j] = make_uint4(0, 0, 0, 0);
    s[j] = 0.0f;
    if (tok[j] >= 0 && tok[j] < len) {
      const int page = tok[j] / P, pid = page_id(row, p.W, page, p.c.pages);
      if (pid >= 0) {
        const int64_t ph = (int64_t)pid * p.c.heads + h[j];
        s[j] = __ldg(p.c.scale[kv] + ph);
        w[j] = __ldg(reinterpret_cast<const uint4*>(p.c.codes[kv] + (ph * P + (tok[j] - page * P)) * kHeadDim + sub * 16));
      } else {
        bad = true;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kReadRows; ++j) {
    if (tok[j] < 0) continue;
    __nv_bfloat16* o = p.out[kv] + b * p.seq[kv] + (int64_t)tok[j] * p.row[kv] + h[j] * kHeadDim + sub * 16;
    const uint32_t in[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo, hi;
      e4m3x4_f16(in[i], lo, hi);
      const float2 a = f16x2_f32(lo), c = f16x2_f32(hi);
      r[2 * i] = pack_bf16x2(a.x * s[j], a.y * s[j]);
      r[2 * i + 1] = pack_bf16x2(c.x * s[j], c.y * s[j]);
    }
    if (p.wide) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                   "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                   : "memory");
    } else {
      st_global_v4(o, make_uint4(r[0], r[1], r[2], r[3]));
      st_global_v4(o + 8, make_uint4(r[4], r[5], r[6], r[7]));
    }
  }
  if (bad) report(p.status, DEMON_DEV_BAD_ARG, 62);
}

}  // namespace kv

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int kv_cache_check(const DemonKvCache* c, const char* who) {
  DEMON_CHECK_ARG(c->pages == 0 || (c->k && c->v && c->k_scale && c->v_scale), "%s: null cache buffer", who);
  DEMON_CHECK_ARG(al16(c->k) && al16(c->v), "%s: cache codes must be 16-byte aligned", who);
  DEMON_CHECK_ARG(((uintptr_t)c->k_scale & 3) == 0 && ((uintptr_t)c->v_scale & 3) == 0,
                  "%s: cache scales must be 4-byte aligned", who);
  DEMON_CHECK_ARG(c->head_dim == kv::kHeadDim, "%s: head_dim must be %d (got %d)", who, kv::kHeadDim, c->head_dim);
  DEMON_CHECK_ARG(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 || c->page_size == 128,
                  "%s: page_size must be 16, 32, 64 or 128 (got %d)", who, c->page_size);
  DEMON_CHECK_ARG(c->heads >= 1 && c->heads <= 1024, "%s: 1 to 1024 kv heads (got %d)", who, c->heads);
  DEMON_CHECK_ARG(c->pages >= 0 && c->pages < ((int64_t)1 << 31), "%s: bad page count %lld", who, (long long)c->pages);
  return DEMON_OK;
}

int kv_table_check(const int32_t* table, int64_t ld, int32_t B, int32_t W, int page_size, const char* who) {
  DEMON_CHECK_ARG(B >= 0 && W >= 0, "%s: bad sizes B=%d W=%d", who, B, W);
  DEMON_CHECK_ARG(table != nullptr || B == 0 || W == 0, "%s: null page table", who);
  DEMON_CHECK_ARG(ld >= W || B <= 1, "%s: table row pitch %lld is below its width %d", who, (long long)ld, W);
  DEMON_CHECK_ARG((int64_t)W * page_size <= kv::kMaxTokens, "%s: the table covers more than 2^30 tokens (W=%d)", who, W);
  return DEMON_OK;
}

kv::Cache kv_cache(const DemonKvCache* c) {
  kv::Cache r;
  r.codes[0] = (uint8_t*)c->k;
  r.codes[1] = (uint8_t*)c->v;
  r.scale[0] = c->k_scale;
  r.scale[1] = c->v_scale;
  r.pages = c->pages;
  r.heads = c->heads;
  r.P = c->page_size;
  return r;
}

}  // namespace demon

using namespace demon;

extern "C" int demon_kv_append(const DemonKvAppendArgs* a, void* stream) {
  DEMON_API_BEGIN();
  DEMON_CHECK_ARG(a != nullptr, "kv_append: null argument block");
  int rc = kv_cache_check(&a->cache, "kv_append");
  if (rc == DEMON_OK) rc = kv_table_check(a->table, a->ld_table, a->B, a->W, a->cache.page_size, "kv_append");
  if (rc != DEMON_OK) return rc;
  DEMON_CHECK_ARG(a->S >= 0 && a->S <= kv::kMaxTokens, "kv_append: bad token count S=%d", a->S);
  if (a->B == 0 || a->S == 0) return DEMON_OK;
  DEMON_CHECK_ARG(a->k && a->v && a->start, "kv_append: null k / v / start");
  DEMON_CHECK_ARG(a->cache.pages == 0 || (a->cache.k != a->cache.v && a->cache.k_scale != a->cache.v_scale),
                  "kv_append: the cache's K and V are one buffer");
  DEMON_CHECK_ARG(al16(a->k) && al16(a->v), "kv_append: k and v must be 16-byte aligned");
  DEMON_CHECK_ARG(a->k_seq % 8 == 0 && a->k_row % 8 == 0 && a->k_head % 8 == 0 && a->v_seq % 8 == 0 &&
                      a->v_row % 8 == 0 && a->v_head % 8 == 0,
                  "kv_append: k / v strides must be multiples of 8 elements");
  kv::AppendParams p{};
  p.c = kv_cache(&a->cache);
  p.x[0] = (const __nv_bfloat16*)a->k;
  p.x[1] = (const __nv_bfloat16*)a->v;
  p.seq[0] = a->k_seq, p.row[0] = a->k_row, p.head[0] = a->k_head;
  p.seq[1] = a->v_seq, p.row[1] = a->v_row, p.head[1] = a->v_head;
  p.table = a->table, p.start = a->start, p.count = a->count, p.ld_table = a->ld_table;
  p.B = a->B, p.S = a->S, p.W = a->W;
  p.T = kv::append_pages(a->S, a->cache.page_size);
  p.groups = kv::kAppendThreads / 32 / (a->cache.page_size / kv::kTokWarp);
  const int64_t units = (int64_t)a->B * p.T * 2 * a->cache.heads;
  DEMON_CHECK_ARG(units < ((int64_t)1 << 31) - 8, "kv_append: too many pages (%lld)", (long long)units);
  p.units = (uint32_t)units;
  p.status = status_word();
  const int64_t grid = (units + p.groups - 1) / p.groups;
  kv::append_kernel<<<(unsigned)grid, kv::kAppendThreads, 0, (cudaStream_t)stream>>>(p);
  DEMON_CUDA(cudaGetLastError());
  return DEMON_OK;
}

extern "C" int demon_kv_read(const DemonKvReadArgs* a, void* stream) {
  DEMON_API_BEGIN();
  DEMON_CHECK_ARG(a != nullptr, "kv_read: null argument block");
  int rc = kv_cache_check(&a->cache, "kv_read");
  if (rc == DEMON_OK) rc = kv_table_check(a->table, a->ld_table, a->B, a->W, a->cache.page_size, "kv_read");
  if (rc != DEMON_OK) return rc;
  DEMON_CHECK_ARG(a->max_len >= 0 && a->max_len <= kv::kMaxTokens, "kv_read: bad max_len %d", a->max_len);
  DEMON_CHECK_ARG(a->B <= 65535, "kv_read: at most 65535 sequences (got %d)", a->B);
  if (a->B == 0 || a->max_len == 0) return DEMON_OK;
  DEMON_CHECK_ARG(a->k_out && a->v_out && a->lens, "kv_read: null output / lens");
  DEMON_CHECK_ARG(al16(a->k_out) && al16(a->v_out), "kv_read: outputs must be 16-byte aligned");
  DEMON_CHECK_ARG(a->k_seq % 8 == 0 && a->k_row % 8 == 0 && a->v_seq % 8 == 0 && a->v_row % 8 == 0,
                  "kv_read: output strides must be multiples of 8 elements");
  const int64_t width = (int64_t)a->cache.heads * kv::kHeadDim;
  DEMON_CHECK_ARG(a->k_row >= width && a->v_row >= width, "kv_read: output rows must hold every head");
  DEMON_CHECK_ARG(a->B == 1 || (a->k_seq >= (a->max_len - 1) * a->k_row + width &&
                                a->v_seq >= (a->max_len - 1) * a->v_row + width),
                  "kv_read: output sequences overlap");
  DEMON_CHECK_ARG(a->k_out != a->v_out, "kv_read: k_out and v_out overlap");
  kv::ReadParams p{};
  p.c = kv_cache(&a->cache);
  p.out[0] = (__nv_bfloat16*)a->k_out;
  p.out[1] = (__nv_bfloat16*)a->v_out;
  p.seq[0] = a->k_seq, p.row[0] = a->k_row, p.seq[1] = a->v_seq, p.row[1] = a->v_row;
  p.table = a->table, p.lens = a->lens, p.ld_table = a->ld_table;
  const int64_t rows = (int64_t)a->max_len * a->cache.heads;
  DEMON_CHECK_ARG(rows < ((int64_t)1 << 31) - 256, "kv_read: too many rows a sequence (%lld)", (long long)rows);
  p.rows = (uint32_t)rows;
  p.W = a->W;
  p.wide = (((uintptr_t)a->k_out | (uintptr_t)a->v_out) & 31) == 0 && a->k_seq % 16 == 0 && a->k_row % 16 == 0 &&
           a->v_seq % 16 == 0 && a->v_row % 16 == 0;
  p.status = status_word();
  const int64_t per = (int64_t)kv::kReadRows * (kv::kReadThreads / 8);
  const int64_t grid = (rows + per - 1) / per;
  kv::read_kernel<<<dim3((unsigned)grid, (unsigned)a->B, 2), kv::kReadThreads, 0, (cudaStream_t)stream>>>(p);
  DEMON_CUDA(cudaGetLastError());
  return DEMON_OK;
}

extern "C" int demon_kv_struct_sizes(int64_t* append_args, int64_t* read_args, int64_t* attn_args) {
  if (!append_args || !read_args || !attn_args) return DEMON_ERR_INVALID;
  *append_args = (int64_t)sizeof(DemonKvAppendArgs);
  *read_args = (int64_t)sizeof(DemonKvReadArgs);
  *attn_args = (int64_t)sizeof(DemonKvAttnArgs);
  return DEMON_OK;
}
