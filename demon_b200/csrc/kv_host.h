// kv_host.h -- host-side checks shared by the entry points of the paged 8-bit K/V cache.
#pragma once
#include "demon_host.h"

namespace demon {
namespace kv {
struct Cache;
struct AttnParams;
// kv_attention_tc.cu: the call's rows in blocks on the tensor cores; at most 128 query heads per kv head.
int attention_tc(AttnParams p, cudaStream_t st);
}  // namespace kv
// DEMON_OK, or DEMON_ERR_INVALID with the message set (`who`: the entry point's name).
int kv_cache_check(const DemonKvCache* c, const char* who);
int kv_table_check(const int32_t* table, int64_t ld, int32_t B, int32_t W, int page_size, const char* who);
kv::Cache kv_cache(const DemonKvCache* c);
}  // namespace demon
