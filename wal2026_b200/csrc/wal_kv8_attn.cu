// Entry points of the attention over the paged 8-bit KV cache; the kernel is in wal_kv8_attn.cuh.
#include "wal_kv8_attn.cuh"

extern "C" {

size_t wal_kv8_attention_workspace(const wal_kv8_cache* cache, int64_t B, int64_t T, int32_t hq) {
  return attention_workspace(cache, B, T, hq);
}

int wal_kv8_attention(const wal_kv8_cache* cache, int32_t layer, const uint16_t* q, int64_t ld_q, int64_t B, int64_t T,
                      int32_t hq, const int32_t* table, int64_t ld_table, int64_t max_pages, const int32_t* lens,
                      const int32_t* new_lens, float scale, uint16_t* out, int64_t ld_out, void* workspace,
                      size_t workspace_bytes, void* stream) {
  Plan plan = {};
  const int st = make_plan(cache, layer, q, ld_q, B, T, hq, table, ld_table, max_pages, lens, new_lens, scale, out, ld_out,
                           workspace, workspace_bytes, &plan);
  if (st != WAL_OK) return st;
  return launch_plan<false>(plan, cache->head_dim, cache->kind, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
