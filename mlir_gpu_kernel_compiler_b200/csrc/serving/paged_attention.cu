// Host side of the attention over a paged cache: checks, the choice of kernel, the launch.
#include "paged_attention_rows.cuh"

namespace tjs {

struct Plan {
  long grid;
  int rows;    // of a tile
  int target;
  int min_chunk;
};

const char* attention_fault(const tj_paged_attention& a) {
  if (a.dtype != TJ_F16 && a.dtype != TJ_BF16) return "q must be f16 or bf16";
  if (const char* why = cache_fault(a.cache)) return why;
  if ((a.cache.dtype == TJ_F16 || a.cache.dtype == TJ_BF16) && a.cache.dtype != a.dtype)
    return "a 16-bit cache must have q's type";
  if (a.cache.dim != 64 && a.cache.dim != 128) return "head dim must be 64 or 128";
  if (a.tokens < 0 || a.batch < 0 || a.q_heads <= 0 || a.max_new <= 0 || a.table_width <= 0 || a.window < 0)
    return "bad extent";
  if (a.q_heads % a.cache.heads) return "query heads must be a multiple of the cache's heads";
  if (a.tokens > 0x7fffffffLL / a.q_heads || a.batch > 0x7fffffLL) return "too many rows";
  if (!a.q_starts && a.tokens != a.batch) return "without q_starts there is one token to a sequence";
  if (!(a.scale > 0.0)) return "scale must be positive";
  return nullptr;
}

Plan plan_rows(const tj_paged_attention& a, const Device& dev) {
  Plan p;
  const long group = a.q_heads / a.cache.heads;
  const bool q8 = a.cache.dtype == TJ_I8 || a.cache.dtype == TJ_E4M3;
  p.rows = 16;
  const long tiles = a.q_starts ? a.tokens * group / 16 + a.batch : a.batch * ((group + 15) / 16);
  p.target = dev.sms * (a.cache.dim == 64 ? 4 : 3) * 2;
  p.min_chunk = q8 ? 256 : 128;
  p.grid = a.cache.heads * (tiles + 1) + p.target;
  return p;
}

template <class T, int CD> void launch_rows_kernel(const AttnParams& p, unsigned grid, cudaStream_t st) {
  if (p.a.cache.dim == 64)
    attention_rows<T, CD, 64><<<grid, 128, 0, st>>>(p);
  else
    attention_rows<T, CD, 128><<<grid, 128, 0, st>>>(p);
}
template <class T> void launch_rows_type(const AttnParams& p, unsigned grid, cudaStream_t st) {
  switch (p.a.cache.dtype) {
    case TJ_I8: launch_rows_kernel<T, TJ_I8>(p, grid, st); break;
    case TJ_E4M3: launch_rows_kernel<T, TJ_E4M3>(p, grid, st); break;
    default: launch_rows_kernel<T, TJ_BF16>(p, grid, st); break;
  }
}

int64_t part_bytes(const tj_paged_attention& a, const Plan& p) { return p.grid * p.rows * (a.cache.dim * 4 + 8); }

}  // namespace tjs

extern "C" int tj_b200_paged_attention_workspace(const tj_paged_attention* args, int64_t* workspace_bytes,
                                                 int64_t* counters_count) {
  using namespace tjs;
  const char* name = "tj_b200_paged_attention_workspace";
  if (!args || !workspace_bytes || !counters_count) return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  if (const char* why = attention_fault(*args)) return refuse(TJ_ERR_INVALID, name, why);
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  const Plan plan = plan_rows(*args, dev);
  *workspace_bytes = part_bytes(*args, plan);
  *counters_count = plan.grid;
  return TJ_OK;
}

extern "C" int tj_b200_paged_attention(const tj_paged_attention* args, void* stream) {
  using namespace tjs;
  const char* name = "tj_b200_paged_attention";
  if (!args) return refuse(TJ_ERR_INVALID, name, "NULL arguments");
  const tj_paged_attention& a = *args;
  if (const char* why = attention_fault(a)) return refuse(TJ_ERR_INVALID, name, why);
  if (a.tokens == 0 || a.batch == 0) return TJ_OK;
  if (!a.q || !a.out || !a.page_table || !a.kv_lens || !a.workspace || !a.counters)
    return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace)) % 16 ||
      (a.q_token | a.q_head | a.out_token | a.out_head) % 8)
    return refuse(TJ_ERR_INVALID, name, "rows must start on 16-byte boundaries");
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  const Plan plan = plan_rows(a, dev);
  if (a.workspace_bytes < part_bytes(a, plan) || a.counters_count < plan.grid)
    return refuse(TJ_ERR_INVALID, name, "workspace or counters too small");
  if (plan.grid > 0x7fffffffL) return refuse(TJ_ERR_INVALID, name, "too many rows");
  AttnParams p;
  p.a = a;
  p.status = dev.status;
  p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.group = static_cast<int>(a.q_heads / a.cache.heads);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.cache.page_size == (1LL << i)) p.page_shift = i;
  p.target = plan.target;
  p.min_chunk = plan.min_chunk;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + plan.grid * plan.rows * a.cache.dim);
  p.counters = a.counters;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.dtype == TJ_BF16)
    launch_rows_type<__nv_bfloat16>(p, static_cast<unsigned>(plan.grid), st);
  else
    launch_rows_type<__half>(p, static_cast<unsigned>(plan.grid), st);
  return launched(name);
}
