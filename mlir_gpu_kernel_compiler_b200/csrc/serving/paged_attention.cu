// Host side of the attention over a paged cache: checks, the choice of kernel, the launch.
#include <algorithm>

#include "paged_attention_rows.cuh"
#include "paged_attention_tiles.cuh"

namespace tjs {

struct Plan {
  bool tiles;      // the tensor-core kernel of many rows
  bool wide;       // the kernel of few rows with one CTA an SM
  long grid;
  long slots;      // partial results kept at once
  int rows;        // of a tile
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

Plan plan(const tj_paged_attention& a, const Device& dev) {
  Plan p;
  const long group = a.q_heads / a.cache.heads;
#ifndef TJS_LIMIT
#define TJS_LIMIT 500000
#endif
  const long row_tiles = a.q_starts ? a.tokens * group / 16 + a.batch : a.batch * ((group + 15) / 16);
  const long reach = a.table_width * a.cache.page_size, keys = a.window > 0 ? std::min<long>(reach, a.window + a.max_new) : reach;
  p.tiles = a.max_new * group > 16 && row_tiles * a.cache.heads * keys * a.cache.dim / 128 > TJS_LIMIT;
  if (p.tiles) {
    p.rows = TILE_ROWS;
    p.grid = dev.sms;
    p.slots = 2 * p.grid;  // a CTA's first and last segment
    p.target = p.min_chunk = 0;
    p.wide = false;
    return p;
  }
  p.rows = 16;
  const long tiles = row_tiles;
  // Few row tiles are cut so that all pieces run at once, one CTA an SM (pieces: at most target + tiles).
  // Many uneven ones are cut for three waves of smaller CTAs, which even out what one wave does not.
  const bool q8 = a.cache.dtype == TJ_I8 || a.cache.dtype == TJ_E4M3;
  const long items = a.cache.heads * tiles;
  p.wide = items <= dev.sms / 2;
  p.target = static_cast<int>(p.wide ? dev.sms - items : 3L * dev.sms * (q8 ? 3 : 2));
  p.min_chunk = 256;
  p.grid = a.cache.heads * (tiles + 1) + p.target;
  p.slots = p.grid;
  return p;
}

// Raises a kernel's shared-memory limit, once a device (doing so twice is harmless).
template <class K> cudaError_t allow(K kernel, int smem, bool (&ready)[MAX_DEVICES], const Device& dev) {
  if (ready[dev.index]) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  ready[dev.index] = e == cudaSuccess;
  return e;
}
template <class T, int CD, int D, bool WIDE> cudaError_t launch_few(const AttnParams& p, unsigned grid, const Device& dev, cudaStream_t st) {
  using R = Rows<T, CD, D, WIDE>;
  static bool ready[MAX_DEVICES];
  if (const cudaError_t e = allow(attention_rows<T, CD, D, WIDE>, R::SMEM, ready, dev)) return e;
  attention_rows<T, CD, D, WIDE><<<grid, R::THREADS, R::SMEM, st>>>(p);
  return cudaSuccess;
}
template <class T, int CD, int D> cudaError_t launch_dim(const AttnParams& p, const Plan& plan, const Device& dev, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>(plan.grid);
  static bool tiles_ready[MAX_DEVICES];
  if (plan.tiles) {
    constexpr int smem = Tiles<T, CD, D>::SMEM;
    if (const cudaError_t e = allow(attention_tiles<T, CD, D>, smem, tiles_ready, dev)) return e;
    attention_tiles<T, CD, D><<<grid, 512, smem, st>>>(p);
  } else {
    return plan.wide ? launch_few<T, CD, D, true>(p, grid, dev, st) : launch_few<T, CD, D, false>(p, grid, dev, st);
  }
  return cudaSuccess;
}
template <class T, int CD> cudaError_t launch_cache(const AttnParams& p, const Plan& plan, const Device& dev, cudaStream_t st) {
  return p.a.cache.dim == 64 ? launch_dim<T, CD, 64>(p, plan, dev, st) : launch_dim<T, CD, 128>(p, plan, dev, st);
}
template <class T> cudaError_t launch_type(const AttnParams& p, const Plan& plan, const Device& dev, cudaStream_t st) {
  switch (p.a.cache.dtype) {
    case TJ_I8: return launch_cache<T, TJ_I8>(p, plan, dev, st);
    case TJ_E4M3: return launch_cache<T, TJ_E4M3>(p, plan, dev, st);
    default: return launch_cache<T, TJ_BF16>(p, plan, dev, st);
  }
}

int64_t part_bytes(const tj_paged_attention& a, const Plan& p) { return p.slots * p.rows * (a.cache.dim * 4 + 8); }

}  // namespace tjs

extern "C" int tj_b200_paged_attention_workspace(const tj_paged_attention* args, int64_t* workspace_bytes,
                                                 int64_t* counters_count) {
  using namespace tjs;
  const char* name = "tj_b200_paged_attention_workspace";
  if (!args || !workspace_bytes || !counters_count) return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  if (const char* why = attention_fault(*args)) return refuse(TJ_ERR_INVALID, name, why);
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  const Plan need = plan(*args, dev);
  *workspace_bytes = part_bytes(*args, need);
  *counters_count = need.grid;
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
  const Plan how = plan(a, dev);
  if (a.workspace_bytes < part_bytes(a, how) || a.counters_count < how.grid)
    return refuse(TJ_ERR_INVALID, name, "workspace or counters too small");
  if (how.grid > 0x7fffffffL) return refuse(TJ_ERR_INVALID, name, "too many rows");
  AttnParams p;
  p.a = a;
  p.status = dev.status;
  p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.group = static_cast<int>(a.q_heads / a.cache.heads);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.cache.page_size == (1LL << i)) p.page_shift = i;
  p.target = how.target;
  p.min_chunk = how.min_chunk;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + how.slots * how.rows * a.cache.dim);
  p.counters = a.counters;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.dtype == TJ_BF16 ? launch_type<__nv_bfloat16>(p, how, dev, st) : launch_type<__half>(p, how, dev, st);
  if (e != cudaSuccess) return refuse(TJ_ERR_CUDA, name, cudaGetErrorString(e));
  return launched(name);
}
