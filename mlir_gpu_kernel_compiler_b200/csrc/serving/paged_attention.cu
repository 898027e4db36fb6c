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
  const int es = element_size(a.cache.dtype);
  if (a.cache.page_stride * es % 16 || a.cache.slot_stride * es % 16 || a.cache.head_stride * es % 16)
    return "cache rows must start on 16-byte boundaries";
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
  const bool q8 = a.cache.dtype == TJ_I8 || a.cache.dtype == TJ_E4M3;
  // Sizes if every sequence has max_new tokens over 4096 keys, or a window's, as lengths are known to the
  // device only: neither tokens of no sequence nor a table's width decide, so they change no bit either.  Where
  // max_new is not known (above the number of tokens), they are what all tokens can come to, those of no sequence
  // among them, if each sequence has one and some have the rest: 64 single tokens are 64 row tiles, not 64 x 64
  // tokens' (over 4096 keys each, 32 heads on 8 of 128: 193 us for the 237 of the other kernel, in 8 bits 143 for
  // 376; 63 single tokens and a chunk of 512 in 8 bits 323, and 556 if max_new says 512).
  const bool known = a.max_new <= a.tokens;
  const long new_max = std::min(a.max_new, a.tokens), packed = new_max * group;
  const auto tiles_of = [&](long per) {
    const long all = a.batch * ((packed + per - 1) / per), rest = std::max<long>(a.tokens - a.batch, 0) * group;
    return static_cast<double>(known ? all : std::min(all, a.batch * ((group + per - 1) / per) + (rest + per - 1) / per));
  };
  const double row_tiles = tiles_of(16);
  // Tokens of one tile of 16 rows take the kernel of few rows.  More do while it passes over less: it reads
  // the keys once for 16 rows, the other once for 256, but starts, joins and ends in 25 us more (16-bit
  // caches) or 30 (8-bit ones, whose keys it also converts, at four times the cost).  Few rows against many, us:
  //   16-bit, dim 128  1 x 16 tokens over 4096 22, 36   1 x 32 42, 44   1 x 64 61, 56   1 x 256 161, 62
  //                    8 x 16 over 2048 68, 40          16 x 8 over 8192 163, 121
  //   i8, dim 128      1 x 32 over 4096 38, 49          1 x 64 57, 64   1 x 128 86, 64
  //                    8 x 16 over 2048 58, 48          16 x 8 over 8192 135, 190
  //   e4m3, dim 128    1 x 32 over 4096 34, 48          1 x 64 52, 62   1 x 128 78, 63
  //                    8 x 16 over 2048 54, 46          16 x 8 over 8192 118, 175
  //   16-bit, dim 64   1 x 32 over 4096 25, 31          1 x 64 39, 39   1 x 128 59, 40
  // Contexts that are not near 4096 keys are taken for that all the same, and get the slower kernel at both ends:
  //   16-bit, dim 128  1 x 300 over 300 32, 56 (many)   1 x 32 over 32768 254, 71 (few)
  //   i8, dim 128      1 x 300 over 300 31, 63 (many)   1 x 64 over 32768 238, 112 (few)
  const double keys = a.window > 0 ? static_cast<double>(a.window) + (known ? new_max : a.tokens / std::max<long>(a.batch, 1)) : 4096;
  const double pass = a.cache.heads * keys * static_cast<double>(a.cache.dim + 64) / 192;
  const double many_tiles = tiles_of(TILE_ROWS);
  p.tiles = packed > 16 && row_tiles * pass > (q8 ? 500e3 + 3.6 * many_tiles * pass : 250e3 + many_tiles * pass);
  if (p.tiles) {
    p.rows = TILE_ROWS;
    p.grid = std::min(dev.sms, MAX_PARTS);
    p.slots = 2 * p.grid;  // a CTA's first and last segment
    p.target = p.min_chunk = 0;
    p.wide = false;
    return p;
  }
  p.rows = 16;
  // Few row tiles are cut so that all pieces run at once, one CTA an SM (pieces: at most target + tiles).
  // Many uneven ones are cut for three waves of smaller CTAs, which even out what one wave does not.
  // (One token over 777 keys 10.5 us in this way, 11.1 in the other; three over 100003 in i8 56, 87, in e4m3 49, 83.)
  const double items = a.cache.heads * row_tiles;
  p.wide = items <= dev.sms / 2;
  p.target = p.wide ? dev.sms - static_cast<int>(items) : 3 * dev.sms * (q8 ? 3 : 2);
  // Keys of a chunk at least: one token over 4096 keys takes 12.1 us with 256, 12.5 with 128, 14.4 with 512; four
  // over 2000 keys of 8 bits 13.8, 13.8, 16.1.
  p.min_chunk = 256;
  const long tiles = a.q_starts ? a.tokens * group / 16 + a.batch : a.batch * ((group + 15) / 16);  // at the most
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
    join_tiles<T, CD, D><<<dim3(grid, TILE_ROWS / 32), 256, 0, st>>>(p);
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
  p.a.window = std::min<int64_t>(a.window, 0x7fffffff);  // no sequence is longer, and the kernels add to it
  p.status = dev.status;
  p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.group = static_cast<int>(a.q_heads / a.cache.heads);
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a.cache.page_size == (1LL << i)) p.page_shift = i;
  p.target = how.target;
  p.tile_ctas = static_cast<int>(how.grid);
  p.min_chunk = how.min_chunk;
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + how.slots * how.rows * a.cache.dim);
  p.counters = a.counters;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = a.dtype == TJ_BF16 ? launch_type<__nv_bfloat16>(p, how, dev, st) : launch_type<__half>(p, how, dev, st);
  if (e != cudaSuccess) return refuse(TJ_ERR_CUDA, name, cudaGetErrorString(e));
  return launched(name);
}
