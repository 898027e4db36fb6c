// Attention of new tokens over a paged cache: what both kernels share.
//
//   o[i, h] = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i k_j - max),   j visible to i
//
// Token i of a sequence's n new tokens stands at position len - n + i; it sees the keys at
// positions up to its own (causal: else those after it too) and, with a window w, none before the last
// w of its own position and those before it.  The G query
// heads that share a cached head are packed with the tokens into rows r = i * G + g, so a key or a
// value is read once for all of them.
//
// An 8-bit cache holds k = ks * code, v = vs * code with one scale for each (token, head).  The
// codes are exact in bf16 and f16, so they enter the matrix products as they are; ks multiplies the
// score's column, and vs enters the exponent:  t = log2e * scale * ks * (q . code) + log2 vs,
// P = 2^(t - m) with m the running maximum of t, and the sum adds P / vs.  So P, rounded to 16 bits
// for the product with the codes, is at most 1 whatever the scales are.  (The kernel of many rows does so for f16
// queries only: bf16 has f32's range, and P is multiplied by vs.)
#pragma once
#include "serving_common.cuh"

namespace tjs {

struct AttnParams {
  tj_paged_attention a;
  int* status;
  float scale_log2;  // scale * log2 e
  int group;         // query heads of a cached head
  int page_shift;    // log2 page_size, or -1
  int target;        // CTAs that the work is to be cut into, all heads together
  int min_chunk;     // keys of a chunk at least
  float* part_o;     // [grid][rows][dim] sums of P V, not yet divided
  float2* part_ml;   // [grid][rows] (maximum, sum)
  int* counters;     // [grid] chunks done, zero between calls
  int tile_ctas;     // CTAs of the kernel of many rows
};

// log2 vs, held at -80 or above: a row of zeros has vs = 0, and a key whose P = 2^(t - m), or whose part of the sum as m
// moves, underflows f32 (2^-126) has to weigh little.  Beside a key with the value scale v it may be lost below 2^-46 v of
// that key's weight: below f32's rounding up to v = 2^20 (values of 1e8), which is the limit that callers are told.
// Values under 127 * 2^-80 thus come out up to that size.  A NaN (the scale of a row that is not finite) stays one.
TJ_DEV float log2_scale(float vs) { return vs == vs ? fmaxf(__log2f(vs), -80.0f) : vs; }

struct Seq {
  int start, n, len;  // first new token, new tokens, keys
};
TJ_DEV Seq sequence(const AttnParams& p, int b) {
  Seq s;
  const int reach = static_cast<int>(min(p.a.table_width * p.a.cache.page_size, static_cast<int64_t>(0x7fffffff)));
  s.len = max(0, min(p.a.kv_lens[b], reach));
  if (p.a.q_starts) {
    const int t = static_cast<int>(p.a.tokens);
    s.start = min(max(p.a.q_starts[b], 0), t);
    s.n = min(max(p.a.q_starts[b + 1], s.start), t) - s.start;
  } else {
    s.start = b;
    s.n = 1;
  }
  return s;
}

// Whether sequence b's token range is turned round.  Where one is, others overlap: rows of the output would have two
// writers and the work more pieces than were launched, so the whole call does nothing.
TJ_DEV bool descending(const AttnParams& p, int b) { return p.a.q_starts && p.a.q_starts[b] > p.a.q_starts[b + 1]; }
// Records what is wrong with the sequences' numbers (lengths only of those with new tokens); `sequence` clamps them.
// Thread `first` of `threads` looks at every so many.  Not inlined: the registers that the caller's loop gets depend
// on it (64 single tokens over 4096 keys of 8 bits 133 us for 129).
static __device__ __noinline__ void report_sequences(const AttnParams& p, int first, int threads) {
  for (int b = first; b < p.a.batch; b += threads) {
    if (sequence(p, b).n > 0 && (p.a.kv_lens[b] < 0 || p.a.kv_lens[b] > p.a.table_width * p.a.cache.page_size))
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_LENGTH);
    if (p.a.q_starts && (p.a.q_starts[b] < 0 || p.a.q_starts[b + 1] > p.a.tokens || descending(p, b)))
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_STARTS);
  }
}

// keys that some of the tokens [t0, t1] of a sequence see
TJ_DEV void key_range(const AttnParams& p, const Seq& s, int t0, int t1, int& lo, int& hi) {
  hi = p.a.causal ? max(0, min(s.len, s.len - s.n + t1 + 1)) : s.len;
  lo = p.a.window > 0 ? static_cast<int>(max(static_cast<int64_t>(0), s.len - s.n + t0 - p.a.window + 1)) : 0;
  lo = min(lo, hi);
}
// the same of one row's token
TJ_DEV void row_range(const AttnParams& p, const Seq& s, int t, int& lo, int& hi) { key_range(p, s, t, t, lo, hi); }

// A CTA's piece of the work: row tile `tile` of sequence `b`, chunk `c` of its keys, of which `cuts` are launched.
struct Piece {
  int b, tile, c, chunk, cuts;
  bool some;
};

// The work is cut on the device, so that neither lengths nor a plan pass through the host: every
// warp adds up the sequences' (row tiles x keys), divides by the wanted number of CTAs for the
// chunk, and finds the piece of unit `unit` among the sequences' counts.  `per_tile` rows are a
// tile; chunks are multiples of `step` keys.  A tile gets as many pieces as the widest of its sequence could
// need; what key_range then gives of its own keys decides how many of them work.
TJ_DEV Piece find_piece(const AttnParams& p, int unit, int per_tile, int step) {
  const int lane = threadIdx.x & 31;
  const int batch = static_cast<int>(p.a.batch), per = (batch + 31) / 32;
  const int b0 = min(lane * per, batch), b1 = min(b0 + per, batch);
  // under a window a tile's keys reach from its first token's window to its last token, or, without the causal
  // mask, to the sequence's end
  const int tokens_per_tile = (per_tile + p.group - 1) / p.group + 1;
  auto tiles = [&](const Seq& s) { return (s.n * p.group + per_tile - 1) / per_tile; };
  auto span = [&](const Seq& s) {
    return p.a.window > 0 ? static_cast<int>(min(static_cast<int64_t>(s.len), p.a.window + (p.a.causal ? tokens_per_tile : s.n))) : s.len;
  };
  long work = 0;
  bool turned = false;
  for (int b = b0; b < b1; ++b) {
    const Seq s = sequence(p, b);
    turned |= descending(p, b);
    work += static_cast<long>(tiles(s)) * span(s);
  }
  Piece g;
  g.some = false;
  if (__any_sync(0xffffffffu, turned)) return g;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
  // (in f32, rounded up generously: pieces may only become fewer; 64-bit divisions take hundreds of clocks)
  const long want = static_cast<long>(static_cast<float>(work * p.a.cache.heads) / static_cast<float>(p.target) * 1.000001f) + 1;
  // (a chunk of 2^30 keys is any sequence's whole: with max_new far too small `want` may pass 32 bits)
  g.chunk = static_cast<int>((min(max(want, static_cast<long>(p.min_chunk)), 1L << 30) + step - 1) / step * step);
  auto cuts_of = [&](const Seq& s) {
    const int n = span(s) + g.chunk - 1, q = static_cast<int>(__fdividef(static_cast<float>(n), static_cast<float>(g.chunk)));
    return max(1, q + (n - q * g.chunk >= g.chunk) - (n - q * g.chunk < 0));  // the estimate is off by one at the most
  };
  auto count = [&](const Seq& s) { return tiles(s) * cuts_of(s); };
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += count(sequence(p, b));
  int before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  before -= mine;
  const bool owner = unit >= before && unit < before + mine;
  const unsigned who = __ballot_sync(0xffffffffu, owner);
  g.some = who != 0;
  if (!g.some) return g;
  int fb = 0, ft = 0, fc = 0, fn = 1;
  if (owner) {
    int left = unit - before;
    for (int b = b0; b < b1; ++b) {
      const Seq s = sequence(p, b);
      const int cuts = cuts_of(s), n = tiles(s) * cuts;
      if (left < n) {
        fb = b;
        ft = left / cuts;
        fc = left - ft * cuts;
        fn = cuts;
        break;
      }
      left -= n;
    }
  }
  const int src = __ffs(who) - 1;
  g.b = __shfl_sync(0xffffffffu, fb, src);
  g.tile = __shfl_sync(0xffffffffu, ft, src);
  g.c = __shfl_sync(0xffffffffu, fc, src);
  g.cuts = __shfl_sync(0xffffffffu, fn, src);
  return g;
}

TJ_DEV float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// P is made 2^shift times as large before it is rounded to 16 bits, and so is the sum: f16 has no
// normal numbers below 2^-14, and a key whose probability is small can have the larger value.  What is left of the
// type's end: a key's part is off by at most 2^-39 of its value (2^-25 of 2^14), however small its probability.
template <class T> constexpr float P_SHIFT = 0.0f;
template <> constexpr float P_SHIFT<__half> = 14.0f;
// So P = 2^(t - base), and a row's base is what the kernels keep in place of its maximum: the maximum less the shift,
// or the maximum itself where f32's steps at that size (4 at 2^25) make more of the shift than f16 has room for.
TJ_DEV float base_of(float top, float shift) {
  const float b = top - shift;
  return top - b > shift + 1.0f ? top : b;
}

template <class T> TJ_DEV uint32_t pack2(float lo, float hi);
template <> TJ_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return tj_pack_bf16x2(lo, hi); }
template <> TJ_DEV uint32_t pack2<__half>(float lo, float hi) { return tj_pack_f16x2(lo, hi); }

}  // namespace tjs
