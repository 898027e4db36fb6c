// Attention over a paged cache for many rows (chunks of a prompt): a tile is 2 x 128 rows, and the
// products run on the tensor cores through tcgen05 with their sums in TMEM.
//
// What bounds it: a key meets 256 rows, 2 x 256 products for each of its elements, so the cache is
// cheap and the kernel is made of the tensor cores' two products and of 64 exponentials a row and block
// of 64 keys (16 a clock and SM: 512 clocks a row tile).  A row tile's scores of the next block are made
// while its softmax works on this one, in a second buffer; so softmax and tensor cores never wait for
// one another's round trip (with 128 keys a block there is TMEM for one buffer only: 4000 clocks for 128
// keys of both tiles, half of them waiting).  The price is a narrower product for the scores, 49 clocks
// a step of 16 where the tensor cores need 32, as shared memory has to give 6 KB for it: 2590 clocks
// for 128 keys at head dim 128.  Warps (512 threads, one CTA an SM):
//   0-3, 4-7   softmax of row tile 0, 1: a thread is a row.  It reads its 64 scores out of TMEM, keeps a
//              running maximum (moved, and the sums in TMEM rescaled, only when a block exceeds it by
//              more than 2^RAISE) and sum, and writes P over the scores, 16 bits each.
//   8-11       producers of the keys (8, 9) and values (10, 11): a warp brings 32 rows of each block.
//              Pages are looked up one key a lane, rows copied asynchronously in the 128-byte-swizzled
//              layout that the matrix unit reads; 8-bit codes are copied two blocks ahead and made
//              16-bit from there.  Pages may have any size and the cache any strides, as no copy spans
//              two rows.
//   12, 13     issue the matrix instructions of row tile 0, 1: per block P V, then the scores of the
//              block after the next over the P that it has read.  (One warp for both was the bound, 2400
//              clocks a block: a wait for a barrier takes 140 clocks even when it is over, as it queues
//              behind the softmax warps' exponentials.)
//   14         looks the next segment up.
//   15         of the first CTA: records faulty lengths and token ranges.
//
// Measured: 2048 tokens over 16384 bf16 keys, 32 heads of 128 on 8 cached ones, 486 us = 1060 TFLOP/s (65 % of
// the measured matrix rate) in short runs and 554 to 566 us under the board's power limit, where variants that
// need fewer clocks take as long.  Over i8 codes 835 us, over e4m3 761: the conversion is made again by every tile of a
// head, and its instructions and the scales' (two products a score) share the schedulers with the softmax; left
// out, in a timing build, they give 531.  Eight producer warps of 16 rows each were no help (884 us for 820).
//
// The work, (tile, block) pairs of all sequences and heads in a row, is cut into as many equal parts as
// there are SMs (each at least 512 keys): a CTA takes a tile's end, whole tiles and a tile's beginning.
// Parts of one tile are joined, in the tile's order, by a second kernel on all SMs.  (By the CTA that
// ends last, which then reads a part's 131 KB for each: 64 tokens over 4096 keys took 115 us.)
//
// Every wait is bounded (TJ_WAIT_NS): one that runs out raises the CTA's abort flag and the status word.
#pragma once
#include <limits.h>

#include <type_traits>

#include "../kernels/attention_sm100.cuh"
#include "paged_attention.cuh"

namespace tjs {

constexpr int TILE_ROWS = 256, TILE_KEYS = 64, MAX_PARTS = 1024;

// The linear order of the work, in keys x group.  A tile weighs its keys, and one block more for what a
// tile costs by itself.  Positions are cut without 64-bit divisions, which a lone warp takes
// hundreds of clocks for.
struct TileWork {
  long per_head;  // of a sequence: all its tiles
  long base;      // a tile's weight without what grows along the sequence
  int tiles;
  int rows;
  bool grows;     // causal without a window: tile t sees 256 (t + 1) / group tokens more
  TJ_DEV long before(int t) const {  // weight of the tiles before t
    return base * t + (grows ? static_cast<long>(TILE_ROWS / 2) * t * (t + 1) : 0);
  }
};
TJ_DEV TileWork tile_work(const AttnParams& p, const Seq& s) {
  TileWork w;
  w.rows = s.n * p.group;
  w.tiles = (w.rows + TILE_ROWS - 1) / TILE_ROWS;
  w.grows = p.a.causal && p.a.window == 0;
  long span = s.len;
  if (w.grows)
    span = max(s.len - s.n, 0);
  else if (p.a.window > 0)
    span = min(span, static_cast<long>(p.a.window) + (p.a.causal ? TILE_ROWS / p.group : s.n));
  w.base = p.group * (span + TILE_KEYS);
  w.per_head = w.before(w.tiles);
  return w;
}

struct TilePart {
  Seq s;
  int b, head, tile;
  long start, weight;  // of the tile, in the linear order
};

TJ_DEV long total_work(const AttnParams& p) {
  const int lane = threadIdx.x & 31;
  long mine = 0;
  bool turned = false;
  for (int b = lane; b < p.a.batch; b += 32) {
    mine += tile_work(p, sequence(p, b)).per_head;
    turned |= descending(p, b);
  }
  if (__any_sync(0xffffffffu, turned)) return 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine * p.a.cache.heads;
}

// The work in `parts` equal parts: part c begins at begin(c).
struct Cut {
  long total, parts, share, rest;
  TJ_DEV Cut(long t, long n) : total(t), parts(n), share(t / n), rest(t - share * n) {}
  TJ_DEV long begin(long c) const { return share * c + min(c, rest); }
  TJ_DEV long part_of(long pos) const {
    const long wide = (share + 1) * rest;
    return pos < wide ? pos / (share + 1) : rest + (pos - wide) / share;
  }
};
// As many parts as CTAs, of 512 keys at the least.
TJ_DEV Cut cut_work(const AttnParams& p, long total, int ctas) {
  return Cut(total, min(static_cast<long>(ctas), max(1L, total / (512L * p.group))));
}
// blocks that a tile with the key range [lo, hi) goes through
TJ_DEV int tile_key_blocks(int lo, int hi) { return max(1, (hi + TILE_KEYS - 1) / TILE_KEYS - lo / TILE_KEYS); }
// How many of a tile's `blocks` key blocks lie before place `a` of its weight: roundings to nearest
// keep the order, so neighbours that ask with the same place agree, and a = weight gives all.
TJ_DEV int blocks_before(long a, long weight, int blocks) {
  return static_cast<int>(static_cast<float>(blocks) * __fdiv_rn(static_cast<float>(a), static_cast<float>(weight)));
}

// the tile at `pos` of the linear order (0 <= pos < total), found by a warp
TJ_DEV TilePart find_tile(const AttnParams& p, long pos) {
  const int lane = threadIdx.x & 31;
  TilePart g;
  long done = 0;
  g.b = -1;
  for (int b0 = 0; b0 < p.a.batch; b0 += 32) {
    const int b = b0 + lane;
    const long mine = b < p.a.batch ? tile_work(p, sequence(p, b)).per_head * p.a.cache.heads : 0;
    long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned in = __ballot_sync(0xffffffffu, pos < done + upto);
    if (in) {
      const int src = __ffs(in) - 1;
      g.b = b0 + src;
      g.start = done + __shfl_sync(0xffffffffu, upto - mine, src);
      break;
    }
    done += __shfl_sync(0xffffffffu, upto, 31);
  }
  g.s = sequence(p, g.b);
  const TileWork w = tile_work(p, g.s);
  const long in_seq = pos - g.start;
  g.head = static_cast<int>(static_cast<float>(in_seq) / static_cast<float>(w.per_head));  // off by one at the most
  while (g.head > 0 && in_seq < g.head * w.per_head) --g.head;
  while (in_seq >= (g.head + 1) * w.per_head) ++g.head;
  const long in_head = in_seq - g.head * w.per_head;
  int lo = 0, hi = w.tiles - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (w.before(mid) <= in_head)
      lo = mid;
    else
      hi = mid - 1;
  }
  g.tile = lo;
  g.start += g.head * w.per_head + w.before(lo);
  g.weight = w.before(lo + 1) - w.before(lo);
  return g;
}

TJ_DEV void cp_async16(uint32_t dst, const void* src, bool on) {
  const int bytes = on ? 16 : 0;  // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TJ_DEV void cp_async4(uint32_t dst, const void* src, bool on) {
  const int bytes = on ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TJ_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> TJ_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// 16 columns of a warp's 32 lanes out of TMEM
TJ_DEV void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
template <int N> TJ_DEV void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> TJ_DEV void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
TJ_DEV void st_shared16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// a row's place in a swizzled operand of `dim` columns: panels of 64 columns, 128 bytes a row, the
// 16-byte pieces of a row permuted by its number
TJ_DEV uint32_t swizzled(int rows, int row, int piece) {
  return static_cast<uint32_t>((piece >> 3) * rows * 128 + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

// A producer warp's rows of 8-bit codes as 16-bit floats into a swizzled operand.
template <class T, int CD, int D, int N>
TJ_DEV void store_rows(uint32_t dst, const uint4 (&raw)[N], int row0) {
  constexpr int LPR = D / 16, PER = 32 / LPR;
  const int lane = threadIdx.x & 31, piece = lane % LPR;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int r = row0 + i * PER + lane / LPR;
    uint32_t h[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = e == 0 ? raw[i].x : e == 1 ? raw[i].y : e == 2 ? raw[i].z : raw[i].w;
      codes4<T, CD>(x, h[e >> 1][(e & 1) * 2], h[e >> 1][(e & 1) * 2 + 1]);
    }
    // at head dim 128 a row's lanes reach both panels, whose banks are the same: the upper half
    // stores its odd piece first
    const bool swap = D == 128 && piece >= LPR / 2;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int o = swap ? e ^ 1 : e;
      st_shared16(dst + swizzled(TILE_KEYS, r, piece * 2 + o), swap ? h[e ^ 1][0] : h[e][0], swap ? h[e ^ 1][1] : h[e][1],
                  swap ? h[e ^ 1][2] : h[e][2], swap ? h[e ^ 1][3] : h[e][3]);
    }
  }
}

TJ_DEV uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <class T, int CD, int D> struct Tiles {
  static constexpr bool Q8 = CD == TJ_I8 || CD == TJ_E4M3;
  static constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  // An 8-bit cache's value scales: bf16 has f32's range, so P is simply multiplied by vs before it is
  // rounded (arrays ks, vs); f16 has vs in the exponent (arrays ks, log2 vs, 1 / vs).  Every softmax
  // thread reads these arrays for every block, so one fewer counts: eight sequences' chunks over i8 codes take
  // 371 us with bf16 products, and 409 with f16 ones, whose codes take fewer instructions.
  static constexpr bool MUL_V = Q8 && BF, EXP_V = Q8 && !BF;
  static constexpr int ARRAYS = MUL_V ? 2 : EXP_V ? 3 : 0;
  static constexpr int STAGES = D == 64 ? 8 : Q8 ? 3 : 4;
  // 8-bit codes and scales wait in shared memory before they are converted, this many blocks of them
  static constexpr int RAWS = Q8 ? 3 : 0;
  static constexpr uint32_t RAW_SCALE = 2 * TILE_KEYS * D, RAW_BYTES = RAW_SCALE + 2 * TILE_KEYS * 4;
  // Scale rows outlive their block's operands: a tile's softmax is up to two blocks behind its scores.
  // Block j + SCALES takes over from block j when the scores of block j + 2 are made, which follow its P.
  static constexpr int SCALES = STAGES + 2;
  static constexpr uint32_t Q_BYTES = 128 * D * 2, KV_BYTES = TILE_KEYS * D * 2;
  static constexpr int SMEM = 1024 + 2 * Q_BYTES + 2 * STAGES * KV_BYTES + SCALES * ARRAYS * TILE_KEYS * 4 + RAWS * RAW_BYTES + 768;
  static_assert(SMEM <= 232448, "shared memory");
  // registers of a softmax, producer and other thread; at launch all have 128
  static constexpr int REGS_S = 152, REGS_P = 104, REGS_M = 104;
  static_assert(256 * REGS_S + 128 * REGS_P + 128 * REGS_M <= 512 * 128, "no more than the block was launched with");
  // TMEM columns: scores of tile t, buffer b at (2 t + b) 64 (P, 32 columns, over them); O_t at 256 + t D
  static constexpr uint32_t TMEM = 512;
  static constexpr float SHIFT = P_SHIFT<T> > 11.0f ? 11.0f : P_SHIFT<T>;  // with RAISE: P < 2^16
  static constexpr float RAISE = P_SHIFT<T> > 0.0f ? 4.0f : 8.0f;
};

// A row's P = 2^(x c + b) (8-bit caches: x + b) of a block: summed into ll, rounded to 16 bits and
// written over the scores at tS.
template <class T, class C>
TJ_DEV void probabilities(const float (&x)[64], uint64_t c, uint64_t b, const float* sc, uint64_t& ll, uint32_t tS) {
  using namespace tja;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    uint32_t pk[16];
    float4 vs = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int i = g * 32 + 2 * k;
      const uint64_t xx = f2_pack(x[i], x[i + 1]);
      const uint64_t e = C::Q8 ? f2_add(xx, b) : f2_fma(xx, c, b);
      float e0, e1;
      f2_unpack(e, e0, e1);
      e0 = exp2_fast(e0);
      e1 = exp2_fast(e1);
      if constexpr (C::EXP_V) {
        if (k % 2 == 0) vs = *reinterpret_cast<const float4*>(sc + 2 * TILE_KEYS + i);  // 1 / vs
        ll = f2_fma(f2_pack(e0, e1), k % 2 ? f2_pack(vs.z, vs.w) : f2_pack(vs.x, vs.y), ll);
      } else {
        ll = f2_add(ll, f2_pack(e0, e1));
      }
      if constexpr (C::MUL_V) {
        if (k % 2 == 0) vs = *reinterpret_cast<const float4*>(sc + TILE_KEYS + i);
        f2_unpack(f2_mul(f2_pack(e0, e1), k % 2 ? f2_pack(vs.z, vs.w) : f2_pack(vs.x, vs.y)), e0, e1);
      }
      pk[k] = pack2<T>(e0, e1);
    }
    tmem_st16(tS + 16 * g, pk);
  }
}

// What a CTA does between two of its barriers: blocks of one tile.
struct Segment {
  Seq s;
  int b, head;
  int r0, rows;     // first packed row of the tile, rows of it
  int lo, hi;       // keys that some row sees
  int key0, nb;     // first key and number of blocks of this segment (0: no segment)
  int all;          // blocks of the tile
  int later;        // the tile began in an earlier part
};

// A CTA's shared memory.
template <class T, int CD, int D> struct TilesShared {
  using C = Tiles<T, CD, D>;
  static constexpr uint32_t Q = 0, K = Q + 2 * C::Q_BYTES, V = K + C::STAGES * C::KV_BYTES, SCALE = V + C::STAGES * C::KV_BYTES,
                            RAW = SCALE + C::SCALES * C::ARRAYS * TILE_KEYS * 4, BARS = RAW + C::RAWS * C::RAW_BYTES, Q_FULL = BARS, K_FULL = Q_FULL + 8,
                            V_FULL = K_FULL + 8 * C::STAGES, K_EMPTY = V_FULL + 8 * C::STAGES, V_EMPTY = K_EMPTY + 8 * C::STAGES,
                            S_FULL = V_EMPTY + 8 * C::STAGES,  // [2 tiles][2 buffers]
                            P_READY = S_FULL + 32,             // [2 tiles][2 buffers]
                            PV_DONE = P_READY + 32,            // [2 tiles][2 buffers]
                            SC_FULL = PV_DONE + 32,            // [SCALES], 8-bit caches
                            DRAIN = SC_FULL + 8 * C::SCALES, SLOT = DRAIN + 16, ABORT = SLOT + 4,
                            SEGMENT = (ABORT + 4 + 15) / 16 * 16, END = SEGMENT + 2 * sizeof(Segment);
  static_assert(END + 1024 <= C::SMEM, "shared memory");
  uint8_t* base;
  TJ_DEV explicit TilesShared(uint8_t* raw) {
    base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  }
  TJ_DEV uint32_t at(uint32_t offset) const { return tjg::smem_u32(base) + offset; }
  TJ_DEV float* scales(int it) const {  // [ARRAYS][64]: ks, vs or log2 vs, 1 / vs
    return reinterpret_cast<float*>(base + SCALE) + (it % C::SCALES) * C::ARRAYS * TILE_KEYS;
  }
  TJ_DEV volatile int* abort_flag() const { return reinterpret_cast<volatile int*>(base + ABORT); }
  TJ_DEV volatile uint32_t* tmem_slot() const { return reinterpret_cast<volatile uint32_t*>(base + SLOT); }
  // volatile: read where it is needed, not kept in registers over the blocks
  TJ_DEV volatile Segment& segment(int seg) const { return reinterpret_cast<volatile Segment*>(base + SEGMENT)[seg & 1]; }
  // Several barriers at once: the polls, each some 140 clocks behind the softmax warps' exponentials, overlap.
  TJ_DEV bool wait3(uint32_t b0, int ph0, uint32_t b1, int ph1, uint32_t b2, int ph2, const AttnParams& p, int site) const {
    const bool x = tjg::mbar_try_wait(at(b0), ph0 & 1), y = tjg::mbar_try_wait(at(b1), ph1 & 1), z = tjg::mbar_try_wait(at(b2), ph2 & 1);
    if (__all_sync(0xffffffffu, x & y & z)) return true;
    return wait(b0, ph0, p, site) && wait(b1, ph1, p, site + 1) && wait(b2, ph2, p, site + 2);
  }
  TJ_DEV bool wait(uint32_t bar, int phase, const AttnParams& p, int site) const {
    return tjg::mbar_wait_warp(at(bar), static_cast<uint32_t>(phase) & 1u, abort_flag(), p.status, OP_ATTENTION * 16 + site);
  }
};

// The next segment at or after `pos` (moved on), by a whole warp.
TJ_DEV void next_segment(const AttnParams& p, long& pos, long to, volatile Segment& out) {
  Segment g;
  g.nb = 0;
  while (pos < to && g.nb == 0) {
    const TilePart w = find_tile(p, pos);
    const long a0 = pos - w.start, a1 = min(w.weight, to - w.start);
    pos = w.start + a1;
    g.s = w.s;
    g.b = w.b;
    g.head = w.head;
    g.r0 = w.tile * TILE_ROWS;
    g.rows = min(TILE_ROWS, w.s.n * p.group - g.r0);
    key_range(p, w.s, g.r0 / p.group, (g.r0 + g.rows - 1) / p.group, g.lo, g.hi);
    const int first = g.lo / TILE_KEYS;
    g.all = tile_key_blocks(g.lo, g.hi);
    const int j0 = blocks_before(a0, w.weight, g.all);
    g.nb = blocks_before(a1, w.weight, g.all) - j0;
    g.key0 = (first + j0) * TILE_KEYS;
    g.later = a0 > 0;
  }
  if ((threadIdx.x & 31) == 0) {
    if (g.nb) {
      out.s.start = g.s.start;
      out.s.n = g.s.n;
      out.s.len = g.s.len;
      out.b = g.b;
      out.head = g.head;
      out.r0 = g.r0;
      out.rows = g.rows;
      out.lo = g.lo;
      out.hi = g.hi;
      out.key0 = g.key0;
      out.all = g.all;
      out.later = g.later;
    }
    out.nb = g.nb;
  }
  __syncwarp();
}

// (token, query head) of packed row r of a sequence
TJ_DEV void row_of(const AttnParams& p, int head, int r, int& tok, int& hd) {
  tok = r / p.group;
  hd = head * p.group + r - tok * p.group;
}

// The end of a segment, by every thread of the CTA: false if a wait ran out.
template <class T, int CD, int D> TJ_DEV bool end_segment(const TilesShared<T, CD, D>& sh) {
  __syncwarp();
  __syncthreads();
  tjg::tc_fence_after();
  return *sh.abort_flag() == 0;
}

// Joins the tiles that were cut: CTA (c, y) the rows 32 y .. 32 y + 31 of the tile that begins in part c and
// goes on in part c + 1, if there is one.
template <class T, int CD, int D> __global__ void __launch_bounds__(256) join_tiles(const __grid_constant__ AttnParams p) {
  __shared__ int s_slots[MAX_PARTS];
  __shared__ int s_whole;
  const long total = total_work(p);
  if (total == 0) return;
  const Cut cut = cut_work(p, total, p.tile_ctas);
  const int c0 = blockIdx.x;
  if (c0 + 1 >= cut.parts) return;
  const long from = cut.begin(c0), to = cut.begin(c0 + 1);
  const TilePart w = find_tile(p, to - 1);
  if (w.start < from || w.start + w.weight <= to) return;
  const int r0 = w.tile * TILE_ROWS, rows = min(TILE_ROWS, w.s.n * p.group - r0);
  if (static_cast<int>(blockIdx.y) * 32 >= rows) return;
  int lo, hi;
  key_range(p, w.s, r0 / p.group, (r0 + rows - 1) / p.group, lo, hi);
  const int all = tile_key_blocks(lo, hi), n = static_cast<int>(cut.part_of(w.start + w.weight - 1)) - c0 + 1;
  if (threadIdx.x == 0) s_whole = 0;
  __syncthreads();
  // where each part was left (-1: it had no block)
  for (int i = threadIdx.x; i < n; i += 256) {
    const long b0 = max(0L, cut.begin(c0 + i) - w.start), b1 = min(w.weight, cut.begin(c0 + i + 1) - w.start);
    const int blocks = blocks_before(b1, w.weight, all) - blocks_before(b0, w.weight, all);
    s_slots[i] = blocks == 0 ? -1 : 2 * (c0 + i) + (i > 0 ? 0 : 1);
    if (blocks == all) s_whole = 1;  // it fell to one part after all, which has stored it
  }
  __syncthreads();
  if (s_whole) return;
  constexpr int V4 = D / 4;
  for (int e = threadIdx.x; e < 32 * V4; e += 256) {
    const int r = blockIdx.y * 32 + e / V4, col = e % V4 * 4;
    if (r >= rows) break;
    float best = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int GO = 4;  // parts whose loads are in flight together
    for (int i = 0; i < n; i += GO) {
      float2 ml[GO];
      float4 v[GO];
#pragma unroll
      for (int k = 0; k < GO; ++k) {
        const int at = i + k < n ? s_slots[i + k] : -1;
        const long slot = static_cast<long>(max(at, 0)) * TILE_ROWS + r;
        ml[k] = __ldcg(p.part_ml + slot);
        v[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + col));
        if (at < 0) ml[k].x = -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < GO; ++k) {
        if (ml[k].x == -INFINITY) continue;
        const float next = fmaxf(best, ml[k].x), f = exp2_fast(best - next), g = exp2_fast(ml[k].x - next);
        acc = make_float4(acc.x * f + v[k].x * g, acc.y * f + v[k].y * g, acc.z * f + v[k].z * g, acc.w * f + v[k].w * g);
        sum = sum * f + ml[k].y * g;
        best = next;
      }
    }
    const bool none = best == -INFINITY;
    const float inv = none ? 0.0f : 1.0f / sum;
    int tok, hd;
    row_of(p, w.head, r0 + r, tok, hd);
    tok += w.s.start;
    uint2 y;
    y.x = pack2<T>(none ? 0.0f : acc.x * inv, none ? 0.0f : acc.y * inv);
    y.y = pack2<T>(none ? 0.0f : acc.z * inv, none ? 0.0f : acc.w * inv);
    *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + tok * p.a.out_token + hd * p.a.out_head + col) = y;
    if (p.a.lse && col == 0)
      p.a.lse[static_cast<long>(tok) * p.a.q_heads + hd] = none ? -INFINITY : (best + log2f(sum)) * 0.69314718055994531f;
  }
}

// ---- producers: the queries of a segment, then its keys and values block by block ------------------------------
template <class T, int CD, int D>
TJ_DEV void produce(const AttnParams& p, const TilesShared<T, CD, D>& sh, int seg, int blocks) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  using S = TilesShared<T, CD, D>;
  constexpr int STAGES = C::STAGES, ES = C::Q8 ? 1 : 2;
  volatile Segment& g = sh.segment(seg);
  const int warp = (threadIdx.x >> 5) - 8, tid = threadIdx.x - 256, lane = threadIdx.x & 31;
  const bool keys = warp < 2;         // this warp brings keys, or values
  const int row0 = (warp & 1) * 32;  // its rows of a block
  const int nb = g.nb, key0 = g.key0 + row0, lo = g.lo, hi = g.hi, head = g.head;
  {
    constexpr int LPR = D / 8;  // 16-byte pieces of a row
    const int piece = tid % LPR, rows = g.rows, r0 = g.r0, first_token = g.s.start, last = rows > 128 ? 256 : 128;
    for (int r = tid / LPR; r < last; r += 128 / LPR) {
      int tok, hd;
      row_of(p, head, r0 + (r < rows ? r : 0), tok, hd);
      const T* src = static_cast<const T*>(p.a.q) + (first_token + tok) * p.a.q_token + hd * p.a.q_head + piece * 8;
      cp_async16(sh.at(S::Q) + (r >> 7) * C::Q_BYTES + swizzled(128, r & 127, piece), src, r < rows);
    }
    cp_async_commit();
  }
  const int* table = p.a.page_table + g.b * p.a.table_row;
  const char* base = static_cast<const char*>(keys ? p.a.cache.k : p.a.cache.v) + head * p.a.cache.head_stride * ES;
  const uint32_t full = keys ? S::K_FULL : S::V_FULL, empty = keys ? S::K_EMPTY : S::V_EMPTY, dst0 = sh.at(keys ? S::K : S::V);
  // This lane's key of block j: its page (looked up a block before it is used), then the byte offset
  // of its row and its place among the scales (-1: not there).
  const int page_size = static_cast<int>(p.a.cache.page_size);
  int next_page;
  bool next_there;  // a look-up's key is one of the tile's (what is looked up is not touched before it is used)
  auto look_up = [&](int j) {
    const int key = key0 + j * TILE_KEYS + lane;
    next_there = j < nb && key >= lo && key < hi;
    if (next_there) next_page = table[p.page_shift >= 0 ? key >> p.page_shift : key / page_size];
  };
  long off, soff;
  auto place = [&](int j) {  // what was looked up last, for block j
    off = soff = -1;
    if (!next_there) return;
    const int page = next_page;
    if (page >= 0 && page < p.a.cache.pages) {
      const int key = key0 + j * TILE_KEYS + lane;
      const int slot = p.page_shift >= 0 ? key & (page_size - 1) : key % page_size;
      off = (page * p.a.cache.page_stride + slot * p.a.cache.slot_stride) * ES;
      if (C::Q8) soff = page * p.a.cache.scale_page + slot * p.a.cache.scale_slot + head * p.a.cache.scale_head;
    } else {
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_PAGE);
    }
  };
  auto arrive = [&](uint32_t bar) {
    fence_proxy_async_smem();
    mbar_arrive(sh.at(bar));
  };
  auto announce = [&](int it) {
#ifdef TJ_TEST_STALL_FIRST_LOAD
    // failure-path test build only: the first keys never arrive, so the wait for them runs out
    if (it == 0 && keys) return;
#endif
    arrive(full + 8 * (it % STAGES));
  };
  look_up(0);
  place(0);
  look_up(1);
  if constexpr (!C::Q8) {
    constexpr int LPR = D / 8, PER = 32 / LPR;  // lanes of a row, rows of a warp's instruction
    const int piece = lane % LPR;
    for (int j = 0; j < nb; ++j) {
      const int it = blocks + j, s = it % STAGES;
      if (!sh.wait(empty + 8 * s, it / STAGES + 1, p, 5)) break;
      const uint32_t dst = dst0 + s * C::KV_BYTES;
#pragma unroll
      for (int i = 0; i < 32 / PER; ++i) {
        const int r = i * PER + lane / LPR;
        const long ro = __shfl_sync(0xffffffffu, off, r);
        cp_async16(dst + swizzled(TILE_KEYS, row0 + r, piece), base + (ro < 0 ? 0 : ro) + piece * 16, ro >= 0);
      }
      cp_async_commit();
      cp_async_wait<1>();  // the copy before this one is there
      if (j == 0)
        arrive(S::Q_FULL);
      else
        announce(it - 1);
      place(j + 1);
      look_up(j + 2);
    }
    cp_async_wait<0>();
    if (!*sh.abort_flag()) announce(blocks + nb - 1);
  } else {
    constexpr int LPR = D / 16, PER = 32 / LPR, N = 32 / PER;
    const int piece = lane % LPR;  // 16 codes: two pieces of the 16-bit row
    // The codes are copied asynchronously two blocks ahead: each thread those that it will convert itself, so
    // that only it has to wait for them.  (Loaded one block ahead into registers, a block took 3200 clocks.)
    const uint32_t raw0 = S::RAW + (warp * N * 32 + lane) * 16, scale0 = S::RAW + C::RAW_SCALE + (row0 + lane) * 4;
    auto load = [&](int j) {  // of block j, whose place is known; every call commits one group
      const uint32_t slot = static_cast<uint32_t>(j % C::RAWS) * C::RAW_BYTES;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const long ro = __shfl_sync(0xffffffffu, off, i * PER + lane / LPR);
        if (j < nb) cp_async16(sh.at(raw0 + slot + i * 512), base + (ro < 0 ? 0 : ro) + piece * 16, ro >= 0);
      }
      if (keys && j < nb) {  // the keys' producers bring both scales
        cp_async4(sh.at(scale0 + slot), p.a.cache.k_scale + (soff < 0 ? 0 : soff), soff >= 0);
        cp_async4(sh.at(scale0 + slot + TILE_KEYS * 4), p.a.cache.v_scale + (soff < 0 ? 0 : soff), soff >= 0);
      }
      cp_async_commit();
      place(j + 1);
      look_up(j + 2);
    };
    load(0);
    load(1);
    for (int j = 0; j < nb; ++j) {
      const int it = blocks + j, s = it % STAGES;
      load(j + 2);
      cp_async_wait<2>();  // block j is there, and the queries
      if (j == 0) arrive(S::Q_FULL);
      if (!sh.wait(empty + 8 * s, it / STAGES + 1, p, 5)) break;
      const uint32_t slot = static_cast<uint32_t>(j % C::RAWS) * C::RAW_BYTES;
      if (keys) {
        const float ks = *reinterpret_cast<const float*>(sh.base + scale0 + slot);
        const float vs = *reinterpret_cast<const float*>(sh.base + scale0 + slot + TILE_KEYS * 4);
        float* sc = sh.scales(it) + row0 + lane;
        sc[0] = ks * p.scale_log2;
        if constexpr (C::MUL_V) sc[TILE_KEYS] = vs;
        if constexpr (C::EXP_V) {
          const float lv = log2_scale(vs);
          sc[TILE_KEYS] = lv;
          sc[2 * TILE_KEYS] = exp2_fast(-lv);
        }
        mbar_arrive(sh.at(S::SC_FULL + 8 * (it % C::SCALES)));
      }
      uint4 raw[N];
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = *reinterpret_cast<const uint4*>(sh.base + raw0 + slot + i * 512);
      store_rows<T, CD, D>(dst0 + s * C::KV_BYTES, raw, row0);
      announce(it);
    }
    cp_async_wait<0>();
  }
}

// ---- matrix instructions -----------------------------------------------------------------------------------------
// Four steps of 16 of the scores' product, both operands K-major: 32 bytes a step.
TJ_DEV void umma_scores4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 a, b;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
      " add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n"
      " add.s64 a, %1, 4;\n add.s64 b, %2, 4;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n"
      " add.s64 a, %1, 6;\n add.s64 b, %2, 6;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, 1;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Four steps of 16 keys of P V: P 8 columns of TMEM a step, V 16 rows of 128 bytes.
TJ_DEV void umma_values4(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 b;\n .reg .b32 a;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      " add.s32 a, %1, 8;\n add.s64 b, %2, 128;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n"
      " add.s32 a, %1, 16;\n add.s64 b, %2, 256;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n"
      " add.s32 a, %1, 24;\n add.s64 b, %2, 384;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, 1;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Row tile t's products.  blocks: key blocks before this segment; tile_blocks: those of them that the tile had.
// A stage of keys or values is free when both tiles are done with it: two arrivals, both by tile 0's
// warp where there is no tile 1.
template <class T, int CD, int D>
TJ_DEV void multiply(const AttnParams& p, const TilesShared<T, CD, D>& sh, uint32_t tmem, int seg, int t, int blocks, int tile_blocks) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  using S = TilesShared<T, CD, D>;
  constexpr int STAGES = C::STAGES;
  constexpr uint32_t IDESC_S = idesc_f16(C::BF, 128, TILE_KEYS, false, false), IDESC_O = idesc_f16(C::BF, 128, D, false, true);
  const int nb = sh.segment(seg).nb;
  const bool alone = sh.segment(seg).rows <= 128;
  const uint64_t dq = desc_sw128(sh.at(S::Q) + t * C::Q_BYTES, 16, 1024), dk = desc_sw128(sh.at(S::K), 16, 1024),
                 dv = desc_sw128(sh.at(S::V), TILE_KEYS * 128, 1024);
  const uint32_t tS = tmem + t * 128, tO = tmem + 256 + t * D;
  const uint32_t s_full = sh.at(S::S_FULL + 16 * t), pv_done = sh.at(S::PV_DONE + 16 * t);
  auto release = [&](uint32_t bar) {
    umma_commit_elect(bar);
    if (alone) umma_commit_elect(bar);
  };
  bool issued = false;
  auto scores = [&](int j) {
    const int buf = (tile_blocks + j) & 1, s = (blocks + j) % STAGES;
    const uint64_t b = dk + ((s * C::KV_BYTES) >> 4);
#pragma unroll
    for (int k = 0; k < D / 64; ++k)
      umma_scores4(tS + buf * 64, dq + k * (128 * 128 >> 4), b + k * (TILE_KEYS * 128 >> 4), IDESC_S, k > 0);
    umma_commit_elect(s_full + 8 * buf);
    release(sh.at(S::K_EMPTY + 8 * s));
    issued = true;
  };
  bool ok = sh.wait(S::Q_FULL, seg, p, 7);
  for (int j = 0; j < min(nb, 2) && ok; ++j) {
    ok = sh.wait(S::K_FULL + 8 * ((blocks + j) % STAGES), (blocks + j) / STAGES, p, 8);
    if (!ok) break;
    tc_fence_after();
    scores(j);
  }
  for (int j = 0; j < nb && ok; ++j) {
    const int it = blocks + j, s = it % STAGES, use = tile_blocks + j, buf = use & 1;
    const int ahead = j + 2 < nb ? it + 2 : it;  // keys that have arrived stand for none
    ok = sh.wait3(S::K_FULL + 8 * (ahead % STAGES), ahead / STAGES, S::V_FULL + 8 * s, it / STAGES, S::P_READY + 8 * (2 * t + buf), use >> 1, p, 8);
    if (!ok) break;
    tc_fence_after();
    umma_values4(tO, tS + buf * 64, dv + ((s * C::KV_BYTES) >> 4), IDESC_O, j > 0);
    if (j + 2 < nb) scores(j + 2);
    umma_commit_elect(pv_done + 8 * buf);
    release(sh.at(S::V_EMPTY + 8 * s));
  }
  if (!ok && issued) {
    umma_commit_elect(sh.at(S::DRAIN + 8 * t));
    volatile int no_abort = 0;
    mbar_wait_warp(sh.at(S::DRAIN + 8 * t), 0, &no_abort, p.status, OP_ATTENTION * 16 + 11, 200000000ull);
  }
}

// ---- softmax -------------------------------------------------------------------------------------------------------
// tile_blocks: blocks of this warp's row tile before the segment
template <class T, int CD, int D>
TJ_DEV void softmax(const AttnParams& p, const TilesShared<T, CD, D>& sh, uint32_t tmem, int seg, int blocks, int tile_blocks) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  using S = TilesShared<T, CD, D>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = warp >> 2, q = warp & 3, r = t * 128 + q * 32 + lane;
  const uint32_t lanes = tmem + (static_cast<uint32_t>(q * 32) << 16);
  const uint32_t tO = lanes + 256 + t * D;
  volatile Segment& g = sh.segment(seg);
  const int nb = g.nb;
  int rlo, rhi;
  {
    Seq s;
    s.start = g.s.start;
    s.n = g.s.n;
    s.len = g.s.len;
    row_range(p, s, (g.r0 + min(r, g.rows - 1)) / p.group, rlo, rhi);
  }
  // keys that every row of this warp sees need no mask; from here on relative to the segment's first key
  rlo -= g.key0;
  rhi -= g.key0;
  int clo = __reduce_max_sync(0xffffffffu, rlo);
  const int chi = __reduce_min_sync(0xffffffffu, rhi);
  float base = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  // Scores of a 16-bit cache go into P by one fused step from their unscaled form.  Where f32's steps are no longer small
  // (1/8 at 2^20), the product that was not rounded is as much off the base, which was, and P with it: by more than the
  // 16-bit types and in the end f32 can hold.  From there on (the same for the warp, clo FAR) products are rounded first.
  constexpr int FAR = INT_MAX;
  float c = C::Q8 ? 1.0f : p.scale_log2;
  bool ok = true;
  for (int j = 0; j < nb; ++j) {
    const int it = blocks + j, use = tile_blocks + j, kb = j * TILE_KEYS;
    const uint32_t tS = lanes + (2 * t + (use & 1)) * 64;
    ok = sh.wait(S::S_FULL + 8 * (2 * t + (use & 1)), use >> 1, p, 12);
    if (C::Q8 && ok) ok = sh.wait(S::SC_FULL + 8 * (it % C::SCALES), it / C::SCALES, p, 15);
    if (!ok) break;
    tc_fence_after();
    uint32_t raw[64];
    tja::tmem_ld64(tS, raw);
    float x[64];
#pragma unroll
    for (int i = 0; i < 64; ++i) x[i] = __uint_as_float(raw[i]);
    const float* sc = sh.scales(it);
    if constexpr (C::Q8) {
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const float4 k = *reinterpret_cast<const float4*>(sc + i);
        uint64_t a = tja::f2_pack(x[i], x[i + 1]), b = tja::f2_pack(x[i + 2], x[i + 3]);
        if constexpr (C::EXP_V) {
          const float4 v = *reinterpret_cast<const float4*>(sc + TILE_KEYS + i);
          a = tja::f2_fma(a, tja::f2_pack(k.x, k.y), tja::f2_pack(v.x, v.y));
          b = tja::f2_fma(b, tja::f2_pack(k.z, k.w), tja::f2_pack(v.z, v.w));
        } else {
          a = f2_mul(a, tja::f2_pack(k.x, k.y));
          b = f2_mul(b, tja::f2_pack(k.z, k.w));
        }
        tja::f2_unpack(a, x[i], x[i + 1]);
        tja::f2_unpack(b, x[i + 2], x[i + 3]);
      }
    }
    const bool masked = kb < clo || kb + TILE_KEYS > chi;  // the same for the warp
    if (masked) {
      const int a = rlo - kb, b = rhi - kb;
      if (!C::Q8 && clo == FAR) {
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] *= p.scale_log2;
      }
#pragma unroll
      for (int i = 0; i < 64; ++i)
        if (i < a || i >= b) x[i] = -INFINITY;
    }
    float h0 = x[0], h1 = x[1], h2 = x[2], h3 = x[3];
#pragma unroll
    for (int i = 4; i < 60; i += 8) {
      h0 = tja::fmax3(h0, x[i], x[i + 4]);
      h1 = tja::fmax3(h1, x[i + 1], x[i + 5]);
      h2 = tja::fmax3(h2, x[i + 2], x[i + 6]);
      h3 = tja::fmax3(h3, x[i + 3], x[i + 7]);
    }
    h0 = tja::fmax3(h0, x[60], x[61]);
    h1 = tja::fmax3(h1, x[62], x[63]);
    const float top = tja::fmax3(h0, h1, fmaxf(h2, h3)) * c;
    float alpha = 1.0f;
    const bool raise = top - base > C::SHIFT + C::RAISE || (base == -INFINITY && top > base);
    if (raise) {
      const float next = base_of(top, C::SHIFT);
      alpha = exp2_fast(base - next);
      base = next;
      l0 *= alpha;
      l1 *= alpha;
    }
    if (__any_sync(0xffffffffu, raise)) {
      if (!C::Q8 && clo != FAR && __any_sync(0xffffffffu, fabsf(top) >= 0x1p20f && fabsf(top) < INFINITY)) {
#pragma unroll
        for (int i = 0; i < 64; ++i) x[i] *= c;
        c = 1.0f;
        clo = FAR;
      }
      if (j > 0) {
        // O at rest.  (A phase is waited for only when the one before it is known to be over: the scores
        // of block j were made after P V of block j - 2.)
        ok = sh.wait(S::PV_DONE + 8 * (2 * t + ((use - 1) & 1)), (use - 1) >> 1, p, 14);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int i = 0; i < D; i += 16) {
          uint32_t o[16];
          tmem_ld16(tO + i, o);
#pragma unroll
          for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
          tja::tmem_st16_wait(tO + i, o);
        }
      }
    }
    const float from = base == -INFINITY ? 0.0f : base;
    const uint64_t cc = tja::f2_pack(c, c), nb2 = tja::f2_pack(-from, -from);
    uint64_t ll = tja::f2_pack(l0, l1);
    probabilities<T, C>(x, cc, nb2, sc, ll, tS);
    tja::f2_unpack(ll, l0, l1);
    tja::tmem_wait_st();
    tc_fence_before();
    mbar_arrive(sh.at(S::P_READY + 8 * (2 * t + (use & 1))));
  }
  const int last = tile_blocks + nb - 1;
  if (!ok || !sh.wait(S::PV_DONE + 8 * (2 * t + (last & 1)), last >> 1, p, 13)) return;
  tc_fence_after();
  const float l = l0 + l1;
  if (l != l && base == -INFINITY) base = 0.0f;  // only NaN scores: the row is NaN, not empty
  const bool none = base == -INFINITY, mine_to_write = r < g.rows;
  if (nb == g.all) {
    const float inv = none ? 0.0f : 1.0f / l;
    int tok, hd;
    row_of(p, g.head, g.r0 + r, tok, hd);
    tok += g.s.start;
    T* dst = static_cast<T*>(p.a.out) + tok * p.a.out_token + hd * p.a.out_head;
#pragma unroll 1
    for (int i = 0; i < D; i += 16) {
      uint32_t o[16];
      tmem_ld16(tO + i, o);
      if (mine_to_write) {
        float y[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) y[k] = none ? 0.0f : __uint_as_float(o[k]) * inv;
        tj_store_vec(dst + i, y);
        tj_store_vec(dst + i + 8, y + 8);
      }
    }
    if (p.a.lse && mine_to_write)
      p.a.lse[static_cast<long>(tok) * p.a.q_heads + hd] = none ? -INFINITY : (base + log2f(l)) * 0.69314718055994531f;
  } else {
    const long slot = (2L * blockIdx.x + (g.later ? 0 : 1)) * TILE_ROWS + r;
    float* dst = p.part_o + slot * D;
#pragma unroll 1
    for (int i = 0; i < D; i += 16) {
      uint32_t o[16];
      tmem_ld16(tO + i, o);
      if (mine_to_write)
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          __stcg(reinterpret_cast<uint4*>(dst + i + k), make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]));
    }
    if (mine_to_write) __stcg(p.part_ml + slot, make_float2(base, l));
  }
  tc_fence_before();
}

template <class T, int CD, int D>
__global__ void __launch_bounds__(512, 1) attention_tiles(const __grid_constant__ AttnParams p) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  using S = TilesShared<T, CD, D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const S sh(smem_raw);
  const int warp = threadIdx.x >> 5;
  if (blockIdx.x == 0 && warp == 15) report_sequences(p, threadIdx.x & 31, 32);  // a warp that has nothing else to do
  const long total = total_work(p);
  if (total == 0) return;
  const Cut cut = cut_work(p, total, gridDim.x);
  if (blockIdx.x >= cut.parts) return;
  long pos = cut.begin(blockIdx.x);
  const long to = cut.begin(blockIdx.x + 1);

  if (threadIdx.x == 0) {
    mbar_init(sh.at(S::Q_FULL), 128);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(sh.at(S::K_FULL + 8 * s), 64);
      mbar_init(sh.at(S::V_FULL + 8 * s), 64);
      mbar_init(sh.at(S::K_EMPTY + 8 * s), 2);
      mbar_init(sh.at(S::V_EMPTY + 8 * s), 2);
    }
    for (int s = 0; s < C::SCALES; ++s) mbar_init(sh.at(S::SC_FULL + 8 * s), 64);
    for (int i = 0; i < 4; ++i) {
      mbar_init(sh.at(S::S_FULL + 8 * i), 1);
      mbar_init(sh.at(S::P_READY + 8 * i), 128);
      mbar_init(sh.at(S::PV_DONE + 8 * i), 1);
    }
    mbar_init(sh.at(S::DRAIN), 1);
    mbar_init(sh.at(S::DRAIN + 8), 1);
    *sh.abort_flag() = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    tmem_alloc(sh.at(S::SLOT), C::TMEM);
    tmem_relinquish();
  }
  if (warp == 14) next_segment(p, pos, to, sh.segment(0));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sh.tmem_slot();
  // every role goes through the same segments; `blocks` and the like count on over them, as the
  // barriers' phases do
  int blocks = 0;
  if (warp < 8) {
    regs_inc<C::REGS_S>();
    int tile_blocks = 0;
    for (int seg = 0; sh.segment(seg).nb; ++seg) {
      const bool busy = warp < 4 || sh.segment(seg).rows > 128;
      if (busy) softmax<T, CD, D>(p, sh, tmem, seg, blocks, tile_blocks);
      blocks += sh.segment(seg).nb;
      if (busy) tile_blocks += sh.segment(seg).nb;
      if (!end_segment(sh)) break;
    }
  } else if (warp < 12) {
    regs_dec<C::REGS_P>();
    for (int seg = 0; sh.segment(seg).nb; ++seg) {
      produce<T, CD, D>(p, sh, seg, blocks);
      blocks += sh.segment(seg).nb;
      if (!end_segment(sh)) break;
    }
  } else {
    regs_dec<C::REGS_M>();
    int tile_blocks = 0;
    for (int seg = 0; sh.segment(seg).nb; ++seg) {
      const bool busy = warp == 12 || (warp == 13 && sh.segment(seg).rows > 128);
      if (busy) multiply<T, CD, D>(p, sh, tmem, seg, warp - 12, blocks, tile_blocks);
      if (warp == 14) next_segment(p, pos, to, sh.segment(seg + 1));
      blocks += sh.segment(seg).nb;
      if (busy) tile_blocks += sh.segment(seg).nb;
      if (!end_segment(sh)) break;
    }
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, C::TMEM);
}

}  // namespace tjs
