// Attention over a paged cache for few rows (single tokens, a few drafted ones): a tile is 16 rows.
//
// What bounds it: the cache is read once and a key meets at most 16 rows, 2 x 16 products for each
// of its bytes at the most, far below the tensor cores' rate; so it is HBM, and the kernel has to keep
// enough reads in flight.  Each warp has a ring of its own in shared memory (8 warps of 24 KB an SM, or
// 12 of 16 KB for 8-bit caches, whose codes take more instructions) that asynchronous copies fill one or
// more blocks ahead, so the main loop has no barrier.  64 single tokens over up to 8192 keys take 231 us, 94 % of
// the rate of a copy (with the loads straight into registers, where a block's are in flight only until
// it is used, 387 us).  Three over up to 100003 keys of i8 take 56 us, 57 %, of e4m3 49 us, 64 %.
//
// The order of the head dimension inside a product is free as long as both operands agree, so 16
// bytes of a key serve a thread as its fragments of two (16-bit) or four (8-bit) steps, read with one
// instruction, and the query's fragments are gathered in that order once.  A value's 16 bytes are
// eight (sixteen) columns of the output, which fixes the order of its columns, undone when it is stored;
// two keys' elements are paired by a byte permutation.  The pieces of a row are permuted by its number
// so that both ways of reading are free of bank conflicts.
//
// An 8-bit cache's codes become f16, bf16 queries too, times a power of two that brings the largest element
// near 2^14: byte permutations and masks run at half rate, and of i8 codes bf16 needs three for a pair where f16
// needs 1.5 (keys) and 2 (values); e4m3 has an instruction to f16.  The rows of a tile are different tokens and
// heads.  While their largest elements are within 2^12 of one another they share the power: f16's step of 2^-24 then
// leaves no element off by more than 2^-27 of its row's largest, less than f32 does in the score.  Otherwise each has
// its own, at a multiplication a score.  (That loop beside the other costs three single tokens over 100003 i8
// keys 56 us for 54: warps wait for instructions, 0.5 an issue.)
//
// A CTA's warps take blocks of KS keys of its chunk in turn, with a running maximum and sum each; their
// results are joined at the end, and the chunks of a row tile by the CTA that
// finishes last (in the order of the chunks, so results do not depend on which that is).
#pragma once
#include <limits.h>

#include "paged_attention.cuh"

namespace tjs {

template <class T> TJ_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> TJ_DEV void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> TJ_DEV void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

TJ_DEV uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

TJ_DEV void copy16(uint32_t dst, const void* src, bool on) {
  const int bytes = on ? 16 : 0;  // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TJ_DEV void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
TJ_DEV void copy4(uint32_t dst, const void* src, bool on) {
  const int bytes = on ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TJ_DEV uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}
TJ_DEV uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}

template <class T, int CD, int D, bool WIDE> struct Rows {
  using C = typename std::conditional<CD == TJ_I8 || CD == TJ_E4M3, __half, T>::type;  // what is multiplied
  static constexpr bool Q8 = CD == TJ_I8 || CD == TJ_E4M3;
  static constexpr int ES = Q8 ? 1 : 2;
  static constexpr int ROW = D * ES;                            // bytes of a key
  static constexpr int KS = !Q8 && D == 128 ? 16 : 32;          // keys of a warp's block
  static constexpr int BLOCK = 2 * KS * ROW;                    // bytes of its keys and values
  // WIDE: an SM's warps are one CTA, for work in few pieces, which is then joined from fewer parts
  static constexpr int WARPS = WIDE ? (Q8 ? 12 : 8) : 4, CTAS = (Q8 ? 12 : 8) / WARPS, THREADS = 32 * WARPS;
  static constexpr int STAGES = (Q8 ? 16384 : 24576) / BLOCK;
  static constexpr int SCALES = Q8 ? STAGES * KS * 3 * 4 : 0;   // ks, log2 vs, 1 / vs
  static constexpr int WARP = STAGES * BLOCK + SCALES;
  static constexpr int SMEM = WARPS * WARP;
  // the 16-byte piece of a row in a block; rows of 4 pieces share a line of 8
  static TJ_DEV uint32_t piece(int row, int i) {
    constexpr int PIECES = ROW / 16;
    if (PIECES == 4) return ((row >> 1) * 8 + ((((row & 1) << 2) | i) ^ (((row >> 1) & 3) << 1))) * 16;
    return (row * PIECES + (i ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2)))) * 16;
  }
};

template <class T, int CD, int D, bool WIDE>
__global__ void __launch_bounds__(Rows<T, CD, D, WIDE>::THREADS, Rows<T, CD, D, WIDE>::CTAS) attention_rows(const __grid_constant__ AttnParams p) {
  using R = Rows<T, CD, D, WIDE>;
  using C = typename R::C;
  constexpr bool Q8 = R::Q8;
  constexpr int KS = R::KS, ES = R::ES, STAGES = R::STAGES, WARPS = R::WARPS;
  constexpr int NT = KS / 8;             // score tiles of 8 keys
  constexpr int KC = D * ES / 64;        // 16-byte pieces of a key a thread reads
  constexpr int STEPS = Q8 ? 4 : 2;      // products' steps of 16 that a piece serves
  constexpr int VB = D * ES / 8;         // bytes of a value a thread reads: 32, 16 or 8
  constexpr int VC = VB > 16 ? 2 : 1;    // ... as loads (of 16 bytes, or one of 8)
  constexpr int VW = VB / 4;             // ... as words
  constexpr int OT = D / 8;              // output tiles of 8 columns
  constexpr int PITCH = D + 4;

  extern __shared__ __align__(128) uint8_t ring[];
  float(*const s_o)[16][PITCH] = reinterpret_cast<float(*)[16][PITCH]>(ring);  // when the loop is done
  static_assert(WARPS * 16 * PITCH * 4 <= R::SMEM, "the warps' results lie over the ring");
  __shared__ float s_m[WARPS][16], s_l[WARPS][16];
  __shared__ int s_last;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int heads = static_cast<int>(p.a.cache.heads);
  const int unit = blockIdx.x / heads, h = blockIdx.x - unit * heads;
  if (blockIdx.x == 0) report_sequences(p, threadIdx.x, R::THREADS);
  const Piece w = find_piece(p, unit, 16, WARPS * KS);
  if (!w.some) return;
  const Seq s = sequence(p, w.b);
  const int rows = min(16, s.n * p.group - w.tile * 16);
  const int r0 = w.tile * 16;
  int lo, hi;
  key_range(p, s, r0 / p.group, (r0 + rows - 1) / p.group, lo, hi);
  // never more chunks than were launched, as each has to arrive at the tile's counter; the last takes what is left
  const int cuts = min(w.cuts, max(1, (hi - lo + w.chunk - 1) / w.chunk));
  if (w.c >= cuts) return;
  const int k0 = lo + w.c * w.chunk, k1 = w.c + 1 < cuts ? k0 + w.chunk : hi;

  const int* table = p.a.page_table + w.b * p.a.table_row;
  const char* kbase = static_cast<const char*>(p.a.cache.k) + h * p.a.cache.head_stride * ES;
  const char* vbase = static_cast<const char*>(p.a.cache.v) + h * p.a.cache.head_stride * ES;
  const float* ksc = Q8 ? p.a.cache.k_scale + h * p.a.cache.scale_head : nullptr;
  const float* vsc = Q8 ? p.a.cache.v_scale + h * p.a.cache.scale_head : nullptr;
  const uint32_t my_ring = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + warp * R::WARP;

  // Lane i looks key base + i of a block up: its page a block ahead, then the byte offset of its row and
  // its place among the scales (-1: not there).
  const int page_size = static_cast<int>(p.a.cache.page_size);
  auto page_of = [&](int base) {  // (nothing may be done to the page here: the look-up would be waited for)
    const int key = base + lane;
    if (lane >= KS || key >= k1) return 0;
    return table[p.page_shift >= 0 ? key >> p.page_shift : key / page_size];
  };
  // Where a lane copies to, and reads from, in a block: its first row's piece; further rows are at constant
  // distances, but for bits that the permutation turns by the row's number, which are constants too.
  constexpr int PIECES = R::ROW / 16, PER = 32 / PIECES;  // lanes of a row, rows of a warp's instruction
  const uint32_t copy_at = R::piece(lane / PIECES, lane % PIECES);
  const uint32_t key_at = R::piece(g, t), value_at0 = R::piece(2 * t, VB == 8 ? g >> 1 : g) + (VB == 8 ? (g & 1) * 8 : 0),
                 value_at1 = R::piece(2 * t + 1, VB == 8 ? g >> 1 : g) + (VB == 8 ? (g & 1) * 8 : 0);
  const char* const my_k = kbase + (lane % PIECES) * 16;
  const long to_v = vbase - kbase;
  auto fetch = [&](int stage, int base, int page) {
    const char* row = my_k;  // this lane looks it up for others, so the piece is added where it is used
    long soff = 0;
    const bool here = lane < KS && base + lane < k1;
    bool on = false;
    if (here && page >= 0 && page < p.a.cache.pages) {
      const int key = base + lane, slot = p.page_shift >= 0 ? key & (page_size - 1) : key % page_size;
      row = kbase + (page * p.a.cache.page_stride + slot * p.a.cache.slot_stride) * ES;
      if (Q8) soff = page * p.a.cache.scale_page + slot * p.a.cache.scale_slot;
      on = true;
    } else if (here) {
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_PAGE);
    }
    const unsigned live = __ballot_sync(0xffffffffu, on);
    const uint32_t dst = my_ring + stage * R::BLOCK;
    const uint32_t mine = live >> (lane / PIECES);
    const long add = (lane % PIECES) * 16;
    constexpr unsigned ALL = KS == 32 ? 0xffffffffu : (1u << KS) - 1;
    if (live == ALL) {
#pragma unroll
      for (int j = 0; j < KS / PER; ++j) {
        const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<long>(row), j * PER + lane / PIECES)) + add;
        const uint32_t at = dst + (copy_at ^ (((j * PER / 2) & 3) << 5)) + j * PER * R::ROW;
        copy16(at, src);
        copy16(at + KS * R::ROW, src + to_v);
      }
    } else if (base < k1) {
#pragma unroll
      for (int j = 0; j < KS / PER; ++j) {
        const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<long>(row), j * PER + lane / PIECES)) + add;
        const uint32_t at = dst + (copy_at ^ (((j * PER / 2) & 3) << 5)) + j * PER * R::ROW;
        const bool there = (mine >> (j * PER)) & 1;
        copy16(at, there ? src : my_k, there);
        copy16(at + KS * R::ROW, there ? src + to_v : my_k, there);
      }
    }
    if (Q8 && base < k1) {
      const uint32_t s = my_ring + STAGES * R::BLOCK + (stage * KS * 3 + lane) * 4;
      copy4(s, ksc + soff, on);
      copy4(s + KS * 4, vsc + soff, on);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  const int first = k0 + warp * KS;
  int ahead = first;  // the block to be fetched next
  int page = page_of(ahead);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    const int now = page;
    page = page_of(ahead + WARPS * KS);
    fetch(i, ahead, now);
    ahead += WARPS * KS;
  }
  // this thread's two rows, g and g + 8: their queries and the keys that they see
  uint32_t qa[KC * STEPS][4];
  int rlo[2], rhi[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i, tok = (r0 + r) / p.group, hd = h * p.group + (r0 + r) - tok * p.group;
    const bool on = r < rows;
    rlo[i] = 0;  // a row that is not there sees all, and is not stored
    rhi[i] = INT_MAX;
    if (on) row_range(p, s, tok, rlo[i], rhi[i]);
    const T* src = static_cast<const T*>(p.a.q) + (s.start + tok) * p.a.q_token + hd * p.a.q_head;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
      // the elements of piece c: 8 (16) of them from c * 32 + t * 8 (c * 64 + t * 16)
      const T* at = src + (c * 4 + t) * (16 / ES);
#pragma unroll
      for (int v = 0; v < STEPS / 2; ++v) {
        const uint4 x = on ? tj_ld16(at + 8 * v) : make_uint4(0, 0, 0, 0);
        qa[c * STEPS + 2 * v][i] = x.x;
        qa[c * STEPS + 2 * v][i + 2] = x.y;
        qa[c * STEPS + 2 * v + 1][i] = x.z;
        qa[c * STEPS + 2 * v + 1][i + 2] = x.w;
      }
    }
  }

  float score_scale = p.scale_log2;
  bool apart = false;  // the same for the warp: the rows' scores are to be multiplied by s_m (free until the end)
  if constexpr (!std::is_same<T, C>::value) {
    uint32_t top[2] = {0, 0};  // this thread's rows' largest elements, as bits
#pragma unroll
    for (int c = 0; c < KC * STEPS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e & 1] = max(top[e & 1], max((qa[c][e] & 0x7fffu) << 16, qa[c][e] & 0x7fff0000u));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    }
    // rows of zeros (or that are not there) go with any power
    const uint32_t most = __reduce_max_sync(0xffffffffu, max(top[0], top[1]));
    const uint32_t least = __reduce_min_sync(0xffffffffu, min(top[0] ? top[0] : most, top[1] ? top[1] : most));
    apart = most >= 0x7f800000u || (most >> 23) > (least >> 23) + 12;
    float up[2], down = 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // 2^(14 - the exponent), within what f32 holds twice over; 1 for zeros, infinities and NaN
      const uint32_t x = apart ? top[i] : most;
      const int raise = x > 0 && x < 0x7f800000u ? min(14 - (static_cast<int>(x >> 23) - 127), 100) : 0;
      up[i] = __int_as_float((127 + raise) << 23);
      down = __int_as_float((127 - raise) << 23);
      if (apart && t == 0) s_m[warp][g + 8 * i] = down;
    }
    if (!apart) score_scale *= down;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < KC * STEPS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t& w = qa[c][e];
        w = tj_pack_f16x2(__uint_as_float(w << 16) * up[e & 1], __uint_as_float(w & 0xffff0000u) * up[e & 1]);
      }
  }

  // keys that all of the tile's rows see need no mask
  const int mlo = __reduce_max_sync(0xffffffffu, max(rlo[0], rlo[1])), mhi = __reduce_min_sync(0xffffffffu, min(rhi[0], rhi[1]));

  float o[OT][4];
#pragma unroll
  for (int i = 0; i < OT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // bases and sums

  // The warp's blocks of keys.  The loop exists twice where rows may have powers of their own: a test inside it costs
  // tiles of like rows as much as the multiplication (64 single tokens over 4096 keys of 8 bits: 152 us for 136).
  const auto walk = [&](auto powers) __attribute__((always_inline)) {
    int stage = 0;
    for (int base = first; base < k1; base += WARPS * KS) {
      {
        const int now = page;
        page = page_of(ahead + WARPS * KS);
        fetch(stage == 0 ? STAGES - 1 : stage - 1, ahead, now);
        ahead += WARPS * KS;
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const uint32_t kblock = my_ring + stage * R::BLOCK, vblock = kblock + KS * R::ROW;
      float* const scale = reinterpret_cast<float*>(ring + warp * R::WARP + STAGES * R::BLOCK) + stage * KS * 3;
      if constexpr (Q8) {
        scale[lane] *= score_scale;
        const float lv = log2_scale(scale[KS + lane]);
        scale[KS + lane] = lv;
        scale[2 * KS + lane] = exp2_fast(-lv);
        __syncwarp();
      }
      if (++stage == STAGES) stage = 0;

      // the tiles' products are independent chains, so they go side by side
      float sc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        uint4 kf[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) kf[j] = lds16(kblock + (key_at ^ (c << 6)) + 8 * j * R::ROW);
#pragma unroll
        for (int e = 0; e < STEPS; ++e) {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t b0, b1;
            if constexpr (Q8) {
              codes4<C, CD>(word(kf[j], e), b0, b1);
            } else {
              b0 = word(kf[j], 2 * e);
              b1 = word(kf[j], 2 * e + 1);
            }
            mma16816<C>(sc[j], qa[c * STEPS + e], b0, b1);
          }
        }
      }
      if constexpr (decltype(powers)::value) {
        const float down[2] = {s_m[warp][g], s_m[warp][g + 8]};
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] *= down[e >> 1];
      }
      // t = scaled score (8-bit cache: + log2 vs); masked keys -inf
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float2 kfac = make_float2(score_scale, score_scale), lv = make_float2(0.0f, 0.0f);
        if constexpr (Q8) {
          kfac = *reinterpret_cast<const float2*>(scale + 8 * j + 2 * t);
          lv = *reinterpret_cast<const float2*>(scale + KS + 8 * j + 2 * t);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float& x = sc[j][e];
          x = Q8 ? fmaf(x, e & 1 ? kfac.y : kfac.x, e & 1 ? lv.y : lv.x) : x * score_scale;
        }
      }
      if (base < mlo || base + KS > mhi) {  // the same for the warp
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = base + 8 * j + 2 * t + (e & 1);
            if (key < rlo[e >> 1] || key >= rhi[e >> 1]) sc[j][e] = -INFINITY;
          }
      }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], fmaxf(sc[j][2 * i], sc[j][2 * i + 1]));
      bool moved = false;
      float from[2], alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        const float next = fmaxf(m[i], base_of(mx[i], P_SHIFT<C>));
        moved |= next > m[i];
        from[i] = next == -INFINITY ? 0.0f : next;
        alpha[i] = exp2_fast(m[i] - from[i]);
        m[i] = next;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) l[i] *= alpha[i];
#pragma unroll
        for (int j = 0; j < OT; ++j) {
          o[j][0] *= alpha[0];
          o[j][1] *= alpha[0];
          o[j][2] *= alpha[1];
          o[j][3] *= alpha[1];
        }
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float2 inv = make_float2(1.0f, 1.0f);
        if constexpr (Q8) inv = *reinterpret_cast<const float2*>(scale + 2 * KS + 8 * j + 2 * t);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[j][e] = exp2_fast(sc[j][e] - from[e >> 1]);
          l[e >> 1] += Q8 ? sc[j][e] * (e & 1 ? inv.y : inv.x) : sc[j][e];
        }
      }
#pragma unroll
      for (int k16 = 0; k16 < KS / 16; ++k16) {
        const uint32_t pa[4] = {pack2<C>(sc[2 * k16][0], sc[2 * k16][1]), pack2<C>(sc[2 * k16][2], sc[2 * k16][3]),
                                pack2<C>(sc[2 * k16 + 1][0], sc[2 * k16 + 1][1]), pack2<C>(sc[2 * k16 + 1][2], sc[2 * k16 + 1][3])};
        uint32_t va[VW], vb[VW], vc[VW], vd[VW];  // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the step
        auto value = [&](uint32_t (&v)[VW], uint32_t at) {
          if constexpr (VB == 8) {
            const uint2 x = lds8(vblock + at);
            v[0] = x.x;
            v[1] = x.y;
          } else {
#pragma unroll
            for (int c = 0; c < VC; ++c) {
              const uint4 x = lds16(vblock + at + c * 128);
              v[(4 * c) % VW] = x.x;
              v[(4 * c + 1) % VW] = x.y;
              v[(4 * c + 2) % VW] = x.z;
              v[(4 * c + 3) % VW] = x.w;
            }
          }
        };
        value(va, value_at0 + k16 * 16 * R::ROW);
        value(vb, value_at1 + k16 * 16 * R::ROW);
        value(vc, value_at0 + (k16 * 16 + 8) * R::ROW);
        value(vd, value_at1 + (k16 * 16 + 8) * R::ROW);
#pragma unroll
        for (int j = 0; j < OT; ++j) {
          uint32_t b0, b1;
          if constexpr (Q8) {
            // byte j % 4 of both keys' words: into both bytes of a half (i8), or the two of the low half
            const int n = j & 3;
            const uint32_t sel = CD == TJ_I8 ? n | (n << 4) | ((n + 4) << 8) | ((n + 4) << 12) : n | ((n + 4) << 4);
            b0 = Codes<C, CD>::make(__byte_perm(va[j >> 2], vb[j >> 2], sel));
            b1 = Codes<C, CD>::make(__byte_perm(vc[j >> 2], vd[j >> 2], sel));
          } else {
            const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
            b0 = __byte_perm(va[j >> 1], vb[j >> 1], sel);
            b1 = __byte_perm(vc[j >> 1], vd[j >> 1], sel);
          }
          mma16816<C>(o[j], pa, b0, b1);
        }
      }
      __syncwarp();  // the block's place may be filled again
    }
  };
  if constexpr (std::is_same<T, C>::value) {
    walk(std::false_type());
  } else {
    if (apart)
      walk(std::true_type());
    else
      walk(std::false_type());
  }

  // join the warps
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (l[i] != l[i] && m[i] == -INFINITY) m[i] = 0.0f;  // only NaN scores: the row is NaN, not empty
    if (t == 0) {
      s_m[warp][g + 8 * i] = m[i];
      s_l[warp][g + 8 * i] = l[i];
    }
  }
  __syncthreads();
  constexpr int NV = VB / ES;           // output columns from one thread's piece of a value, of each of ...
  constexpr int RUN = NV > 16 / ES ? 16 / ES : NV;  // ... RUN consecutive ones at a time
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    float top = s_m[0][r];
#pragma unroll
    for (int k = 1; k < WARPS; ++k) top = fmaxf(top, s_m[k][r]);
    const float f = m[i] == -INFINITY ? 0.0f : exp2_fast(m[i] - top);
#pragma unroll
    for (int j = 0; j < OT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = (j / RUN) * 8 * RUN + (2 * t + e) * RUN + j % RUN;
        s_o[warp][r][col] = o[j][2 * i + e] * f;
      }
  }
  __syncthreads();

  // Four columns of a row a thread.
  const auto store = [&](int row, int col, float4 v, float best, float sum) {
    int tok = (r0 + row) / p.group;
    const int hd = h * p.group + (r0 + row) - tok * p.group;
    tok += s.start;
    const bool none = best == -INFINITY;  // nothing visible: zeros
    const float div = 1.0f / sum;
    uint2 y = make_uint2(0, 0);
    if (!none) y = make_uint2(pack2<T>(v.x * div, v.y * div), pack2<T>(v.z * div, v.w * div));
    *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + tok * p.a.out_token + hd * p.a.out_head + col) = y;
    if (p.a.lse && col == 0)
      p.a.lse[static_cast<long>(tok) * p.a.q_heads + hd] = none ? -INFINITY : (best + log2f(sum)) * 0.69314718055994531f;
  };
  const int positions = rows * (D / 4);
  for (int at = threadIdx.x; at < positions; at += R::THREADS) {
    const int row = at / (D / 4), col = (at - row * (D / 4)) * 4;
    float best = s_m[0][row], sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int k = 1; k < WARPS; ++k) best = fmaxf(best, s_m[k][row]);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(&s_o[k][row][col]);
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
      sum += s_m[k][row] == -INFINITY ? 0.0f : s_l[k][row] * exp2_fast(s_m[k][row] - best);
    }
    if (cuts == 1) {
      store(row, col, v, best, sum);
    } else {
      const long slot = static_cast<long>(blockIdx.x) * 16 + row;
      __stcg(reinterpret_cast<float4*>(p.part_o + slot * D + col), v);
      if (col == 0) __stcg(p.part_ml + slot, make_float2(best, sum));
    }
  }
  if (cuts == 1) return;
  __threadfence();
  __syncthreads();
  const int first_cta = blockIdx.x - w.c * heads;  // the tile's first chunk
  if (threadIdx.x == 0) {
    const int done = atomicAdd(p.counters + first_cta, 1);
    s_last = done == cuts - 1;
    if (s_last) p.counters[first_cta] = 0;  // ready for the next call
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  // The chunks, in order.  Where there are fewer positions than threads, threads share a position's
  // chunks and are joined in shared memory.
  int shares = 1;
  while (shares * 2 * positions <= R::THREADS && shares * 2 <= cuts) shares *= 2;
  float* const joint = reinterpret_cast<float*>(ring);  // [shares * positions][6]
  for (int at = threadIdx.x; at < positions * shares; at += R::THREADS) {
    const int share = at / positions, pos = at - share * positions, row = pos / (D / 4), col = (pos - row * (D / 4)) * 4;
    float best = -INFINITY, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int GO = 8;  // chunks whose loads are in flight together
    for (int k = share; k < cuts; k += GO * shares) {
      float2 ml[GO];
      float4 x[GO];
      float top = best;
#pragma unroll
      for (int i = 0; i < GO; ++i) {
        const long slot = static_cast<long>(first_cta + min(k + i * shares, cuts - 1) * heads) * 16 + row;
        ml[i] = __ldcg(p.part_ml + slot);
        x[i] = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + col));
      }
#pragma unroll
      for (int i = 0; i < GO; ++i) {
        if (k + i * shares >= cuts) ml[i].x = -INFINITY;
        top = fmaxf(top, ml[i].x);
      }
      if (top == -INFINITY) continue;
      const float f = exp2_fast(best - top);
      v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
      sum *= f;
#pragma unroll
      for (int i = 0; i < GO; ++i) {
        if (ml[i].x == -INFINITY) continue;
        const float e = exp2_fast(ml[i].x - top);
        v = make_float4(v.x + x[i].x * e, v.y + x[i].y * e, v.z + x[i].z * e, v.w + x[i].w * e);
        sum += ml[i].y * e;
      }
      best = top;
    }
    if (shares == 1) {
      store(row, col, v, best, sum);
    } else {
      float* const j = joint + at * 6;
      j[0] = v.x;
      j[1] = v.y;
      j[2] = v.z;
      j[3] = v.w;
      j[4] = best;
      j[5] = sum;
    }
  }
  if (shares == 1) return;
  __syncthreads();
  for (int pos = threadIdx.x; pos < positions; pos += R::THREADS) {
    float best = -INFINITY, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int share = 0; share < shares; ++share) best = fmaxf(best, joint[(share * positions + pos) * 6 + 4]);
    for (int share = 0; share < shares; ++share) {
      const float* const j = joint + (share * positions + pos) * 6;
      if (j[4] == -INFINITY) continue;
      const float e = exp2_fast(j[4] - best);
      v = make_float4(v.x + j[0] * e, v.y + j[1] * e, v.z + j[2] * e, v.w + j[3] * e);
      sum += j[5] * e;
    }
    store(pos / (D / 4), (pos - pos / (D / 4) * (D / 4)) * 4, v, best, sum);
  }
}

}  // namespace tjs
