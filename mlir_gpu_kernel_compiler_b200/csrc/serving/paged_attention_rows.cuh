// Attention over a paged cache for few rows (single tokens, a few drafted ones): a tile is 16 rows.
//
// What bounds it: the cache is read once and a key meets at most 16 rows, 2 x 16 products for each
// of its bytes at the most, far below the tensor cores' rate; so it is HBM, and the kernel is made
// of loads.  Keys and values go from global memory straight into the registers that the matrix
// instruction wants, 16 bytes a load and no shared memory: the order of the head dimension inside a
// product is free as long as both operands agree, so a thread's 16 bytes of a key serve as its
// fragments of two (16-bit) or four (8-bit) steps, and the query's fragments are gathered in that
// order once.  A value's 16 bytes are eight (sixteen) columns of the output, which fixes the order of
// its columns, undone when it is stored; two keys' bytes are paired by one byte permutation.
//
// A warp takes every fourth block of KS keys of its CTA's chunk with a running maximum and sum of
// its own, so the main loop has no barrier; the four warps' results are joined at the end, and the
// chunks of a row tile by the CTA that finishes last (in the order of the chunks, so results do not
// depend on which that is).
#pragma once
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

template <class T, int CD, int D>
__global__ void __launch_bounds__(128, D == 64 ? 4 : 3) attention_rows(const __grid_constant__ AttnParams p) {
  constexpr bool Q8 = CD == TJ_I8 || CD == TJ_E4M3;
  constexpr int KS = Q8 ? 32 : 16;       // keys of a warp's block
  constexpr int NT = KS / 8;             // score tiles of 8 keys
  constexpr int ES = Q8 ? 1 : 2;
  constexpr int KC = D * ES / 64;        // 16-byte pieces of a key a thread holds
  constexpr int STEPS = Q8 ? 4 : 2;      // products' steps of 16 that a piece serves
  constexpr int VB = D * ES / 8;         // bytes of a value a thread holds: 32, 16 or 8
  constexpr int VC = VB > 16 ? 2 : 1;    // ... as loads (of 16 bytes, or one of 8)
  constexpr int VW = VB / 4;             // ... as words
  constexpr int OT = D / 8;              // output tiles of 8 columns
  constexpr int PITCH = D + 4;

  __shared__ float s_o[4][16][PITCH];
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_last;

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int heads = static_cast<int>(p.a.cache.heads);
  const int unit = blockIdx.x / heads, h = blockIdx.x - unit * heads;
  const Piece w = find_piece(p, unit, 16, 4 * KS);
  if (!w.some) return;
  const Seq s = sequence(p, w.b);
  const int rows = min(16, s.n * p.group - w.tile * 16);
  const int r0 = w.tile * 16;
  int lo, hi;
  key_range(p, s, r0 / p.group, (r0 + rows - 1) / p.group, lo, hi);
  const int cuts = max(1, (hi - lo + w.chunk - 1) / w.chunk);
  if (w.c >= cuts) return;
  const int k0 = lo + w.c * w.chunk, k1 = min(hi, k0 + w.chunk);
  if (threadIdx.x == 0 && w.c == 0 && h == 0 &&
      (p.a.kv_lens[w.b] < 0 || p.a.kv_lens[w.b] > p.a.table_width * p.a.cache.page_size))
    tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_LENGTH);

  // this thread's two rows, g and g + 8: their queries and the keys that they see
  uint32_t qa[KC * STEPS][4];
  int rlo[2], rhi[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i, tok = (r0 + r) / p.group, hd = h * p.group + (r0 + r) - tok * p.group;
    const bool on = r < rows;
    rlo[i] = rhi[i] = 0;
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

  float o[OT][4];
#pragma unroll
  for (int i = 0; i < OT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

  const int* table = p.a.page_table + w.b * p.a.table_row;
  const char* kbase = static_cast<const char*>(p.a.cache.k) + h * p.a.cache.head_stride * ES;
  const char* vbase = static_cast<const char*>(p.a.cache.v) + h * p.a.cache.head_stride * ES;
  const float* ksc = Q8 ? p.a.cache.k_scale + h * p.a.cache.scale_head : nullptr;
  const float* vsc = Q8 ? p.a.cache.v_scale + h * p.a.cache.scale_head : nullptr;

  // lane i < KS looks key base + i up: the byte offset of its row (-1: not there), and its scales
  auto look_up = [&](int base, long& off, float& ks, float& vs) {
    off = -1;
    ks = vs = 0.0f;
    const int key = base + lane;
    if (lane < KS && key < k1) {
      const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / static_cast<int>(p.a.cache.page_size);
      const int sl = key - pg * static_cast<int>(p.a.cache.page_size);
      const int page = table[pg];
      if (page >= 0 && page < p.a.cache.pages) {
        off = (page * p.a.cache.page_stride + sl * p.a.cache.slot_stride) * ES;
        if (Q8) {
          const long so = page * p.a.cache.scale_page + sl * p.a.cache.scale_slot;
          ks = __ldg(ksc + so);
          vs = __ldg(vsc + so);
        }
      } else {
        tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_PAGE);
      }
    }
  };

  long off;
  float ks, vs;
  int base = k0 + warp * KS;
  if (base < k1) look_up(base, off, ks, vs);
  for (; base < k1; base += 4 * KS) {
    uint4 kf[NT][KC];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const long ro = __shfl_sync(0xffffffffu, off, 8 * j + g);
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kf[j][c] = ro >= 0 ? tj_ld16_stream(kbase + ro + (c * 4 + t) * 16) : make_uint4(0, 0, 0, 0);
    }
    uint32_t vf[KS / 4][VW];  // [16-key step][key 2t, 2t + 1, 2t + 8, 2t + 9]
#pragma unroll
    for (int j = 0; j < KS / 4; ++j) {
      const long ro = __shfl_sync(0xffffffffu, off, (j >> 2) * 16 + 2 * t + (j & 1) + ((j & 2) ? 8 : 0));
      if (VB == 8) {
        const uint2 x = ro >= 0 ? __ldg(reinterpret_cast<const uint2*>(vbase + ro + g * 8)) : make_uint2(0, 0);
        vf[j][0] = x.x;
        vf[j][1] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const uint4 x = ro >= 0 ? tj_ld16_stream(vbase + ro + (c * 8 + g) * 16) : make_uint4(0, 0, 0, 0);
          vf[j][(4 * c) % VW] = x.x;
          vf[j][(4 * c + 1) % VW] = x.y;
          vf[j][(4 * c + 2) % VW] = x.z;
          vf[j][(4 * c + 3) % VW] = x.w;
        }
      }
    }
    const float my_ks = ks, my_vs = vs;
    if (base + 4 * KS < k1) look_up(base + 4 * KS, off, ks, vs);

    float sc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.0f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        if constexpr (Q8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t x = word(kf[j][c], e);
            const uint32_t b0 = Codes<T, CD>::make(__byte_perm(x, 0, CD == TJ_I8 ? 0x4140 : 0x1404));
            const uint32_t b1 = Codes<T, CD>::make(__byte_perm(x, 0, CD == TJ_I8 ? 0x4342 : 0x3424));
            mma16816<T>(sc[j], qa[c * 4 + e], b0, b1);
          }
        } else {
          mma16816<T>(sc[j], qa[c * 2], kf[j][c].x, kf[j][c].y);
          mma16816<T>(sc[j], qa[c * 2 + 1], kf[j][c].z, kf[j][c].w);
        }
      }
    }
    // t = scaled score (+ log2 vs); masked keys -inf
    float inv[NT][2];
    const float lane_lv = Q8 ? fmaxf(__log2f(my_vs), MIN_LOG2_SCALE) : 0.0f;
    const float lane_inv = Q8 ? exp2_fast(-lane_lv) : 1.0f, lane_k = my_ks * p.scale_log2;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int kk = 8 * j + 2 * t + e, key = base + kk;
        float kfac = p.scale_log2, lv = 0.0f;
        if (Q8) {
          kfac = __shfl_sync(0xffffffffu, lane_k, kk);
          lv = __shfl_sync(0xffffffffu, lane_lv, kk);
          inv[j][e] = __shfl_sync(0xffffffffu, lane_inv, kk);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float& x = sc[j][2 * i + e];
          x = Q8 ? fmaf(x, kfac, lv) : x * kfac;
          if (key < rlo[i] || key >= rhi[i] || key >= k1) x = -INFINITY;
          mx[i] = fmaxf(mx[i], x);
        }
      }
    }
    bool moved = false;
    float base_m[2], alpha[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float next = fmaxf(m[i], mx[i]);
      moved |= next > m[i];
      const float from = next == -INFINITY ? 0.0f : next;
      alpha[i] = exp2_fast(m[i] - from);
      base_m[i] = from - P_SHIFT<T>;
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
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        sc[j][e] = exp2_fast(sc[j][e] - base_m[e >> 1]);
        l[e >> 1] += Q8 ? sc[j][e] * inv[j][e & 1] : sc[j][e];
      }
#pragma unroll
    for (int k16 = 0; k16 < KS / 16; ++k16) {
      const uint32_t pa[4] = {pack2<T>(sc[2 * k16][0], sc[2 * k16][1]), pack2<T>(sc[2 * k16][2], sc[2 * k16][3]),
                              pack2<T>(sc[2 * k16 + 1][0], sc[2 * k16 + 1][1]), pack2<T>(sc[2 * k16 + 1][2], sc[2 * k16 + 1][3])};
      const uint32_t(&va)[VW] = vf[4 * k16], (&vb)[VW] = vf[4 * k16 + 1], (&vc)[VW] = vf[4 * k16 + 2], (&vd)[VW] = vf[4 * k16 + 3];
#pragma unroll
      for (int j = 0; j < OT; ++j) {
        uint32_t b0, b1;
        if constexpr (Q8) {
          // byte j % 4 of both keys' words, into both bytes of a half
          const int n = j & 3;
          const uint32_t sel = n | (n << 4) | ((n + 4) << 8) | ((n + 4) << 12);
          b0 = Codes<T, CD>::make(__byte_perm(va[j >> 2], vb[j >> 2], sel));
          b1 = Codes<T, CD>::make(__byte_perm(vc[j >> 2], vd[j >> 2], sel));
        } else {
          const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
          b0 = __byte_perm(va[j >> 1], vb[j >> 1], sel);
          b1 = __byte_perm(vc[j >> 1], vd[j >> 1], sel);
        }
        mma16816<T>(o[j], pa, b0, b1);
      }
    }
  }

  // join the four warps
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
  constexpr int PER = NV > 16 / ES ? 16 / ES : NV;  // ... PER consecutive ones at a time
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
    const float f = m[i] == -INFINITY ? 0.0f : exp2_fast(m[i] - top);
#pragma unroll
    for (int j = 0; j < OT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = (j / PER) * 8 * PER + (2 * t + e) * PER + j % PER;
        s_o[warp][r][col] = o[j][2 * i + e] * f;
      }
  }
  __syncthreads();

  // 8 threads a row, D / 8 columns each
  constexpr int W = D / 8;
  const int r = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * W;
  const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
  float sum = 0.0f, acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = s_o[0][r][c0 + i] + s_o[1][r][c0 + i] + s_o[2][r][c0 + i] + s_o[3][r][c0 + i];
#pragma unroll
  for (int k = 0; k < 4; ++k) sum += s_m[k][r] == -INFINITY ? 0.0f : s_l[k][r] * exp2_fast(s_m[k][r] - top);
  float best = top;
  if (cuts > 1) {
    if (r < rows) {
      float* po = p.part_o + (static_cast<long>(blockIdx.x) * 16 + r) * D + c0;
#pragma unroll
      for (int i = 0; i < W; i += 4) __stcg(reinterpret_cast<float4*>(po + i), make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]));
      if ((threadIdx.x & 7) == 0) __stcg(p.part_ml + static_cast<long>(blockIdx.x) * 16 + r, make_float2(top, sum));
    }
    __threadfence();
    __syncthreads();
    const int first = blockIdx.x - w.c * heads;  // the tile's first chunk
    if (threadIdx.x == 0) {
      const int done = atomicAdd(p.counters + first, 1);
      s_last = done == cuts - 1;
      if (s_last) p.counters[first] = 0;  // ready for the next call
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    if (r >= rows) return;
    best = -INFINITY;
    for (int k = 0; k < cuts; ++k) best = fmaxf(best, __ldcg(p.part_ml + static_cast<long>(first + k * heads) * 16 + r).x);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] = 0.0f;
    for (int k = 0; k < cuts; ++k) {
      const long at = static_cast<long>(first + k * heads) * 16 + r;
      const float2 ml = __ldcg(p.part_ml + at);
      const float f = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - best);
      sum += ml.y * f;
#pragma unroll
      for (int i = 0; i < W; i += 4) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * D + c0 + i));
        acc[i] += v.x * f;
        acc[i + 1] += v.y * f;
        acc[i + 2] += v.z * f;
        acc[i + 3] += v.w * f;
      }
    }
  }
  if (r >= rows) return;
  const int tok = (r0 + r) / p.group, hd = h * p.group + (r0 + r) - tok * p.group;
  const bool none = best == -INFINITY;  // nothing visible: zeros
  const float div = none ? 0.0f : 1.0f / sum;
  T* dst = static_cast<T*>(p.a.out) + (s.start + tok) * p.a.out_token + hd * p.a.out_head + c0;
#pragma unroll
  for (int i = 0; i < W; i += 8) {
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = none ? 0.0f : acc[i + k] * div;
    tj_store_vec(dst + i, y);
  }
  if (p.a.lse && (threadIdx.x & 7) == 0)
    p.a.lse[(s.start + tok) * p.a.q_heads + hd] = none ? -INFINITY : (best - P_SHIFT<T> + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace tjs
