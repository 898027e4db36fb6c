// Attention over a paged cache for many rows (chunks of a prompt): a tile is 2 x 128 rows, and the
// products run on the tensor cores through tcgen05 with their sums in TMEM.
//
// What bounds it: a key meets 256 rows, 2 x 256 products for each of its elements, so the cache is
// cheap and the kernel is made of the tensor cores' two products a block (128 keys: 2 x 512 clocks a
// row tile at head dim 128) and of 128 exponentials a row and block (16 a clock and SM: 1024 clocks a
// row tile).  Both are about the same, and each row tile needs them in turn; two row tiles in
// antiphase keep both units busy.  Warps (512 threads, one CTA an SM):
//   0-3, 4-7   softmax of row tile 0, 1: a thread is a row.  It reads its 128 scores out of TMEM,
//              keeps a running maximum (moved, and the sums in TMEM rescaled, only when a block
//              exceeds it by more than 2^RAISE) and sum, and writes P over the scores, 16 bits each.
//   8-11       producers: warp w brings keys 32 w .. 32 w + 31 of each block: pages are looked up one
//              key a lane, rows copied asynchronously (16-bit caches) or converted to 16 bits on the
//              way (8-bit ones), in the 128-byte-swizzled layout that the matrix unit reads.  Pages may
//              have any size and the cache any strides, as no copy spans two rows.
//   12         issues the matrix instructions: per block, tile 0's P V then its next scores, then tile
//              1's; a tile's next scores overwrite its P, and follow the product that reads it.
//
// The work, (tile, block) pairs of all sequences and heads in a row, is cut into as many equal parts as
// there are SMs (each at least 4 blocks): a CTA takes a tile's end, whole tiles and a tile's beginning.
// Parts of one tile are joined by the CTA whose part comes last, in the tile's order.
//
// Every wait is bounded (TJ_WAIT_NS): one that runs out raises the CTA's abort flag and the status word.
#pragma once
#include <type_traits>

#include "../kernels/attention_sm100.cuh"
#include "paged_attention.cuh"

namespace tjs {

constexpr int TILE_ROWS = 256, TILE_KEYS = 128;

// The linear order of the work, in keys x group.  A tile weighs its keys, and one block more for what a
// tile costs by itself.
struct TileWork {
  long per_head;  // of a sequence: all its tiles
  long base;      // a tile's weight without what grows along the sequence
  int tiles;
  int rows;
  bool grows;     // causal without a window: tile t sees 256 (t + 1) / group tokens more
  TJ_DEV long before(int t) const {  // weight of the tiles before t
    if (!grows) return base * t;
    return t < tiles ? base * t + static_cast<long>(TILE_ROWS / 2) * t * (t + 1) : per_head;
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
    span = min(span, static_cast<long>(p.a.window) + TILE_ROWS / p.group);
  w.base = p.group * (span + TILE_KEYS);
  w.per_head = w.base * w.tiles;
  if (w.grows && w.tiles) w.per_head += static_cast<long>(TILE_ROWS / 2) * (w.tiles - 1) * w.tiles + w.rows;
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
  for (int b = lane; b < p.a.batch; b += 32) {
    mine += tile_work(p, sequence(p, b)).per_head;
    if (blockIdx.x == 0 && threadIdx.x < 32 && (p.a.kv_lens[b] < 0 || p.a.kv_lens[b] > p.a.table_width * p.a.cache.page_size))
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_ATTENTION * 16 + SITE_LENGTH);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  return mine * p.a.cache.heads;
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
  g.head = static_cast<int>(in_seq / w.per_head);
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
  if (lo + 1 == w.tiles) g.weight = w.per_head - w.before(lo);
  return g;
}

TJ_DEV void cp_async16(uint32_t dst, const void* src, bool on) {
  const int bytes = on ? 16 : 0;  // 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
TJ_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> TJ_DEV void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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

template <class T, int CD, int D> struct Tiles {
  static constexpr bool Q8 = CD == TJ_I8 || CD == TJ_E4M3;
  static constexpr int STAGES = D == 128 ? 2 : 4;
  static constexpr int SCALES = STAGES + 2;  // scale rows outlive their block's operands
  static constexpr uint32_t Q_BYTES = 128 * D * 2, KV_BYTES = TILE_KEYS * D * 2;
  static constexpr int SMEM = 1024 + 2 * Q_BYTES + 2 * STAGES * KV_BYTES + (Q8 ? SCALES * 3 * TILE_KEYS * 4 : 0) + 512;
  // TMEM columns: S_0, S_1 (128 each; P, 64 columns, over them), O_0, O_1 (D each)
  static constexpr uint32_t TMEM = 512;
  static constexpr float SHIFT = P_SHIFT<T> > 11.0f ? 11.0f : P_SHIFT<T>;  // with RAISE: P < 2^16
  static constexpr float RAISE = P_SHIFT<T> > 0.0f ? 4.0f : 8.0f;
};

// A CTA's shared memory and its piece of the work.
template <class T, int CD, int D> struct TilesShared {
  using C = Tiles<T, CD, D>;
  static constexpr int STAGES = C::STAGES;
  uint8_t *sQ, *sK, *sV;
  float* scales;  // [SCALES][3][128]: ks, log2 vs, 1 / vs
  uint64_t *q_full, *k_full, *v_full, *k_empty, *v_empty, *s_full, *p_ready, *o_done, *drain;
  uint32_t* tmem_slot;
  volatile int* abort_flag;
  int* s_last;
  long total, parts, from, to;
  TJ_DEV TilesShared(uint8_t* raw) {
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    sQ = smem;
    sK = sQ + 2 * C::Q_BYTES;
    sV = sK + STAGES * C::KV_BYTES;
    scales = reinterpret_cast<float*>(sV + STAGES * C::KV_BYTES);
    q_full = reinterpret_cast<uint64_t*>(scales + (C::Q8 ? C::SCALES * 3 * TILE_KEYS : 0));
    k_full = q_full + 1;
    v_full = k_full + STAGES;
    k_empty = v_full + STAGES;
    v_empty = k_empty + STAGES;
    s_full = v_empty + STAGES;  // [2]
    p_ready = s_full + 2;       // [2]
    o_done = p_ready + 2;
    drain = o_done + 1;
    tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    s_last = reinterpret_cast<int*>(tmem_slot + 2);
  }
};

enum class Role { softmax, producer, matrix };

// The segments of a CTA as one of its roles goes through them.
template <Role ROLE, class T, int CD, int D>
TJ_DEV void tiles_role(const AttnParams& p, const TilesShared<T, CD, D>& sh, uint32_t tmem) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  constexpr bool Q8 = C::Q8;
  constexpr int STAGES = C::STAGES, ES = Q8 ? 1 : 2;
  constexpr uint32_t Q_BYTES = C::Q_BYTES, KV_BYTES = C::KV_BYTES;
  constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_S = idesc_f16(BF, 128, TILE_KEYS, false, false), IDESC_O = idesc_f16(BF, 128, D, false, true);
  constexpr int WHERE = OP_ATTENTION * 16;
  uint8_t *const sQ = sh.sQ, *const sK = sh.sK, *const sV = sh.sV;
  float* const scales = sh.scales;
  uint64_t *const q_full = sh.q_full, *const k_full = sh.k_full, *const v_full = sh.v_full, *const k_empty = sh.k_empty,
                  *const v_empty = sh.v_empty, *const s_full = sh.s_full, *const p_ready = sh.p_ready, *const o_done = sh.o_done,
                  *const drain = sh.drain;
  volatile int* const abort_flag = sh.abort_flag;
  int* const s_last = sh.s_last;
  const long total = sh.total, parts = sh.parts, from = sh.from, to = sh.to;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // segments, and key blocks of row tile 0 and 1, before this segment: barrier phases run on
  int seg = 0, blocks = 0, blocks1 = 0;
  bool failed = false;
  for (long pos = from; pos < to && !failed;) {
    const TilePart w = find_tile(p, pos);
    const long a0 = pos - w.start, a1 = min(w.weight, to - w.start);
    pos = w.start + a1;
    const int r0 = w.tile * TILE_ROWS, rows = min(TILE_ROWS, w.s.n * p.group - r0);
    int lo, hi;
    key_range(p, w.s, r0 / p.group, (r0 + rows - 1) / p.group, lo, hi);
    const int first = lo / TILE_KEYS, all = max(1, (hi + TILE_KEYS - 1) / TILE_KEYS - first);
    const int j0 = static_cast<int>(a0 * all / w.weight), nb = static_cast<int>(a1 * all / w.weight) - j0;
    if (nb == 0) continue;
    const bool whole = nb == all;
    const int key0 = (first + j0) * TILE_KEYS;
    const int ntiles = rows > 128 ? 2 : 1;

    if constexpr (ROLE == Role::producer) {
      // ---------------- producers ----------------
      const int pw = warp - 8, tid = threadIdx.x - 256;
      bool ok = true;
      // queries: the packed rows' heads
      {
        constexpr int LPR = D / 8;  // 16-byte pieces of a row
        const int piece = tid % LPR;
        for (int r = tid / LPR; r < ntiles * 128; r += 128 / LPR) {
          const bool on = r < rows;
          const int rr = r0 + (on ? r : 0), tok = rr / p.group, hd = w.head * p.group + rr - tok * p.group;
          const T* src = static_cast<const T*>(p.a.q) + (w.s.start + tok) * p.a.q_token + hd * p.a.q_head + piece * 8;
          cp_async16(smem_u32(sQ) + (r >> 7) * Q_BYTES + swizzled(128, r & 127, piece), src, on);
        }
        cp_async_commit();
      }
      const int* table = p.a.page_table + w.b * p.a.table_row;
      const char* kbase = static_cast<const char*>(p.a.cache.k) + w.head * p.a.cache.head_stride * ES;
      const char* vbase = static_cast<const char*>(p.a.cache.v) + w.head * p.a.cache.head_stride * ES;
      auto look_up = [&](int j, long& off, long& scale_off) {
        const int key = key0 + j * TILE_KEYS + pw * 32 + lane;
        off = scale_off = -1;
        if (j < nb && key >= lo && key < hi) {
          const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / static_cast<int>(p.a.cache.page_size);
          const int sl = key - pg * static_cast<int>(p.a.cache.page_size);
          const int page = table[pg];
          if (page >= 0 && page < p.a.cache.pages) {
            off = (page * p.a.cache.page_stride + sl * p.a.cache.slot_stride) * ES;
            scale_off = page * p.a.cache.scale_page + sl * p.a.cache.scale_slot + w.head * p.a.cache.scale_head;
          } else {
            tj_report(p.status, TJ_STATUS_BOUNDS, WHERE + SITE_PAGE);
          }
        }
      };
      long off, soff;
      look_up(0, off, soff);
      if constexpr (!Q8) {
        constexpr int LPR = D / 8, PER = 32 / LPR;  // lanes of a row, rows of a warp's instruction
        const int piece = lane % LPR;
        auto copy = [&](uint8_t* dst, const char* base) {
#pragma unroll
          for (int i = 0; i < 32 / PER; ++i) {
            const int r = i * PER + lane / LPR;
            const long ro = __shfl_sync(0xffffffffu, off, r);
            cp_async16(smem_u32(dst) + swizzled(TILE_KEYS, pw * 32 + r, piece), base + (ro < 0 ? 0 : ro) + piece * 16, ro >= 0);
          }
          cp_async_commit();
        };
        auto arrive = [&](uint64_t* bar) {
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(bar));
        };
        for (int j = 0; j < nb; ++j) {
          const int it = blocks + j, s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          ok = mbar_wait_warp(smem_u32(&k_empty[s]), ph ^ 1u, abort_flag, p.status, WHERE + 5);
          if (!ok) break;
          copy(sK + s * KV_BYTES, kbase);
          if (j == 0) {
            cp_async_wait<1>();
            arrive(q_full);
          } else {
            cp_async_wait<1>();  // the block before's values
            arrive(&v_full[(it - 1) % STAGES]);
          }
          ok = mbar_wait_warp(smem_u32(&v_empty[s]), ph ^ 1u, abort_flag, p.status, WHERE + 6);
          if (!ok) break;
          copy(sV + s * KV_BYTES, vbase);
          look_up(j + 1, off, soff);
          cp_async_wait<1>();
#ifdef TJ_TEST_STALL_FIRST_LOAD
          // failure-path test build only: the first keys never arrive, so the wait for them runs out
          if (it == 0) continue;
#endif
          arrive(&k_full[s]);
        }
        cp_async_wait<0>();
        if (ok) arrive(&v_full[(blocks + nb - 1) % STAGES]);
      } else {
        constexpr int LPR = D / 16, PER = 32 / LPR, N = 32 / PER;
        const int piece = lane % LPR;  // 16 codes: two pieces of the 16-bit row
        uint4 kr[N], vr[N];
        float ks, vs;
        auto load = [&]() {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const long ro = __shfl_sync(0xffffffffu, off, i * PER + lane / LPR);
            kr[i] = vr[i] = make_uint4(0, 0, 0, 0);
            if (ro >= 0) {
              kr[i] = tj_ld16_stream(kbase + ro + piece * 16);
              vr[i] = tj_ld16_stream(vbase + ro + piece * 16);
            }
          }
          ks = vs = 0.0f;
          if (soff >= 0) {
            ks = __ldg(p.a.cache.k_scale + soff);
            vs = __ldg(p.a.cache.v_scale + soff);
          }
        };
        auto store = [&](uint8_t* dst, const uint4 (&raw)[N]) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int r = pw * 32 + i * PER + lane / LPR;
            uint32_t h[2][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = e == 0 ? raw[i].x : e == 1 ? raw[i].y : e == 2 ? raw[i].z : raw[i].w;
              h[e >> 1][(e & 1) * 2] = Codes<T, CD>::make(__byte_perm(x, 0, CD == TJ_I8 ? 0x4140 : 0x1404));
              h[e >> 1][(e & 1) * 2 + 1] = Codes<T, CD>::make(__byte_perm(x, 0, CD == TJ_I8 ? 0x4342 : 0x3424));
            }
            // at head dim 128 a row's lanes reach both panels, whose banks are the same: the upper
            // half stores its odd piece first
            const bool swap = D == 128 && piece >= LPR / 2;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int o = swap ? e ^ 1 : e;
              st_shared16(smem_u32(dst) + swizzled(TILE_KEYS, r, piece * 2 + o), swap ? h[e ^ 1][0] : h[e][0],
                          swap ? h[e ^ 1][1] : h[e][1], swap ? h[e ^ 1][2] : h[e][2], swap ? h[e ^ 1][3] : h[e][3]);
            }
          }
        };
        load();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        mbar_arrive(smem_u32(q_full));
        for (int j = 0; j < nb; ++j) {
          const int it = blocks + j, s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          look_up(j + 1, off, soff);
          ok = mbar_wait_warp(smem_u32(&k_empty[s]), ph ^ 1u, abort_flag, p.status, WHERE + 5);
          if (!ok) break;
          float* sc = scales + (it % C::SCALES) * 3 * TILE_KEYS + pw * 32 + lane;
          const float lv = fmaxf(__log2f(vs), MIN_LOG2_SCALE);
          sc[0] = ks * p.scale_log2;
          sc[TILE_KEYS] = lv;
          sc[2 * TILE_KEYS] = exp2_fast(-lv);
          store(sK + s * KV_BYTES, kr);
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(&k_full[s]));
          ok = mbar_wait_warp(smem_u32(&v_empty[s]), ph ^ 1u, abort_flag, p.status, WHERE + 6);
          if (!ok) break;
          store(sV + s * KV_BYTES, vr);
          fence_proxy_async_smem();
          mbar_arrive(smem_u32(&v_full[s]));
          if (j + 1 < nb) load();
        }
      }
    } else if constexpr (ROLE == Role::matrix) {
      if (warp == 12) {
      // ---------------- matrix instructions ----------------
      const uint64_t dq = desc_sw128(smem_u32(sQ), 16, 1024), dk = desc_sw128(smem_u32(sK), 16, 1024),
                     dv = desc_sw128(smem_u32(sV), TILE_KEYS * 128, 1024);
      bool ok = mbar_wait_warp(smem_u32(q_full), seg & 1, abort_flag, p.status, WHERE + 7);
      bool issued = false;
      auto scores = [&](int t, int s) {
        const uint64_t a = dq + ((t * Q_BYTES) >> 4), b = dk + ((s * KV_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t step = (k >> 2) * (128 * 128 >> 4) + (k & 3) * 2;
          umma_f16_elect(tmem + t * 128, a + step, b + step, IDESC_S, k > 0);
        }
        umma_commit_elect(smem_u32(&s_full[t]));
        issued = true;
      };
      auto values = [&](int t, int s, bool acc) {
        const uint64_t b = dv + ((s * KV_BYTES) >> 4);
#pragma unroll
        for (int k = 0; k < TILE_KEYS / 16; ++k)
          tja::umma_f16_ts_elect(tmem + 256 + t * D, tmem + t * 128 + k * 8, b + ((k * 16 * 128) >> 4), IDESC_O, (acc || k > 0) ? 1u : 0u);
      };
      if (ok) ok = mbar_wait_warp(smem_u32(&k_full[blocks % STAGES]), (blocks / STAGES) & 1, abort_flag, p.status, WHERE + 8);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < ntiles; ++t) scores(t, blocks % STAGES);
        umma_commit_elect(smem_u32(&k_empty[blocks % STAGES]));
      }
      for (int j = 0; j < nb && ok; ++j) {
        const int it = blocks + j, s = it % STAGES, s1 = (it + 1) % STAGES;
        ok = mbar_wait_warp(smem_u32(&v_full[s]), (it / STAGES) & 1, abort_flag, p.status, WHERE + 9);
        for (int t = 0; t < ntiles && ok; ++t) {
          ok = mbar_wait_warp(smem_u32(&p_ready[t]), ((t == 0 ? blocks : blocks1) + j) & 1, abort_flag, p.status, WHERE + 10);
          if (!ok) break;
          tc_fence_after();
          values(t, s, j > 0);
          if (t == ntiles - 1) umma_commit_elect(smem_u32(&v_empty[s]));
          if (j + 1 < nb) {
            if (t == 0) ok = mbar_wait_warp(smem_u32(&k_full[s1]), ((it + 1) / STAGES) & 1, abort_flag, p.status, WHERE + 8);
            if (!ok) break;
            tc_fence_after();
            scores(t, s1);
            if (t == ntiles - 1) umma_commit_elect(smem_u32(&k_empty[s1]));
          }
        }
      }
      if (ok) umma_commit_elect(smem_u32(o_done));
      if (!ok && issued) {
        umma_commit_elect(smem_u32(drain));
        volatile int no_abort = 0;
        mbar_wait_warp(smem_u32(drain), 0, &no_abort, p.status, WHERE + 11, 200000000ull);
      }
      }
    } else {
      // ---------------- softmax ----------------
      const int t = warp >> 2, q = warp & 3, r = t * 128 + q * 32 + lane;
      const uint32_t at = static_cast<uint32_t>(q * 32) << 16;
      const uint32_t tS = tmem + at + t * 128, tO = tmem + at + 256 + t * D;
      if (t < ntiles) {
        const int rr = min(r, rows - 1), tok = (r0 + rr) / p.group, hd = w.head * p.group + (r0 + rr) - tok * p.group;
        int rlo, rhi;
        row_range(p, w.s, tok, rlo, rhi);
        // keys that every row of this warp sees need no mask
        const int clo = __reduce_max_sync(0xffffffffu, rlo), chi = __reduce_min_sync(0xffffffffu, rhi);
        float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        bool ok = true;
        for (int j = 0; j < nb; ++j) {
          const int it = blocks + j, kb = key0 + j * TILE_KEYS;
          ok = mbar_wait_warp(smem_u32(&s_full[t]), ((t == 0 ? blocks : blocks1) + j) & 1, abort_flag, p.status, WHERE + 12);
          if (Q8 && ok)  // the scales were written before the keys' barrier
            ok = mbar_wait_warp(smem_u32(&k_full[it % STAGES]), (it / STAGES) & 1, abort_flag, p.status, WHERE + 12);
          if (!ok) break;
          tc_fence_after();
          uint32_t raw[128];
#pragma unroll
          for (int i = 0; i < 4; ++i) tja::tmem_ld32_async(tS + 32 * i, raw + 32 * i);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          float x[128];
#pragma unroll
          for (int i = 0; i < 128; ++i) {
            asm volatile("" : "+r"(raw[i]));  // not before the wait
            x[i] = __uint_as_float(raw[i]);
          }
          const float* sc = scales + (it % C::SCALES) * 3 * TILE_KEYS;
          if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < 128; i += 4) {
              const float4 k = *reinterpret_cast<const float4*>(sc + i), v = *reinterpret_cast<const float4*>(sc + TILE_KEYS + i);
              x[i] = fmaf(x[i], k.x, v.x);
              x[i + 1] = fmaf(x[i + 1], k.y, v.y);
              x[i + 2] = fmaf(x[i + 2], k.z, v.z);
              x[i + 3] = fmaf(x[i + 3], k.w, v.w);
            }
          }
          if (kb < clo || kb + TILE_KEYS > chi) {
            const int a = rlo - kb, b = rhi - kb;
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (i < a || i >= b) x[i] = -INFINITY;
          }
          float h0 = x[0], h1 = x[1], h2 = x[2], h3 = x[3];
#pragma unroll
          for (int i = 4; i < 124; i += 8) {
            h0 = tja::fmax3(h0, x[i], x[i + 4]);
            h1 = tja::fmax3(h1, x[i + 1], x[i + 5]);
            h2 = tja::fmax3(h2, x[i + 2], x[i + 6]);
            h3 = tja::fmax3(h3, x[i + 3], x[i + 7]);
          }
          h0 = tja::fmax3(h0, x[124], x[125]);
          h1 = tja::fmax3(h1, x[126], x[127]);
          const float c = Q8 ? 1.0f : p.scale_log2;
          const float top = tja::fmax3(h0, h1, fmaxf(h2, h3)) * c;
          float alpha = 1.0f;
          const bool raise = top > m + C::RAISE || (m == -INFINITY && top > m);
          if (raise) {
            alpha = exp2_fast(m - top);
            m = top;
            l0 *= alpha;
            l1 *= alpha;
          }
          const float base = (m == -INFINITY ? 0.0f : m) - C::SHIFT;
          const uint64_t cc = tja::f2_pack(c, c), nb2 = tja::f2_pack(-base, -base);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t pk[16];
            uint64_t ll = tja::f2_pack(l0, l1);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const int i = g * 32 + 2 * k;
              float e0, e1;
              if constexpr (Q8)
                tja::f2_unpack(tja::f2_add(tja::f2_pack(x[i], x[i + 1]), nb2), e0, e1);
              else
                tja::f2_unpack(tja::f2_fma(tja::f2_pack(x[i], x[i + 1]), cc, nb2), e0, e1);
              e0 = exp2_fast(e0);
              e1 = exp2_fast(e1);
              if constexpr (Q8) {
                const float2 inv = *reinterpret_cast<const float2*>(sc + 2 * TILE_KEYS + i);
                ll = tja::f2_fma(tja::f2_pack(e0, e1), tja::f2_pack(inv.x, inv.y), ll);
              } else {
                ll = tja::f2_add(ll, tja::f2_pack(e0, e1));
              }
              pk[k] = pack2<T>(e0, e1);
            }
            tja::f2_unpack(ll, l0, l1);
            tja::tmem_st16(tS + 16 * g, pk);
          }
          if (j > 0 && __any_sync(0xffffffffu, raise)) {
            // the scores' barrier followed the previous product's, so O is at rest
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              float o[32];
              tmem_ld32(tO + i, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= alpha;
              tja::tmem_st32_wait(tO + i, o);
            }
          }
          tja::tmem_wait_st();
          tc_fence_before();
          mbar_arrive(smem_u32(&p_ready[t]));
        }
        if (ok) ok = mbar_wait_warp(smem_u32(o_done), seg & 1, abort_flag, p.status, WHERE + 13);
        if (ok) {
          tc_fence_after();
          const float l = l0 + l1;
          if (l != l && m == -INFINITY) m = 0.0f;  // only NaN scores: the row is NaN, not empty
          const bool none = m == -INFINITY;
          if (whole) {
            const float inv = none ? 0.0f : 1.0f / l;
            T* dst = static_cast<T*>(p.a.out) + (w.s.start + tok) * p.a.out_token + hd * p.a.out_head;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              float o[32];
              tmem_ld32(tO + i, o);
              if (r < rows) {
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = none ? 0.0f : o[k] * inv;
#pragma unroll
                for (int k = 0; k < 32; k += 8) tj_store_vec(dst + i + k, o + k);
              }
            }
            if (p.a.lse && r < rows)
              p.a.lse[(w.s.start + tok) * p.a.q_heads + hd] = none ? -INFINITY : (m - C::SHIFT + log2f(l)) * 0.69314718055994531f;
          } else {
            const long slot = (2L * blockIdx.x + (a0 > 0 ? 0 : 1)) * TILE_ROWS + r;
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              float o[32];
              tmem_ld32(tO + i, o);
              if (r < rows)
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                  __stcg(reinterpret_cast<float4*>(p.part_o + slot * D + i + k), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
            }
            if (r < rows) __stcg(p.part_ml + slot, make_float2(m, l));
          }
          tc_fence_before();
        }
      }
    }
    ++seg;
    blocks += nb;
    if (ntiles == 2) blocks1 += nb;
    __syncwarp();
    if (!whole) __threadfence();
    __syncthreads();
    tc_fence_after();
    failed = *abort_flag != 0;
    if (!whole && !failed) {
      const int c0 = static_cast<int>(((w.start + 1) * parts - 1) / total),
                c1 = static_cast<int>(((w.start + w.weight) * parts - 1) / total);
      if (threadIdx.x == 0) {
        const int done = atomicAdd(p.counters + c0, nb) + nb;
        *s_last = done == all;
        if (done == all) p.counters[c0] = 0;  // ready for the next call
      }
      __syncthreads();
      if (*s_last) {
        __threadfence();
        constexpr int V4 = D / 4;
        for (int e = threadIdx.x; e < rows * V4; e += 512) {
          const int r = e / V4, col = (e - r * V4) * 4;
          float best = -INFINITY, sum = 0.0f;
          float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int c = c0; c <= c1; ++c) {
            const long pc = total * c / parts, b0 = max(0L, pc - w.start), b1 = min(w.weight, total * (c + 1) / parts - w.start);
            if (b0 * all / w.weight == b1 * all / w.weight) continue;
            const long slot = (2L * c + (b0 > 0 ? 0 : 1)) * TILE_ROWS + r;
            const float2 ml = __ldcg(p.part_ml + slot);
            if (ml.x == -INFINITY) continue;
            const float next = fmaxf(best, ml.x), f = exp2_fast(best - next), g = exp2_fast(ml.x - next);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + col));
            acc = make_float4(acc.x * f + v.x * g, acc.y * f + v.y * g, acc.z * f + v.z * g, acc.w * f + v.w * g);
            sum = sum * f + ml.y * g;
            best = next;
          }
          const bool none = best == -INFINITY;
          const float inv = none ? 0.0f : 1.0f / sum;
          const int tok = (r0 + r) / p.group, hd = w.head * p.group + (r0 + r) - tok * p.group;
          T* dst = static_cast<T*>(p.a.out) + (w.s.start + tok) * p.a.out_token + hd * p.a.out_head + col;
          uint2 y;
          y.x = pack2<T>(none ? 0.0f : acc.x * inv, none ? 0.0f : acc.y * inv);
          y.y = pack2<T>(none ? 0.0f : acc.z * inv, none ? 0.0f : acc.w * inv);
          *reinterpret_cast<uint2*>(dst) = y;
          if (p.a.lse && col == 0)
            p.a.lse[(w.s.start + tok) * p.a.q_heads + hd] = none ? -INFINITY : (best - C::SHIFT + log2f(sum)) * 0.69314718055994531f;
        }
      }
    }
  }
}

template <class T, int CD, int D>
__global__ void __launch_bounds__(512, 1) attention_tiles(const __grid_constant__ AttnParams p) {
  using namespace tjg;
  using C = Tiles<T, CD, D>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  TilesShared<T, CD, D> sh(smem_raw);
  const int warp = threadIdx.x >> 5;
  sh.total = total_work(p);
  sh.parts = min(static_cast<long>(gridDim.x), max(1L, sh.total / (4L * TILE_KEYS * p.group)));
  if (sh.total == 0 || blockIdx.x >= sh.parts) return;
  sh.from = sh.total * blockIdx.x / sh.parts;
  sh.to = sh.total * (blockIdx.x + 1) / sh.parts;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(sh.q_full), 128);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(smem_u32(&sh.k_full[s]), 128);
      mbar_init(smem_u32(&sh.v_full[s]), 128);
      mbar_init(smem_u32(&sh.k_empty[s]), 1);
      mbar_init(smem_u32(&sh.v_empty[s]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&sh.s_full[t]), 1);
      mbar_init(smem_u32(&sh.p_ready[t]), 128);
    }
    mbar_init(smem_u32(sh.o_done), 1);
    mbar_init(smem_u32(sh.drain), 1);
    *sh.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(sh.tmem_slot), C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *sh.tmem_slot;
  // 512 threads of 128 registers at launch: 2 x 168 + 112 + 64 = 4 x 128 of them afterwards
  if (warp < 8) {
    regs_inc<168>();
    tiles_role<Role::softmax, T, CD, D>(p, sh, tmem);
  } else if (warp < 12) {
    regs_dec<112>();
    tiles_role<Role::producer, T, CD, D>(p, sh, tmem);
  } else {
    regs_dec<64>();
    tiles_role<Role::matrix, T, CD, D>(p, sh, tmem);
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, C::TMEM);
}

}  // namespace tjs
