// Rotary positions, and the paged cache's writes and reads: everything a decoder does to the
// rows (token, head) of its queries, keys and values besides attending.
//
// Mathematics.  A row's first `rot` elements are rot / 2 pairs, (2i, 2i + 1) or (i, i + rot / 2);
// each is turned by the angle of the token's position and the pair's frequency, whose cosine and
// sine the table holds in f32:  a' = a c - b s,  b' = b c + a s  (inverse: s -> -s, which is also
// the gradient).  A quantised cache keeps, of each row, x = code * scale with scale = max|x| / 127
// (i8, code = x / scale to the nearest even integer) or max|x| / 448 (e4m3, code rounded to
// nearest even).  Products and the sum are rounded one by one (no FMA) and quotients are IEEE
// divisions, so the codes are the same for every layout of the work and equal those of the same
// formulas evaluated elementwise in f32.
//
// One kernel does them all, because they read the same rows: with rotary positions and a cache
// write in one launch the rotated keys never travel through memory, and single-token steps, whose
// cost is the launch, pay for one.
//
// Layout.  A row is cut into slots of two 8-element units; a lane holds one slot, so a rotary
// pair (half layout: units u and u + rot / 16) is in one lane's registers, max|x| is a shuffle
// over the row's lanes, and every access is 16 bytes.  Neighbouring lanes hold neighbouring units.  A lane keeps its slot's cosines and sines
// in registers over the heads of its token: the table is read once per token, not once per row.
// A warp takes 32 / lanes rows at a time and loads four such groups, unconverted, before it looks anything
// up: the kernel is bound by HBM, and so by the reads in flight.  Measured for 16384 tokens of 40 f16
// heads of 128 (us): four groups and 24 warps an SM 69, four and 20 72, two and 32 73, one and 32 86; with four
// more groups in flight while these are stored, which leaves registers for 12 warps, 71.
#include <algorithm>

#include "serving_common.cuh"

static __device__ __align__(16) int tj_serving_words[4];

namespace tjs {

struct RowsParams {
  tj_rows a;
  int* status;
  int lanes_log2;  // lanes of a row
  int slots;       // slots of a row: ceil(dim / 16)
  int iters;       // warp iterations over a token's rows; times the number of warps that share it below 2^32
  Div segs;        // warps that share a token
  Div page;        // slots of a page
  int op;
};

// a plain (coherent) load that stays out of L1: rows are read once, and may be written in place
TJ_DEV uint4 ld16_row(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
// a unit of 8 elements as it is read
template <class T> struct Unit {
  uint4 v[sizeof(T) / 2];
  TJ_DEV void load(const T* p) {
    v[0] = ld16_row(p);
    if constexpr (sizeof(T) == 4) v[1] = ld16_row(p + 4);
  }
  TJ_DEV void get(float* f) const {
    tj_unpack(v[0], f, (const T*)nullptr);
    if constexpr (sizeof(T) == 4) tj_unpack(v[1], f + 4, (const T*)nullptr);
  }
};
TJ_DEV void store8(float* p, const float* f) {
  tj_store_vec(p, f);
  tj_store_vec(p + 4, f + 4);
}
template <class T> TJ_DEV void store8(T* p, const float* f) { tj_store_vec(p, f); }

TJ_DEV uint32_t e4m3x4(const float* f) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
TJ_DEV uint32_t i8x4(const float* f) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= static_cast<uint32_t>(max(-127, min(127, __float2int_rn(f[i]))) & 0xff) << (8 * i);
  return w;
}

// ROT: 0 none; 1 half layout, whole units; 2 interleaved, whole units; 3 either, any even rot
// (pairs that cross units: partners and table entries one by one).
// CACHE: 0 none, 1 a 16-bit one, 2 i8, 3 e4m3.
template <class T, int ROT, int CACHE>
__global__ void __launch_bounds__(128, ROT == 3 ? 2 : 6) rows_kernel(const __grid_constant__ RowsParams p) {
  const tj_rows& a = p.a;
  const int lane = threadIdx.x & 31, wid = static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int token = p.segs(wid), seg = wid - token * static_cast<int>(p.segs.d);
  if (token >= a.tokens) return;
  const int dim = static_cast<int>(a.dim), rot = static_cast<int>(a.rot), half = rot >> 1;
  const int lpr = 1 << p.lanes_log2, sub = lane >> p.lanes_log2, per = 32 >> p.lanes_log2, s = lane & (lpr - 1);
  const bool on = s < p.slots;

  // the slot's two units
  int ua = s, ub = s + p.slots;
  if (ROT == 1) {
    const int pairs = rot >> 4;
    ua = s < pairs ? s : s + pairs;
    ub = s < pairs ? s + pairs : s + p.slots;
  }
  const bool has_b = on && ub * 8 < dim;

  const int nq = a.q ? static_cast<int>(a.q_heads) : 0, nk = a.k ? static_cast<int>(a.kv_heads) : 0,
            nv = a.v ? static_cast<int>(a.kv_heads) : 0;
  const int rows = nq + nk + nv;
  const T* const q = static_cast<const T*>(a.q) + token * a.q_token;
  const T* const k = static_cast<const T*>(a.k) + token * a.k_token;
  const T* const v = static_cast<const T*>(a.v) + token * a.v_token;
  auto source = [&](int r) { return r < nq ? q + r * a.q_head : r < nq + nk ? k + (r - nq) * a.k_head : v + (r - nq - nk) * a.v_head; };
  constexpr int BATCH = sizeof(T) == 4 ? 2 : 4;
  Unit<T> raw[BATCH][2];
  const int segs = static_cast<int>(p.segs.d);
  const int i0 = static_cast<int>(static_cast<unsigned>(seg) * p.iters / segs), i1 = static_cast<int>(static_cast<unsigned>(seg + 1) * p.iters / segs);
  auto load = [&](int it) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int r = (it + j) * per + sub;
      if (it + j < i1 && r < rows && on) {
        const T* src = source(r);
        raw[j][0].load(src + ua * 8);
        if (has_b) raw[j][1].load(src + ub * 8);
      }
    }
  };
  load(i0);  // in flight while the table's row and the slot are looked up

  float cs[8] = {}, sn[8] = {};
  const float* trow = nullptr;
  bool lost = false;  // a position outside the table: the row becomes NaN
  if constexpr (ROT != 0) {
    const int pos = a.positions[token];
    lost = pos < 0 || pos >= a.table_rows;
    if (lost && lane == 0) tj_report(p.status, TJ_STATUS_BOUNDS, p.op * 16 + SITE_POSITION);
    trow = a.table + (lost ? 0 : static_cast<long>(pos) * rot);
    const float sign = a.inverse ? -1.0f : 1.0f;
    if (ROT == 1 && on && ua * 8 < half) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        tj_unpack(tj_ld16(trow + ua * 8 + i), cs + i, (const float*)nullptr);
        tj_unpack(tj_ld16(trow + half + ua * 8 + i), sn + i, (const float*)nullptr);
      }
    }
    if (ROT == 2 && on) {  // unit u holds pairs 4u .. 4u + 3
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int u = i ? ub : ua;
        if (u * 8 < rot) {
          tj_unpack(tj_ld16(trow + u * 4), cs + 4 * i, (const float*)nullptr);
          tj_unpack(tj_ld16(trow + half + u * 4), sn + 4 * i, (const float*)nullptr);
        }
      }
    }
    if (ROT != 3) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sn[i] *= sign;
        if (lost) cs[i] = sn[i] = __int_as_float(0x7fffffff);
      }
    }
  }
  long crow = -1, srow = 0;
  if constexpr (CACHE != 0) {
    const int slot = a.slots[token];
    const long cap = a.cache.pages * a.cache.page_size;
    if (slot >= 0 && slot < cap) {
      const int page = p.page(slot), at = slot - page * static_cast<int>(p.page.d);
      crow = page * a.cache.page_stride + at * a.cache.slot_stride;
      srow = page * a.cache.scale_page + at * a.cache.scale_slot;
    } else if (slot >= cap && lane == 0) {
      tj_report(p.status, TJ_STATUS_BOUNDS, p.op * 16 + SITE_SLOT);
    }
  }

  for (int it = i0; it < i1; it += BATCH) {
    if (it != i0) load(it);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const int r = (it + j) * per + sub;
      if (it + j >= i1) break;
      const bool mine = r < rows && on;
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.0f;
      if (mine) {
        raw[j][0].get(x);
        if (has_b) raw[j][1].get(x + 8);
      }
      if (ROT == 1 && r < nq + nk && ua * 8 < half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = x[i], w = x[i + 8];
          x[i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(w, sn[i]));
          x[i + 8] = __fadd_rn(__fmul_rn(w, cs[i]), __fmul_rn(u, sn[i]));
        }
      }
      if (ROT == 2 && r < nq + nk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if ((i < 4 ? ua : ub) * 8 < rot) {
            const float u = x[2 * i], w = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(w, sn[i]));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(w, cs[i]), __fmul_rn(u, sn[i]));
          }
        }
      }
      if constexpr (ROT == 3) {
        if (mine && r < nq + nk) {
          const T* src = source(r);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int e = (i < 8 ? ua : ub) * 8 + (i & 7);
            if (e >= rot || (i >= 8 && !has_b)) continue;
            const bool second = a.interleaved ? (e & 1) : e >= half;
            const int pair = a.interleaved ? e >> 1 : (second ? e - half : e);
            const int other = a.interleaved ? e ^ 1 : (second ? e - half : e + half);
            float c = trow[pair], sv = trow[half + pair] * (a.inverse ? -1.0f : 1.0f);
            if (lost) c = sv = __int_as_float(0x7fffffff);
            // read again: the partner may be in another lane, and x is overwritten in place
            const float mate = tj_f32(src[other]), own = tj_f32(src[e]);
            x[i] = second ? __fadd_rn(__fmul_rn(own, c), __fmul_rn(mate, sv)) : __fsub_rn(__fmul_rn(own, c), __fmul_rn(mate, sv));
          }
        }
        __syncwarp();  // every lane has read the row before any lane stores over it (outputs in place)
      }
      if (CACHE == 0 || r < nq) {
        if (mine) {
          T* dst = r < nq ? static_cast<T*>(a.q_out) + token * a.qo_token + r * a.qo_head
                          : static_cast<T*>(a.k_out) + token * a.ko_token + (r - nq) * a.ko_head;
          store8(dst + ua * 8, x);
          if (has_b) store8(dst + ub * 8, x + 8);
        }
      }
      if constexpr (CACHE != 0) {
        const bool key = r < nq + nk, put = mine && r >= nq && crow >= 0;
        const int h = key ? r - nq : r - nq - nk;
        void* base = key ? a.cache.k : a.cache.v;
        const long off = crow + h * a.cache.head_stride;
        if constexpr (CACHE == 1) {
          if (put) {
            if (a.cache.dtype == TJ_BF16) {
              store8(static_cast<__nv_bfloat16*>(base) + off + ua * 8, x);
              if (has_b) store8(static_cast<__nv_bfloat16*>(base) + off + ub * 8, x + 8);
            } else {
              store8(static_cast<__half*>(base) + off + ua * 8, x);
              if (has_b) store8(static_cast<__half*>(base) + off + ub * 8, x + 8);
            }
          }
        } else {
          // max|x| over the row's lanes, as bits: an infinity or a NaN orders above every number
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
          for (int o = lpr >> 1; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          float scale = __fdiv_rn(__uint_as_float(top), CACHE == 2 ? 127.0f : 448.0f);
          if (put) {
            // a row with an infinity or a NaN is held as NaN (scale) times zero codes
            const bool bad = top >= 0x7f800000u;
            if (bad) scale = __int_as_float(0x7fffffff);
            const bool zero = bad || scale == 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = zero ? 0.0f : __fdiv_rn(x[i], scale);
            uint8_t* dst = static_cast<uint8_t*>(base) + off;
            uint2 w0, w1;
            if (CACHE == 2) {
              w0 = make_uint2(i8x4(x), i8x4(x + 4));
              w1 = make_uint2(i8x4(x + 8), i8x4(x + 12));
            } else {
              w0 = make_uint2(e4m3x4(x), e4m3x4(x + 4));
              w1 = make_uint2(e4m3x4(x + 8), e4m3x4(x + 12));
            }
            *reinterpret_cast<uint2*>(dst + ua * 8) = w0;
            if (has_b) *reinterpret_cast<uint2*>(dst + ub * 8) = w1;
            if (s == 0) (key ? a.cache.k_scale : a.cache.v_scale)[srow + h * a.cache.scale_head] = scale;
          }
        }
      }
    }
  }
}

struct ReadParams {
  tj_kv_cache c;
  const int* slots;
  void* out[2];
  int rows;  // n * heads
  int* status;
  int lanes_log2;  // lanes of a row: a lane holds 8 elements (64: two rounds of a warp)
  int group;       // rows of a warp, 32 at the most
  Div heads, page;
};

// Rows (slot, head) of the keys and of the values back as T: value = code * scale in f32, rounded
// once.  CD: the cache's dtype.  A slot of -1 reads as zeros.  A lane holds eight elements, so that both
// its reads and its writes are contiguous with its neighbours'.  Where a row is takes more instructions than
// converting eight elements, so each lane looks one row of the warp's up and hands its address round:
// 32768 slots of 8 heads of 128 i8 codes take 36 us, 46 when every lane looks its rows up.
template <class T, int CD>
__global__ void __launch_bounds__(128) read_kernel(const __grid_constant__ ReadParams p) {
  constexpr int BATCH = 4, ES = CD == TJ_I8 || CD == TJ_E4M3 ? 1 : 2;
  using Raw = typename std::conditional<ES == 1, uint2, uint4>::type;
  const int lane = threadIdx.x & 31, dim = static_cast<int>(p.c.dim);
  const int lanes = min(p.lanes_log2, 5), sub = lane >> lanes, per = 32 >> lanes, s0 = lane & ((1 << lanes) - 1);
  const bool val = blockIdx.y;
  T* const out = static_cast<T*>(p.out[val]);
  const int first = (static_cast<int>(blockIdx.x) * 4 + (threadIdx.x >> 5)) * p.group, n = min(p.group, p.rows - first);
  if (n <= 0) return;

  long address = 0;  // 0: zeros
  float scale = 1.0f;
  if (lane < n) {
    const int token = p.heads(first + lane), head = first + lane - token * static_cast<int>(p.heads.d), slot = __ldg(p.slots + token);
    if (slot >= static_cast<int>(p.c.pages * p.c.page_size)) {
      tj_report(p.status, TJ_STATUS_BOUNDS, OP_CACHE_READ * 16 + SITE_SLOT);
    } else if (slot >= 0) {
      const int page = p.page(slot), at = slot - page * static_cast<int>(p.page.d);
      address = reinterpret_cast<long>(val ? p.c.v : p.c.k) + (page * p.c.page_stride + at * p.c.slot_stride + head * p.c.head_stride) * ES;
      if (ES == 1) scale = __ldg((val ? p.c.v_scale : p.c.k_scale) + page * p.c.scale_page + at * p.c.scale_slot + head * p.c.scale_head);
    }
  }
  for (int s = s0; s < (1 << p.lanes_log2); s += 32) {
    const bool on = s * 8 < dim;
    for (int from = 0; from < n; from += BATCH * per) {
      Raw raw[BATCH];
      float factor[BATCH];
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int r = min(from + j * per + sub, 31);
        const long src = __shfl_sync(0xffffffffu, address, r);
        factor[j] = __shfl_sync(0xffffffffu, scale, r);
        raw[j] = Raw{};
        if (src && on && from + j * per + sub < n) raw[j] = __ldg(reinterpret_cast<const Raw*>(src + s * 8 * ES));
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int r = from + j * per + sub;
        if (r >= n || !on) continue;
        float x[8];
        if constexpr (CD == TJ_BF16) {
          tj_unpack(raw[j], x, (const __nv_bfloat16*)nullptr);
        } else if constexpr (CD == TJ_F16) {
          tj_unpack(raw[j], x, (const __half*)nullptr);
        } else {
          const uint32_t w[2] = {raw[j].x, raw[j].y};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t lo, hi;  // exact in f16
            codes4<__half, CD>(w[i], lo, hi);
            const float2 a = __half22float2(reinterpret_cast<const __half2&>(lo)), b = __half22float2(reinterpret_cast<const __half2&>(hi));
            x[4 * i] = a.x * factor[j];
            x[4 * i + 1] = a.y * factor[j];
            x[4 * i + 2] = b.x * factor[j];
            x[4 * i + 3] = b.y * factor[j];
          }
        }
        store8(out + static_cast<long>(first + r) * dim + s * 8, x);
      }
    }
  }
}

// 64-bit indices as 32-bit ones.  What does not fit saturates, so that it stays out of every range that the operators
// check; cut off to its low half it would be another, valid index.
__global__ void __launch_bounds__(256) narrow_kernel(const int64_t* src, long n, long cols, long row_stride, long col_stride, int32_t* dst) {
  const long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const long r = i / cols, c = i - r * cols, v = src[r * row_stride + c * col_stride];
  dst[i] = static_cast<int32_t>(max(-0x7fffffffL, min(0x7fffffffL, v)));
}

struct Setup {
  std::once_flag once;
  Device dev{};
  cudaError_t err = cudaSuccess;
};
Setup g_devices[MAX_DEVICES];

int current_device(Device* out) {
  int d = 0;
  const cudaError_t e = cudaGetDevice(&d);
  if (e != cudaSuccess) return refuse(TJ_ERR_CUDA, "serving", cudaGetErrorString(e));
  if (d < 0 || d >= MAX_DEVICES) return refuse(TJ_ERR_INVALID, "serving", "device index out of range");
  Setup& s = g_devices[d];
  try {
    std::call_once(s.once, [&] {
      void* w = nullptr;
      s.err = cudaGetSymbolAddress(&w, tj_serving_words);
      if (s.err == cudaSuccess) s.err = cudaDeviceGetAttribute(&s.dev.sms, cudaDevAttrMultiProcessorCount, d);
      s.dev.index = d;
      s.dev.status = static_cast<int*>(w);
    });
  } catch (...) {  // nothing may pass a C entry
    return refuse(TJ_ERR_CUDA, "serving", "the device's set-up failed");
  }
  if (s.err != cudaSuccess) return refuse(TJ_ERR_CUDA, "serving", cudaGetErrorString(s.err));
  *out = s.dev;
  return TJ_OK;
}

const char* rows_fault(const tj_rows& a, bool write) {
  if (a.dtype != TJ_F32 && a.dtype != TJ_F16 && a.dtype != TJ_BF16) return "rows must be f32, f16 or bf16";
  if (a.tokens < 0 || a.q_heads < 0 || a.kv_heads < 0) return "negative extent";
  if (a.dim <= 0 || a.dim % 8 || a.dim > 512) return "head dim must be a multiple of 8, at most 512";
  if (a.rot < 0 || a.rot % 2 || a.rot > a.dim) return "rot must be even, from 0 to the head dim";
  if (a.rot && (!a.positions || !a.table || a.table_rows <= 0)) return "rotary positions need positions and a table";
  if (a.q && !a.q_out) return "q needs an output";
  const int unit = 16 / element_size(a.dtype);
  const auto bad = [&](const void* p, int64_t t, int64_t h) {
    return p && (reinterpret_cast<uintptr_t>(p) % 16 || t % unit || h % unit);
  };
  if (bad(a.q, a.q_token, a.q_head) || bad(a.k, a.k_token, a.k_head) || bad(a.v, a.v_token, a.v_head) ||
      bad(a.q_out, a.qo_token, a.qo_head) || bad(a.k_out, a.ko_token, a.ko_head) || reinterpret_cast<uintptr_t>(a.table) % 16)
    return "rows must start on 16-byte boundaries";
  if (write) {
    if (!a.k || !a.v || !a.slots) return "a cache write needs k, v and slots";
    if (a.cache.dim != a.dim || a.cache.heads != a.kv_heads) return "k and v do not have the cache's heads and head dim";
    return cache_fault(a.cache);
  }
  if (!a.q && !a.k) return "nothing to rotate";
  if (a.v || a.slots) return "a rotation takes neither v nor slots";
  if (a.k && !a.k_out) return "k needs an output";
  if (!a.rot) return "rot must be positive";
  return nullptr;
}

template <class T, int ROT> void launch_cache(const RowsParams& p, bool write, unsigned grid, cudaStream_t st) {
  if (!write) {
    if constexpr (ROT != 0) rows_kernel<T, ROT, 0><<<grid, 128, 0, st>>>(p);
  } else if (p.a.cache.dtype == TJ_I8) {
    rows_kernel<T, ROT, 2><<<grid, 128, 0, st>>>(p);
  } else if (p.a.cache.dtype == TJ_E4M3) {
    rows_kernel<T, ROT, 3><<<grid, 128, 0, st>>>(p);
  } else {
    rows_kernel<T, ROT, 1><<<grid, 128, 0, st>>>(p);
  }
}
template <class T> void launch_rows(const RowsParams& p, int mode, bool write, unsigned grid, cudaStream_t st) {
  switch (mode) {
    case 0: launch_cache<T, 0>(p, write, grid, st); break;
    case 1: launch_cache<T, 1>(p, write, grid, st); break;
    case 2: launch_cache<T, 2>(p, write, grid, st); break;
    default: launch_cache<T, 3>(p, write, grid, st); break;
  }
}

int run_rows(const char* name, int op, const tj_rows* a, bool write, void* stream) {
  if (!a) return refuse(TJ_ERR_INVALID, name, "NULL arguments");
  if (const char* why = rows_fault(*a, write)) return refuse(TJ_ERR_INVALID, name, why);
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  const long rows = (a->q ? a->q_heads : 0) + (a->k ? a->kv_heads : 0) + (a->v ? a->kv_heads : 0);
  if (a->tokens == 0 || rows == 0) return TJ_OK;
  RowsParams p;
  p.a = *a;
  p.status = dev.status;
  p.op = op;
  p.slots = static_cast<int>((a->dim + 15) / 16);
  int mode = 0;
  if (a->rot) mode = a->interleaved ? (a->rot % 8 ? 3 : 2) : (a->rot % 16 ? 3 : 1);
  if (mode == 1) p.slots = static_cast<int>(a->rot / 16 + ((a->dim - a->rot) / 8 + 1) / 2);
  p.lanes_log2 = 0;
  while ((1 << p.lanes_log2) < p.slots) ++p.lanes_log2;
  if (rows > 0x40000000L) return refuse(TJ_ERR_INVALID, name, "too many rows");
  const int per = 32 >> p.lanes_log2;
  p.iters = static_cast<int>((rows + per - 1) / per);
  // four groups a warp; with few tokens one each, so that the rows of a single-token step spread over the
  // multiprocessors
  const bool few = a->tokens * p.iters < 16L * dev.sms;
  const int segs = static_cast<int>(std::min<long>(few ? p.iters : (p.iters + 3) / 4, 0xffffffffL / p.iters));
  p.segs = Div(static_cast<uint32_t>(segs));
  p.page = Div(write ? static_cast<uint32_t>(a->cache.page_size) : 1u);
  const long warps = a->tokens * segs, grid = (warps + 3) / 4;
  if (warps > 0x7fffff00L) return refuse(TJ_ERR_INVALID, name, "too many rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == TJ_F32)
    launch_rows<float>(p, mode, write, static_cast<unsigned>(grid), st);
  else if (a->dtype == TJ_F16)
    launch_rows<__half>(p, mode, write, static_cast<unsigned>(grid), st);
  else
    launch_rows<__nv_bfloat16>(p, mode, write, static_cast<unsigned>(grid), st);
  return launched(name);
}

template <class T> void launch_read(const ReadParams& p, dim3 grid, cudaStream_t st) {
  switch (p.c.dtype) {
    case TJ_F16: read_kernel<T, TJ_F16><<<grid, 128, 0, st>>>(p); break;
    case TJ_BF16: read_kernel<T, TJ_BF16><<<grid, 128, 0, st>>>(p); break;
    case TJ_I8: read_kernel<T, TJ_I8><<<grid, 128, 0, st>>>(p); break;
    default: read_kernel<T, TJ_E4M3><<<grid, 128, 0, st>>>(p); break;
  }
}

}  // namespace tjs

extern "C" int tj_b200_rotary(const tj_rows* args, void* stream) {
  return tjs::run_rows("tj_b200_rotary", tjs::OP_ROTARY, args, false, stream);
}

extern "C" int tj_b200_cache_write(const tj_rows* args, void* stream) {
  return tjs::run_rows("tj_b200_cache_write", tjs::OP_CACHE_WRITE, args, true, stream);
}

extern "C" int tj_b200_cache_read(const tj_kv_cache* cache, const int32_t* slots, int64_t count, void* k_out, void* v_out,
                                  int32_t dtype, void* stream) {
  using namespace tjs;
  const char* name = "tj_b200_cache_read";
  if (!cache) return refuse(TJ_ERR_INVALID, name, "NULL cache");
  if (const char* why = cache_fault(*cache)) return refuse(TJ_ERR_INVALID, name, why);
  if (dtype != TJ_F32 && dtype != TJ_F16 && dtype != TJ_BF16) return refuse(TJ_ERR_INVALID, name, "rows must be f32, f16 or bf16");
  if (count < 0) return refuse(TJ_ERR_INVALID, name, "negative extent");
  if (count == 0) return TJ_OK;
  if (!slots || !k_out || !v_out) return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16)
    return refuse(TJ_ERR_INVALID, name, "rows must start on 16-byte boundaries");
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  ReadParams p;
  p.c = *cache;
  p.slots = slots;
  p.out[0] = k_out;
  p.out[1] = v_out;
  if (count > 0x7fff0000LL / cache->heads) return refuse(TJ_ERR_INVALID, name, "too many rows");
  p.rows = static_cast<int>(count * cache->heads);
  p.heads = Div(static_cast<uint32_t>(cache->heads));
  p.page = Div(static_cast<uint32_t>(cache->page_size));
  p.status = dev.status;
  p.lanes_log2 = 0;
  while ((8 << p.lanes_log2) < cache->dim) ++p.lanes_log2;
  // 32 rows a warp; with few rows what a warp has in flight at once, so that they spread
  const long at_once = 4L * std::max(1, 32 >> p.lanes_log2);
  p.group = static_cast<int>(p.rows >= 32L * 16 * dev.sms ? 32 : std::min(32L, at_once));
  const long grid = (p.rows + 4L * p.group - 1) / (4L * p.group);
  const dim3 g(static_cast<unsigned>(grid), 2);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TJ_F32)
    launch_read<float>(p, g, st);
  else if (dtype == TJ_F16)
    launch_read<__half>(p, g, st);
  else
    launch_read<__nv_bfloat16>(p, g, st);
  return launched(name);
}

extern "C" int tj_b200_narrow_indices(const int64_t* src, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int32_t* dst,
                                      void* stream) {
  using namespace tjs;
  const char* name = "tj_b200_narrow_indices";
  if (rows < 0 || cols < 0) return refuse(TJ_ERR_INVALID, name, "negative extent");
  if (rows == 0 || cols == 0) return TJ_OK;
  if (!src || !dst) return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  if (rows > 0x7fffffffLL * 256 / cols) return refuse(TJ_ERR_INVALID, name, "too many indices");
  narrow_kernel<<<static_cast<unsigned>((rows * cols + 255) / 256), 256, 0, static_cast<cudaStream_t>(stream)>>>(src, rows * cols, cols, row_stride,
                                                                                                               col_stride, dst);
  return launched(name);
}

// Waits for `stream`, reads the status words back and clears them.
extern "C" int tj_b200_serving_status(int32_t* code, int32_t* where, void* stream) {
  using namespace tjs;
  const char* name = "tj_b200_serving_status";
  if (!code || !where) return refuse(TJ_ERR_INVALID, name, "NULL pointer");
  *code = *where = 0;
  Device dev;
  if (const int rc = current_device(&dev)) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  int words[4] = {0, 0, 0, 0};
  cudaError_t e = cudaMemcpyAsync(words, dev.status, sizeof(words), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && words[0]) {
    e = cudaMemsetAsync(dev.status, 0, sizeof(words), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) return refuse(TJ_ERR_CUDA, name, cudaGetErrorString(e));
  *code = words[0];
  *where = words[1];
  if (!words[0]) return TJ_OK;
  return refuse(TJ_ERR_DEVICE_STATUS, name, "a kernel met an index out of range");
}
