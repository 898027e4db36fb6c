// Shared by the serving operators (rotary positions, paged cache, attention over the cache):
// argument checks, the device status words, and the 8-bit cache formats.
#pragma once
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdio>
#include <mutex>
#include <type_traits>

#include "../../../include/tj_b200.h"
#include "../kernels/tj_common.cuh"

// defined in tj_b200_runtime.cpp (same library, not exported)
void tj_b200_internal_set_error(const char* msg);

namespace tjs {

constexpr int MAX_DEVICES = 64;

// Where a status word's `where` points: operator * 16 + site.
enum : int { SITE_SLOT = 1, SITE_POSITION = 2, SITE_PAGE = 3, SITE_LENGTH = 4, SITE_STARTS = 6 };
enum : int { OP_ROTARY = 0, OP_CACHE_WRITE = 1, OP_CACHE_READ = 2, OP_ATTENTION = 3 };

// cache_rows.cu: the current device's status words and its multiprocessor count.
struct Device {
  int index;
  int* status;
  int sms;
};
int current_device(Device* out);

inline int refuse(int code, const char* op, const char* why) {
  char buf[512];
  snprintf(buf, sizeof(buf), "%s: %s", op, why);
  tj_b200_internal_set_error(buf);
  return code;
}
inline int launched(const char* op) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? TJ_OK : refuse(TJ_ERR_CUDA, op, cudaGetErrorString(e));
}

inline int element_size(int64_t dtype) {
  switch (dtype) {
    case TJ_F32: return 4;
    case TJ_F16: case TJ_BF16: return 2;
    case TJ_I8: case TJ_E4M3: return 1;
  }
  return 0;
}

// NULL if the cache's description is sound, else what is wrong with it.
inline const char* cache_fault(const tj_kv_cache& c) {
  if (!c.k || !c.v) return "NULL cache pointer";
  if (c.dtype != TJ_F16 && c.dtype != TJ_BF16 && c.dtype != TJ_I8 && c.dtype != TJ_E4M3) return "bad cache dtype";
  const bool quantised = c.dtype == TJ_I8 || c.dtype == TJ_E4M3;
  if (quantised != (c.k_scale != nullptr) || quantised != (c.v_scale != nullptr))
    return "an i8 or e4m3 cache has scales, a 16-bit one has none";
  if (c.pages <= 0 || c.page_size <= 0 || c.heads <= 0 || c.dim <= 0) return "cache extents must be positive";
  if (c.pages * c.page_size > 0x7fffffffLL) return "more than 2^31 - 1 cache slots";
  if (c.dim % 8 || c.dim > 512) return "head dim must be a multiple of 8, at most 512";
  const int es = element_size(c.dtype), unit = es == 1 ? 8 : 16;
  if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) % 16 || c.page_stride * es % unit ||
      c.slot_stride * es % unit || c.head_stride * es % unit)
    return "cache rows must start on 16-byte (8-bit caches: 8-byte) boundaries";
  return nullptr;
}

// Two codes as two exact 16-bit floats.  i8: each in the low byte of a 16-bit half of `w`, the other byte is anything;
// e4m3: both in the low half of `w`, converted by the instruction for it, NaN among them.
template <class T, int CD> struct Codes;
// i8 -> bf16: 0x4300 | low 7 bits is 128 + them; less 128, or 256 where the sign bit is set
template <> struct Codes<__nv_bfloat16, TJ_I8> {
  static TJ_DEV uint32_t make(uint32_t w) {
    const uint32_t x = (w & 0x007f007fu) | 0x43004300u, y = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(reinterpret_cast<const __nv_bfloat162&>(x), reinterpret_cast<const __nv_bfloat162&>(y));
    return reinterpret_cast<const uint32_t&>(d);
  }
};
// i8 -> f16: 0x6400 | (code + 128) is 1024 + that
template <> struct Codes<__half, TJ_I8> {
  static TJ_DEV uint32_t less(uint32_t x) {
    const uint32_t y = 0x64806480u;
    const __half2 d = __hsub2(reinterpret_cast<const __half2&>(x), reinterpret_cast<const __half2&>(y));
    return reinterpret_cast<const uint32_t&>(d);
  }
  static TJ_DEV uint32_t make(uint32_t w) { return less((w & 0x00ff00ffu) ^ 0x64806480u); }
};
template <> struct Codes<__half, TJ_E4M3> {
  static TJ_DEV uint32_t make(uint32_t w) {
    const __half2_raw d = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w), __NV_E4M3);
    return reinterpret_cast<const uint32_t&>(d);
  }
};
template <> struct Codes<__nv_bfloat16, TJ_E4M3> {
  static TJ_DEV uint32_t make(uint32_t w) {
    const uint32_t h = Codes<__half, TJ_E4M3>::make(w);
    const float2 f = __half22float2(reinterpret_cast<const __half2&>(h));
    return tj_pack_bf16x2(f.x, f.y);
  }
};

// The four codes of a word, in order, as two words of 16-bit floats.
template <class T, int CD> TJ_DEV void codes4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CD == TJ_I8 && std::is_same<T, __half>::value) {
    w ^= 0x80808080u;
    lo = Codes<T, CD>::less(__byte_perm(w, 0x64646464u, 0x4140));
    hi = Codes<T, CD>::less(__byte_perm(w, 0x64646464u, 0x4342));
  } else {
    lo = Codes<T, CD>::make(CD == TJ_I8 ? __byte_perm(w, 0, 0x4140) : w);
    hi = Codes<T, CD>::make(CD == TJ_I8 ? __byte_perm(w, 0, 0x4342) : w >> 16);
  }
}

// n / d for 0 <= n < 2^31 by a multiplication and a shift (Granlund and Montgomery 1994, "Division by invariant
// integers using multiplication").
struct Div {
  uint32_t mul, shift, d;
  Div() = default;
  explicit Div(uint32_t by) : d(by) {
    shift = 0;
    while ((1ull << shift) < by) ++shift;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - by)) / by + 1);
  }
  TJ_DEV int operator()(int n) const { return static_cast<int>((__umulhi(mul, static_cast<uint32_t>(n)) + static_cast<uint32_t>(n)) >> shift); }
};

}  // namespace tjs
