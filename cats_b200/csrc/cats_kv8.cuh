// Paged key/value cache in 8 bits: layout, formats and small helpers that its kernels share.
//
// Layout: codes [layers, pages, 2 (keys, values), kv_heads, page, head_dim] e4m3, so that the rows
// of one head of one page are one contiguous block (8 KB at 64 x 128: whole DRAM bursts) and a page
// of one layer is one contiguous block too (what a copy moves); scales [layers, pages, 2, kv_heads]
// fp32.  A value is code * scale.  Scales are powers of two, 2^-24 .. 2^60: multiplying by one is
// exact, so a page whose scale grows when a larger row arrives keeps its older rows bit for bit
// (but for codes that drop below e4m3's normal range), and e4m3 being a floating-point format, an
// arbitrary scale would not make the relative step any smaller.
#pragma once

#include "../../include/cats_b200.h"
#include "cats_common.cuh"

namespace cats {

constexpr int kKvExpMin = -24, kKvExpMax = 60;
constexpr int kKvMaxSeqs = 1024;      // sequences of one cache: one thread each in the planning CTAs
constexpr int kPlanThreads = 1024;

// bits of the cache's status word
enum { KV_POOL_EMPTY = 1, KV_BAD_PAGE = 2, KV_TOO_LONG = 4, KV_BAD_PARENT = 8, KV_BAD_SPAN = 16, KV_WAIT = 32, KV_REFUSED = 64 };

__device__ __forceinline__ void kv_flag(const cats_kv8& c, int bit) { atomicOr(c.status, bit); }

// The last words of the status array, a bit for every sequence: the last grow that had tokens for it did
// not lengthen it, so that its last positions are older tokens', which append must not take for the new.
constexpr int kKvRefusedAt = CATS_KV8_STATUS_INTS - kKvMaxSeqs / 32;
__device__ __forceinline__ bool kv_refused(const cats_kv8& c, int b) { return (c.status[kKvRefusedAt + (b >> 5)] >> (b & 31)) & 1; }
// Called by all lanes of a warp, lane = sequence: the bits of the sequences in `set` become `refused`.
__device__ __forceinline__ void kv_set_refused(const cats_kv8& c, int b, bool set, bool refused) {
  const unsigned which = __ballot_sync(0xffffffffu, set), bits = __ballot_sync(0xffffffffu, set && refused);
  if ((b & 31) == 0 && which) {
    int* w = c.status + kKvRefusedAt + (b >> 5);
    *w = (int)(((unsigned)*w & ~which) | bits);
  }
}

// bytes of one head's rows in a page / of a page in one layer
__device__ __forceinline__ size_t kv_block(const cats_kv8& c) { return (size_t)c.page * c.head_dim; }
__device__ __forceinline__ size_t kv_page_bytes(const cats_kv8& c) {
  return 2 * (size_t)c.n_kv_heads * kv_block(c);
}
// start of the rows of (layer, page, keys / values, head)
__device__ __forceinline__ uint8_t* kv_rows(const cats_kv8& c, int layer, int page, int kv, int head) {
  return static_cast<uint8_t*>(c.codes) + ((size_t)layer * c.n_pages + page) * kv_page_bytes(c) +
         ((size_t)kv * c.n_kv_heads + head) * kv_block(c);
}
__device__ __forceinline__ float* kv_scale(const cats_kv8& c, int layer, int page, int kv, int head) {
  return c.scales + (((size_t)layer * c.n_pages + page) * 2 + kv) * c.n_kv_heads + head;
}

// exponent of a power-of-two scale (mantissa bits, which a valid scale does not have, are ignored)
__device__ __forceinline__ int kv_exp_of(float scale) {
  return (int)((__float_as_uint(scale) >> 23) & 255u) - 127;
}
__device__ __forceinline__ float kv_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Least e with amax <= 448 * 2^e, clamped: 448 = 1.75 * 2^8, so with amax = m * 2^x, 1 <= m < 2, it
// is x - 8, and one more when m > 1.75.  Integer arithmetic on the bits, exact.
__device__ __forceinline__ int kv_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, kKvExpMin), kKvExpMax);
}

// two fp32 -> two e4m3 codes (round to nearest even, saturating at 448; NaN stays NaN)
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return e4m3x2(a, b) | (e4m3x2(c, d) << 16);
}
// two e4m3 codes (low 16 bits) -> f16x2, exact
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}

// four e4m3 codes -> two f16x2 (codes 0, 1 and 2, 3), exact
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}

// New tokens of sequence b: [first, first + count) of the packed tokens.  cu == nullptr: every
// sequence has `uniform` of them.
struct KvSpan {
  int first, count;
};
__device__ __forceinline__ KvSpan kv_span(const int* cu, int uniform, int b) {
  if (!cu) return {b * uniform, uniform};
  const int a = __ldg(cu + b), z = __ldg(cu + b + 1);
  return {a, z > a ? (int)min((unsigned)z - (unsigned)a, 0x7fffffffu) : 0};
}
// cu goes down behind sequence b: the spans could overlap, and be more than the call's tokens together
__device__ __forceinline__ bool kv_descends(const int* cu, int b) { return __ldg(cu + b + 1) < __ldg(cu + b); }

// pages that `count` new tokens can touch
__host__ __device__ inline int kv_units(int count, int page) {
  return count < 1 ? 0 : (int)(((unsigned)count + page - 2u) / page) + 1;
}

// eight elements, 16-byte aligned
template <typename T>
__device__ __forceinline__ void load8_cached(const T* p, float* f) {
  const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
  VecT<T>::unpack(a, f);
  if (sizeof(T) == 4) {
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    VecT<T>::unpack(b, f + VecT<T>::N % 8);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  __align__(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = VecT<T>::from_f(f[i]);
  const uint4* s = reinterpret_cast<const uint4*>(v);
  uint4* d = reinterpret_cast<uint4*>(p);
  d[0] = s[0];
  if (sizeof(T) == 4) d[1] = s[1];
}

}  // namespace cats
