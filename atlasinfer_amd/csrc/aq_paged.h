// aq_paged.h -- what the kernels over a paged key/value cache share: the two
// 16-bit types, and where a packed batch's sequences, rows and pages are.
#pragma once

#include "aq_common.h"

namespace paged {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) short4v lds_s4;

// What differs between fp16 and bf16 data: conversions, products, and from
// where on the bits of a magnitude are those of an infinity or NaN.
struct Half {
  static constexpr uint16_t kInf = 0x7C00;
  static __device__ __forceinline__ float to_f32(uint16_t b) { return (float)bits_to_h(b); }
  // two numbers to nearest (one conversion)
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{a, b}, half2v));
  }
  // s + the sum of both
  static __device__ __forceinline__ float add2(uint32_t p, float s) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, p), half2v{(f16)1.0f, (f16)1.0f}, s, false);
  }
  static __device__ __forceinline__ float16v mfma32(u32x4 a, u32x4 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4v mfma16(u32x4 a, u32x4 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
  }
};

struct Bf16 {
  static constexpr uint16_t kInf = 0x7F80;
  static __device__ __forceinline__ float to_f32(uint16_t b) { return __builtin_bit_cast(float, (uint32_t)b << 16); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{a, b}, bf2v));
  }
  static __device__ __forceinline__ float add2(uint32_t p, float s) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf2v, p), bf2v{(__bf16)1.0f, (__bf16)1.0f}, s, false);
  }
  static __device__ __forceinline__ float16v mfma32(u32x4 a, u32x4 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float4v mfma16(u32x4 a, u32x4 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8v, a), __builtin_bit_cast(bf8v, b), c, 0, 0, 0);
  }
};

// The packed batch.  Device numbers are not trusted: rows are cut to 0 .. T, a
// sequence that contradicts the host's bounds is left out, a page outside the
// cache is neither read nor written.
typedef const __attribute__((address_space(4))) int const_int;

// p[i] for an i that all lanes of a wave share, by the scalar unit.
__device__ __forceinline__ int scalar_int(const int* p, int64_t i) {
  return ((const_int*)(uintptr_t)p)[i];
}

struct Batch {
  const int *starts, *lengths, *table;
  int T, S, W, pages, shift;  // rows, sequences, table entries a sequence, pages, log2(page size)
  int max_new, max_length;

  __device__ __forceinline__ int start(int s) const { return min(max(starts[s], 0), T); }
  __device__ __forceinline__ int scalar_start(int s) const { return min(max(scalar_int(starts, s), 0), T); }
};

// The last of 0 .. n - 1 with value(s) <= x, -1 if there is none, the values
// ascending: a wave looks at 64 of them at a time, one look up to 64 of them, two up to
// 4096, three up to 65535 (a look waits for memory).
template <class F>
__device__ __forceinline__ int last_at_most(int n, int x, F value) {
  const int ln = threadIdx.x & 63;
  int lo = 0;
  for (;;) {
    const int step = (n + 63) >> 6, s = ln * step;
    const uint64_t mask = __ballot(s < n && value(lo + min(s, n - 1)) <= x);
    if (!mask) return lo - 1;
    const int k = 63 - __builtin_clzll(mask);
    lo = __builtin_amdgcn_readfirstlane(lo + k * step);
    if (step == 1) return lo;
    n = min(step, n - k * step);
  }
}

// The sequence whose rows hold row t, -1 for none; the same for all lanes.
__device__ __forceinline__ int sequence_of(const Batch& b, int t) {
  const int s = last_at_most(b.S, t, [&](int i) { return b.start(i); });
  return s >= 0 && t < b.scalar_start(s + 1) ? s : -1;
}

}  // namespace paged
