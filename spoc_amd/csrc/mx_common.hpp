// Microscaled matrices: what the kernels that write them (mx_kernels.hip) and the products that read them (gemm_mx.hip) share.
//
// A row of k values is held in blocks of 32 along the row.  A block's scale is 2^E, E = floor(log2 of its largest magnitude) less the
// exponent of the format's largest value (448 = 1.75 2^8 in e4m3, 6 = 1.5 2^2 in e2m1), held as the byte E + 127, at least 0; a value
// v is held as the code nearest to v / 2^E, ties to the even code, past the largest value as the largest.  A block with a NaN or an
// infinity in it has the byte 255 and stands for 32 NaNs.
// Layout: rows of kp = k rounded up to 256 codes, one byte each (e4m3) or two to a byte (e2m1, the first in the low half), so that a row
// of 4-bit codes is whole 128-byte lines; kp / 32 scale bytes to a row.  What is behind k is zeros.
#pragma once
#include <hip/hip_runtime.h>

#include "common.hpp"

namespace sarek_hip {

constexpr int kMxBlock = 32, kMxRow = 256;
inline int64_t mx_row_values(int64_t k) { return (k + kMxRow - 1) / kMxRow * kMxRow; }

namespace {

// bf16 as it lies in memory: the kernels work on float32 and only load and store it.
struct Bf16 { uint16_t bits; };

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;
typedef __attribute__((ext_vector_type(4))) float f32x4v;
typedef u32x4_t u32x4_any __attribute__((aligned(2)));   // at any 16-bit element's address
typedef f32x4v f32x4_any __attribute__((aligned(4)));

__device__ __forceinline__ float bf16_to_f32(uint32_t bits) { return __uint_as_float(bits << 16); }
// Round to nearest even, by the conversion instruction (a NaN stays one).
__device__ __forceinline__ uint32_t f32_pair_to_bf16(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
  const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint32_t f32_pair_to_f16(float lo, float hi) {
  typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
  const f16x2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
  return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const _Float16 *p) { return static_cast<float>(*p); }
__device__ __forceinline__ float load_one(const Bf16 *p) { return bf16_to_f32(p->bits); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(_Float16 *p, float v) { *p = static_cast<_Float16>(v); }
__device__ __forceinline__ void store_one(Bf16 *p, float v) { p->bits = static_cast<uint16_t>(f32_pair_to_bf16(v, 0.f)); }

template <class T> __device__ __forceinline__ float round_to(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (__is_same(T, Bf16)) return bf16_to_f32(f32_pair_to_bf16(v, 0.f) & 0xFFFFu);
  else return static_cast<float>(static_cast<_Float16>(v));
}

// Eight values as they lie in memory, `count` of them (1 to 8, past the end: zeros) from p on, at any element's address.
template <class T> struct Raw8;
template <> struct Raw8<float> { f32x4v lo, hi; };
template <> struct Raw8<Bf16> { u32x4_t w; };
template <> struct Raw8<_Float16> { u32x4_t w; };

template <class T> __device__ __forceinline__ Raw8<T> load8(const T *p, int64_t count) {
  Raw8<T> r;
  if (count >= 8) {
    if constexpr (sizeof(T) == 4) {
      r.lo = *reinterpret_cast<const f32x4_any *>(p);
      r.hi = *reinterpret_cast<const f32x4_any *>(p + 4);
    } else {
      r.w = *reinterpret_cast<const u32x4_any *>(p);
    }
    return r;
  }
  // Past the end the last value is loaded again and dropped: eight loads on their way at once, where conditional ones wait for each other.
  const int last = static_cast<int>(count) - 1;
  if constexpr (sizeof(T) == 4) {
    r.lo = r.hi = f32x4v{0.f, 0.f, 0.f, 0.f};
    if (last < 0) return r;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[min(j, last)];
#pragma unroll
    for (int j = 0; j < 8; ++j) (j < 4 ? r.lo : r.hi)[j & 3] = j <= last ? v[j] : 0.f;
  } else {
    r.w = u32x4_t{0u, 0u, 0u, 0u};
    if (last < 0) return r;
    const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = q[min(j, last)];
#pragma unroll
    for (int j = 0; j < 8; ++j) r.w[j >> 1] |= j <= last ? v[j] << (16 * (j & 1)) : 0u;
  }
  return r;
}

// The same from column c of a row of k values, k at least 8: what begins past k - 8 is loaded from there and moved down, zeros behind it.
// (No branch but for the lanes at a row's end, and few registers: kernels that hold a row load it so.)
template <class T> __device__ __forceinline__ Raw8<T> load8_of_row(const T *row, int c, int k) {
  const int from = min(c, k - 8), over = c - from;
  Raw8<T> r = load8(row + from, 8);
  if (over == 0) return r;
  if constexpr (sizeof(T) == 4) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < 4 ? r.lo[j & 3] : r.hi[j & 3];
#pragma unroll
    for (int s = 1; s <= 4; s *= 2)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = over & s ? (j + s < 8 ? v[j + s] : 0.f) : v[j];
#pragma unroll
    for (int j = 0; j < 8; ++j) (j < 4 ? r.lo : r.hi)[j & 3] = over < 8 ? v[j] : 0.f;
  } else {
    typedef __attribute__((ext_vector_type(2))) unsigned long long u64x2_t;
    u64x2_t v = __builtin_bit_cast(u64x2_t, r.w);
    const int s = over * 16;
    v[0] = s < 64 ? v[0] >> s | v[1] << 1 << (63 - s) : s < 128 ? v[1] >> (s - 64) : 0;
    v[1] = s < 64 ? v[1] >> s : 0;
    r.w = __builtin_bit_cast(u32x4_t, v);
  }
  return r;
}

template <class T> __device__ __forceinline__ void widen8(const Raw8<T> &r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) {
      v[j] = j < 4 ? r.lo[j & 3] : r.hi[j & 3];
    } else if constexpr (__is_same(T, Bf16)) {
      v[j] = j & 1 ? __uint_as_float(r.w[j >> 1] & 0xFFFF0000u) : bf16_to_f32(r.w[j >> 1]);
    } else {
      v[j] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(r.w[j >> 1] >> (16 * (j & 1)))));
    }
  }
}

template <class T> __device__ __forceinline__ void store8(T *p, int64_t count, const float (&v)[8]) {
  if (count >= 8) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_any *>(p) = f32x4v{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4_any *>(p + 4) = f32x4v{v[4], v[5], v[6], v[7]};
    } else {
      u32x4_t w;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = __is_same(T, Bf16) ? f32_pair_to_bf16(v[2 * j], v[2 * j + 1]) : f32_pair_to_f16(v[2 * j], v[2 * j + 1]);
      *reinterpret_cast<u32x4_any *>(p) = w;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) store_one(p + j, v[j]);
}

// Calls f with the element type of a SAREK_HIP_TYPE_* value that has been checked.
template <class F> int by_type(int type, F &&f) {
  if (type == SAREK_HIP_TYPE_F32) return f(static_cast<float *>(nullptr));
  if (type == SAREK_HIP_TYPE_BF16) return f(static_cast<Bf16 *>(nullptr));
  return f(static_cast<_Float16 *>(nullptr));
}
inline bool known_type(int type) { return type == SAREK_HIP_TYPE_F32 || type == SAREK_HIP_TYPE_BF16 || type == SAREK_HIP_TYPE_F16; }
// (any row of a matrix that starts so does too)
inline bool misaligned(const void *codes, const void *scales) {
  return (reinterpret_cast<uintptr_t>(codes) & 15) != 0 || (reinterpret_cast<uintptr_t>(scales) & 7) != 0;
}
inline bool known_format(int format) { return format == SAREK_HIP_MX_FP8 || format == SAREK_HIP_MX_FP4; }

}  // namespace
}  // namespace sarek_hip
