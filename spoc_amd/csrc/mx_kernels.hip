// Rows in microscaled 8- and 4-bit floating point (layout: mx_common.hpp): bringing a matrix to them and back, the root-mean-square
// norm that writes 8-bit rows for the product behind it, and that norm's gradient.  All of them pass over memory once.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "mx_common.hpp"

namespace sarek_hip {
namespace {

// The scale byte of a block from the bits of its largest magnitude (of magnitudes, the bits are in the numbers' order; an infinity is
// the exponent 255 and a NaN is past it).  A largest magnitude below the normal numbers has the exponent 0 here: byte 0.
template <bool Fp8> __device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
  const int exponent = static_cast<int>(most >> 23);
  return exponent == 255 ? 255u : static_cast<uint32_t>(max(exponent - (Fp8 ? 8 : 2), 0));
}

// Eight values of a block whose scale byte is `byte`: 8 bytes of codes (e4m3) or 4 (e2m1).  The product with 2^-E is exact (below the
// normal numbers every code is 0), so the conversion makes the only rounding; it saturates for e2m1, for e4m3 the clamp does.
template <bool Fp8> __device__ __forceinline__ u32x2_t codes_of(const float (&v)[8], uint32_t byte) {
  if (byte == 255) return u32x2_t{0u, 0u};
  const float inverse = __uint_as_float((254u - byte) << 23);
  float q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = v[j] * inverse;
  u32x2_t out = {0u, 0u};
  if constexpr (Fp8) {
    typedef __attribute__((ext_vector_type(2))) short s16x2;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      s16x2 c = {0, 0};
      auto clamped = [&](int j) { return __builtin_amdgcn_fmed3f(q[4 * w + j], -448.f, 448.f); };
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, clamped(0), clamped(1), 1.f, false);
      c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, clamped(2), clamped(3), 1.f, true);
      out[w] = __builtin_bit_cast(uint32_t, c);
    }
  } else {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[0], q[1], 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[2], q[3], 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[4], q[5], 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[6], q[7], 1.f, 3);
    out[0] = c;
  }
  return out;
}

// The bits of the largest magnitude of a block, of which four neighbouring lanes hold eight values each.
__device__ __forceinline__ uint32_t block_most(const float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[j]) & 0x7FFFFFFFu);
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 1, 64)));
  most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 2, 64)));
  return most;
}

// Writes eight values from column c (a multiple of 8) of a row: their codes, and with the block's first eight its scale byte.
template <bool Fp8>
__device__ __forceinline__ void write_codes(const float (&v)[8], uint8_t *__restrict__ code_row, uint8_t *__restrict__ scale_row, int64_t c) {
  const uint32_t byte = scale_byte<Fp8>(block_most(v));
  const u32x2_t q = codes_of<Fp8>(v, byte);
  if constexpr (Fp8) *reinterpret_cast<u32x2_t *>(code_row + c) = q;
  else *reinterpret_cast<uint32_t *>(code_row + c / 2) = q[0];
  if ((c & (kMxBlock - 1)) == 0) scale_row[c / kMxBlock] = static_cast<uint8_t>(byte);
}

// ---- to 8 or 4 bits and back -------------------------------------------------------------------------------------------------------

// One thread to eight values of the padded rows, four threads to a block of 32, 32 to 256 values of one row.  Memory bounds both: 11008 x
// 4096 in bf16 to 8 bits 26.9 us, back 26.1, 5.1 and 5.2 TB/s (one piece to a thread, the row by a 64-bit division: 29.5 and 31.3).
struct Rows {
  uint32_t count, per_row, inverse;   // pieces of 256 values in all and of a row, and 2^32 over the latter, rounded down (2^32 - 1 for 1)
};
// The row and column of the eight values of piece u that are this thread's.
__device__ __forceinline__ void place_of(const Rows &p, uint32_t u, int64_t &row, int64_t &column) {
  uint32_t q = __umulhi(u, p.inverse), left = u - q * p.per_row;   // at most two short
  if (left >= p.per_row) ++q, left -= p.per_row;
  if (left >= p.per_row) ++q, left -= p.per_row;
  row = q;
  column = static_cast<int64_t>(left) * kMxRow + (threadIdx.x & 31) * 8;
}
template <class T, bool Fp8, int kAtOnce>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *__restrict__ x, int64_t stride, uint8_t *__restrict__ codes,
                                                          uint8_t *__restrict__ scales, Rows pieces, int64_t k, int64_t kp) {
  for (uint32_t u = blockIdx.x * (8 * kAtOnce) + threadIdx.x / 32; u < pieces.count; u += gridDim.x * (8 * kAtOnce)) {
    int64_t row[kAtOnce], c[kAtOnce];
    Raw8<T> raw[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u + 8 * i >= pieces.count) break;
      place_of(pieces, u + 8 * i, row[i], c[i]);
      raw[i] = load8(x + row[i] * stride + c[i], k - c[i]);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u + 8 * i >= pieces.count) break;
      float v[8];
      widen8<T>(raw[i], v);
      write_codes<Fp8>(v, codes + row[i] * (Fp8 ? kp : kp / 2), scales + row[i] * (kp / kMxBlock), c[i]);
    }
  }
}

template <class T, bool Fp8, int kAtOnce>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                            T *__restrict__ out, int64_t stride, Rows pieces, int64_t k, int64_t kp) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  for (uint32_t u = blockIdx.x * (8 * kAtOnce) + threadIdx.x / 32; u < pieces.count; u += gridDim.x * (8 * kAtOnce)) {
    int64_t row[kAtOnce], c[kAtOnce];
    u32x2_t q[kAtOnce];
    uint32_t byte[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u + 8 * i >= pieces.count) break;
      place_of(pieces, u + 8 * i, row[i], c[i]);
      byte[i] = scales[row[i] * (kp / kMxBlock) + c[i] / kMxBlock];
      if constexpr (Fp8) q[i] = *reinterpret_cast<const u32x2_t *>(codes + row[i] * kp + c[i]);
      else q[i][0] = *reinterpret_cast<const uint32_t *>(codes + row[i] * (kp / 2) + c[i] / 2);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (u + 8 * i >= pieces.count) break;
      const float scale = byte[i] == 255 ? __uint_as_float(0x7FC00000u) : byte[i] == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte[i] << 23);
      float v[8];
      auto put = [&](int j, f32x2 pair) { v[j] = pair.x * scale, v[j + 1] = pair.y * scale; };
      if constexpr (Fp8) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          put(4 * w, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i][w], 1.f, false));
          put(4 * w + 2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[i][w], 1.f, true));
        }
      } else {
        put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i][0], 1.f, 0));
        put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i][0], 1.f, 1));
        put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i][0], 1.f, 2));
        put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i][0], 1.f, 3));
      }
      store8(out + row[i] * stride + c[i], k - c[i], v);
    }
  }
}

// ---- norm --------------------------------------------------------------------------------------------------------------------------

// The sum over the Threads threads of a row, in the same order on every run.  shared: Threads / 64 floats that nobody reads any more.
template <int Threads> __device__ __forceinline__ float row_sum(float v, float *shared) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (Threads > 64) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < Threads / 64; ++w) v += shared[w];
  }
  return v;
}

// 1 / sqrt(v) and what it is short by: the next code is taken where an error of r's or of a product's last bit carries h r weight past the
// middle between two, so the norm is rounded once, not three times (of 444 million codes 221 then differ from those of 64 bits, for
// 273; one row of 4096 takes 3.2 us for 3.1, 4095 rows the same).  v = 0 or infinite: no remainder.
struct Root { float r, low; };
__device__ __forceinline__ Root inverse_root(float v) {
  const float r = 1.f / sqrtf(v), s = v * r;   // s: sqrt(v), which neither overflows nor loses bits where r r would
  const float left = fmaf(-s, r, 1.f) - fmaf(v, r, -s) * r;
  return {r, r > 0.f && r < __builtin_inff() ? 0.5f * r * left : 0.f};
}
__device__ __forceinline__ float norm_of(float h, Root root, float weight) {
  const float n = h * root.r, low = fmaf(h, root.low, fmaf(h, root.r, -n));
  return fmaf(n, weight, low * weight);
}

template <class T> struct NormArgs {
  const T *x, *residual, *weight;
  T *h;
  uint8_t *codes, *scales;
  float *rstd;
  int64_t x_stride, residual_stride, h_stride, rows, k, kp;
  float eps;
};

// h = x + residual rounded to T (h = x without one), r = (mean of h^2 + eps)^-1/2, and the 8-bit form of h r weight.  Threads of a
// workgroup to a row, Vectors times eight values each: the row stays in registers between its sum and its codes, so that memory is read
// once and written once, which is what bounds it (4095 x 4096 in bf16 with a residual 20.3 us, 5.8 TB/s, some of it out of the caches; 999 x 11007 in float32,
// four rows to a compute unit, 14.4, 3.8).
template <class T, int Threads, int Vectors>
__global__ __launch_bounds__(Threads < 256 ? 256 : Threads) void rms_norm_kernel(NormArgs<T> p) {
  constexpr int kRows = Threads < 256 ? 256 / Threads : 1;
  __shared__ float shared[Threads / 64];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / Threads;
  if (row >= p.rows) return;   // (a whole wave where there are several rows to a workgroup, and no barrier then)
  const int first = static_cast<int>(threadIdx.x % Threads) * 8, k = static_cast<int>(p.k), kp = static_cast<int>(p.kp);
  const T *const x = p.x + row * p.x_stride, *const residual = p.residual ? p.residual + row * p.residual_stride : nullptr;
  Raw8<T> raw[Vectors], more[Vectors], w[Vectors];
#pragma unroll
  for (int v = 0; v < Vectors; ++v) {
    const int c = first + v * Threads * 8;
    raw[v] = load8_of_row(x, c, k);
    if (residual) more[v] = load8_of_row(residual, c, k);
    w[v] = load8_of_row(p.weight, c, k);
  }
  float h[Vectors][8], sum = 0.f;
#pragma unroll
  for (int v = 0; v < Vectors; ++v) {
    widen8<T>(raw[v], h[v]);
    if (residual) {
      float m[8];
      widen8<T>(more[v], m);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[v][j] = round_to<T>(h[v][j] + m[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += h[v][j] * h[v][j];
  }
  const Root root = inverse_root(row_sum<Threads>(sum, shared) / static_cast<float>(k) + p.eps);
  if (p.rstd && first == 0) p.rstd[row] = root.r;
#pragma unroll
  for (int v = 0; v < Vectors; ++v) {
    const int c = first + v * Threads * 8;
    if (c >= kp) break;
    if (p.h && c < k) store8(p.h + row * p.h_stride + c, k - c, h[v]);
    float y[8];
    widen8<T>(w[v], y);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = c + j < k ? norm_of(h[v][j], root, y[j]) : 0.f;   // (0 times an infinite or undefined r is not 0)
    write_codes<true>(y, p.codes + row * kp, p.scales + row * (kp / kMxBlock), c);
  }
}

// The same for rows that registers do not hold: a workgroup goes over its row twice.
template <class T>
__global__ __launch_bounds__(1024) void rms_norm_long_kernel(NormArgs<T> p) {
  __shared__ float shared[16];
  const int64_t row = blockIdx.x;
  auto sums = [&](int64_t c, float (&v)[8]) {
    widen8<T>(load8(p.x + row * p.x_stride + c, p.k - c), v);
    if (p.residual) {
      float m[8];
      widen8<T>(load8(p.residual + row * p.residual_stride + c, p.k - c), m);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = round_to<T>(v[j] + m[j]);
    }
  };
  float sum = 0.f;
  for (int64_t c = threadIdx.x * 8; c < p.k; c += 1024 * 8) {
    float v[8];
    sums(c, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += v[j] * v[j];
  }
  const Root root = inverse_root(row_sum<1024>(sum, shared) / static_cast<float>(p.k) + p.eps);
  if (p.rstd && threadIdx.x == 0) p.rstd[row] = root.r;
  for (int64_t c = threadIdx.x * 8; c < p.kp; c += 1024 * 8) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < p.k) {
      float w[8];
      sums(c, v);
      if (p.h) store8(p.h + row * p.h_stride + c, p.k - c, v);
      widen8<T>(load8(p.weight + c, p.k - c), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = norm_of(v[j], root, w[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < p.k ? v[j] : 0.f;
    write_codes<true>(v, p.codes + row * p.kp, p.scales + row * (p.kp / kMxBlock), c);
  }
}

// Calls f with (threads to a row, times eight values) for rows of k values of type T; `longer` for those that registers are not made
// for, and for less than one load.  A wave to a row up to 1024 values (no barrier), then 256 threads, then 512, and 1024 for float32, whose 32
// values of a thread the gradient's registers would not hold (gradient of 3000 x 8190 in fp16, us: 256 threads 62.9, 512 46.5; 2000 x 16384
// in bf16: 512 threads 54, 1024 60).  Three loads to a thread
// where two of twice the threads would leave a quarter of them and more without values: past 8192 values always (3000 x 12000 in float32,
// gradient 136 us, so 93; 4095 x 11008 in bf16, norm 73 us, so 62; 16 rows the same), below where the caller's many rows make up for
// what a row alone takes longer (`many`): for a caller with Wave3 a wave up to 1536 values, with Block3 256 threads up to 6144.
template <class T, bool Wave3, bool Block3, class F, class Long> int by_length(int64_t k, bool many, F &&f, Long &&longer) {
  if (k < 8) return longer();   // (load8_of_row)
  if (k <= 512) return f(std::integer_sequence<int, 64, 1>{});
  if (k <= 1024) return f(std::integer_sequence<int, 64, 2>{});
  if constexpr (Wave3)
    if (k <= 1536 && many) return f(std::integer_sequence<int, 64, 3>{});
  if (k <= 2048) return f(std::integer_sequence<int, 256, 1>{});
  if (k <= 4096) return f(std::integer_sequence<int, 256, 2>{});
  if constexpr (Block3)
    if (k <= 6144 && many) return f(std::integer_sequence<int, 256, 3>{});
  if (k <= 8192) return f(std::integer_sequence<int, 512, 2>{});
  if (k <= 12288) return f(std::integer_sequence<int, 512, 3>{});
  if (k <= 16384) return f(std::conditional_t<sizeof(T) == 4, std::integer_sequence<int, 1024, 2>, std::integer_sequence<int, 512, 4>>{});
  return longer();
}
// The norm's, of 16-bit rows: from 2048 rows on (16000 x 1200 with a residual 38 us, so 28; 4000 x 5500 35.5, so 31.1); of fewer some gain and
// some lose (2000 x 1536 7.8, so 7.1; 1000 x 1536 4.4, so 4.7; 500 x 5500 7.2, so 7.3).  Float32 rows, with twice the bytes under way, gain
// nothing (4000 x 5500 55.6, 54.9).
template <class T> constexpr bool kNormByThree = sizeof(T) == 2;
bool many_for_norm(int64_t rows) { return rows >= 2048; }
// The gradient's, of a wave only: from 1024 rows on (16000 x 1200 in bf16 57 us, so 30, 1000 x 1536 8.6, so 8.2, 500 x 1536 12.0, so 12.3;
// float32 76 us, so 46); 256 threads lose (4000 x 5500 in bf16 47 us, 55).
bool many_for_gradient(int64_t rows) { return rows >= 1024; }

template <class T> struct BackwardArgs {
  const T *dy, *h, *weight, *dh;
  const float *rstd;
  T *dx;
  float *planes;
  int64_t dy_stride, h_stride, dh_stride, dx_stride, rows, k;
};

// With n = h r and g = weight dy:  dx = r (g - n mean(n g)) + dh,  dweight = sum over the rows of dy n.  A workgroup takes every
// gridDim.x-th row (or group of rows, a wave to a row) and keeps their share of dweight in registers; it goes into a plane of its own, and
// rms_norm_planes_kernel adds the planes up in order.  The next row is asked for before this one's sum is waited for: memory bounds
// it (8192 x 4096 in bf16 with dh 48.9 us and 4.7 for the planes, 5.0 TB/s).
template <class T, int Threads, int Vectors>
__global__ __launch_bounds__(Threads < 256 ? 256 : Threads) void rms_norm_backward_kernel(BackwardArgs<T> p) {
  constexpr int kRows = Threads < 256 ? 256 / Threads : 1;
  __shared__ float shared[2][Threads / 64];
  __shared__ float parts[kRows > 1 ? kRows : 1][kRows > 1 ? Threads * Vectors * 8 : 1];
  const int first = static_cast<int>(threadIdx.x % Threads) * 8, k = static_cast<int>(p.k), sub = threadIdx.x / Threads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  float w[Vectors][8], dw[Vectors][8];
#pragma unroll
  for (int v = 0; v < Vectors; ++v) {
    const int c = first + v * Threads * 8;
    widen8<T>(load8_of_row(p.weight, c, k), w[v]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[v][j] = 0.f;
  }
  Raw8<T> dy[Vectors], h[Vectors];
  float r = 0.f;
  auto load = [&](int64_t row) {
#pragma unroll
    for (int v = 0; v < Vectors; ++v) {
      const int c = first + v * Threads * 8;
      dy[v] = load8_of_row(p.dy + row * p.dy_stride, c, k);
      h[v] = load8_of_row(p.h + row * p.h_stride, c, k);
    }
    r = p.rstd[row];
  };
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + sub;
  if (row < p.rows) load(row);
  for (int turn = 0; row < p.rows; row += step, turn ^= 1) {
    float n[Vectors][8], g[Vectors][8], sum = 0.f;
    Raw8<T> add[Vectors];
    const float now = r;
    if (p.dh)
#pragma unroll
      for (int v = 0; v < Vectors; ++v) add[v] = load8_of_row(p.dh + row * p.dh_stride, first + v * Threads * 8, k);
#pragma unroll
    for (int v = 0; v < Vectors; ++v) {
      widen8<T>(dy[v], g[v]);
      widen8<T>(h[v], n[v]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[v][j] *= now;
        dw[v][j] += g[v][j] * n[v][j];
        g[v][j] *= w[v][j];
        sum += n[v][j] * g[v][j];
      }
    }
    if (row + step < p.rows) load(row + step);
    const float mean = row_sum<Threads>(sum, shared[turn]) / static_cast<float>(k);
#pragma unroll
    for (int v = 0; v < Vectors; ++v) {
      const int c = first + v * Threads * 8;
      if (c >= k) break;
      float out[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p.dh) widen8<T>(add[v], out);
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] += now * (g[v][j] - n[v][j] * mean);
      store8(p.dx + row * p.dx_stride + c, k - c, out);
    }
  }
  float *const plane = p.planes + blockIdx.x * p.k;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int v = 0; v < Vectors; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) parts[sub][first + v * Threads * 8 + j] = dw[v][j];
    __syncthreads();
    for (int c = threadIdx.x; c < k; c += 256) {
      float sum = 0.f;
#pragma unroll
      for (int q = 0; q < kRows; ++q) sum += parts[q][c];
      plane[c] = sum;
    }
  } else {
#pragma unroll
    for (int v = 0; v < Vectors; ++v) {
      const int c = first + v * Threads * 8;
      if (c < k) store8(plane + c, k - c, dw[v]);
    }
  }
}

// The same for longer rows, which a workgroup goes over twice; its plane of dweight is in memory all along.
template <class T>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_kernel(BackwardArgs<T> p) {
  __shared__ float shared[2][16];
  float *const plane = p.planes + blockIdx.x * p.k;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float r = p.rstd[row];
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < p.k; c += 1024 * 8) {
      float d[8], v[8], w[8];
      widen8<T>(load8(p.dy + row * p.dy_stride + c, p.k - c), d);
      widen8<T>(load8(p.h + row * p.h_stride + c, p.k - c), v);
      widen8<T>(load8(p.weight + c, p.k - c), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j] * r * (w[j] * d[j]);
    }
    const float mean = row_sum<1024>(sum, shared[turn]) / static_cast<float>(p.k);
    for (int64_t c = threadIdx.x * 8; c < p.k; c += 1024 * 8) {
      float d[8], v[8], w[8], e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      widen8<T>(load8(p.dy + row * p.dy_stride + c, p.k - c), d);
      widen8<T>(load8(p.h + row * p.h_stride + c, p.k - c), v);
      widen8<T>(load8(p.weight + c, p.k - c), w);
      if (p.dh) widen8<T>(load8(p.dh + row * p.dh_stride + c, p.k - c), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = v[j] * r;
        if (c + j < p.k) plane[c + j] = (row == blockIdx.x ? 0.f : plane[c + j]) + d[j] * n;
        e[j] += r * (w[j] * d[j] - n * mean);
      }
      store8(p.dx + row * p.dx_stride + c, p.k - c, e);
    }
  }
}

// dweight[c] = the planes' values of column c, added in an order that their number fixes: 32 threads to 4 columns, each a share of the
// planes, 32 columns (a line of every plane) to a workgroup.
__global__ __launch_bounds__(256) void rms_norm_planes_kernel(const float *__restrict__ planes, float *__restrict__ dweight, int count,
                                                              int64_t k) {
  __shared__ float sums[32][33];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * 32;
  const int quad = threadIdx.x & 7, share = threadIdx.x >> 3;
  const int64_t c = first + quad * 4;
  f32x4v sum = {0.f, 0.f, 0.f, 0.f};
  if (c + 4 <= k) {
#pragma unroll 16
    for (int q = share; q < count; q += 32) sum += *reinterpret_cast<const f32x4_any *>(planes + q * k + c);
  } else if (c < k) {
    for (int q = share; q < count; q += 32)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < k) sum[j] += planes[q * k + c + j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) sums[share][quad * 4 + j] = sum[j];
  __syncthreads();
  if (threadIdx.x < 32 && first + threadIdx.x < k) {
    float total = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) total += sums[q][threadIdx.x];
    dweight[first + threadIdx.x] = total;
  }
}

// Workgroups of the gradient, each with a plane of k floats: two to a compute unit, one where the planes would take over 8 MiB (they are
// written and read again), at most as many as there are (groups of) rows.  Never more for fewer rows: a workspace serves those, too (so
// not by the groups of rows where only many rows go by groups).
int backward_planes(int64_t rows, int64_t k) { return static_cast<int>(std::min<int64_t>(k <= 1024 ? ceil_div(rows, 4) : rows, k <= 4096 ? 512 : 256)); }

int check_matrix(const char *what, int64_t rows, int64_t k) {
  if (rows < 0 || k <= 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: rows must not be negative and k must be positive (%lld x %lld)", what,
                                      static_cast<long long>(rows), static_cast<long long>(k));
  if (rows >= int64_t{1} << 22 || k > int64_t{1} << 28)   // (a workgroup of 1024 to a row: below 2^32 threads)
    return fail(SAREK_HIP_E_UNSUPPORTED, "%s: %lld x %lld: rows are below 2^22, k at most 2^28", what, static_cast<long long>(rows), static_cast<long long>(k));
  return SAREK_HIP_OK;
}
// Workgroups for `wanted`, at most 2^21: a launch has below 2^32 threads, the kernels go on from there in turns.
dim3 grid_of(int64_t wanted) { return dim3(static_cast<unsigned>(std::min<int64_t>(wanted, int64_t{1} << 21))); }
int check_stride(const char *what, const char *name, int64_t stride, int64_t k) {
  if (stride < k) return fail(SAREK_HIP_E_INVALID_ARG, "%s: rows of %s are %lld values apart, less than k = %lld", what, name,
                              static_cast<long long>(stride), static_cast<long long>(k));
  return SAREK_HIP_OK;
}
// From here on a thread of mx_quantize and mx_dequantize asks for several pieces at once: eight workgroups to a compute unit then still.
constexpr uint32_t kManyPieces = 1 << 16;
int pieces_of(const char *what, int64_t rows, int64_t kp, Rows *out) {
  const int64_t per_row = kp / kMxRow, count = rows * per_row;
  if (count > 0x7FFFFFFF) return fail(SAREK_HIP_E_UNSUPPORTED, "%s: 2^39 values or more", what);
  *out = {static_cast<uint32_t>(count), static_cast<uint32_t>(per_row), per_row == 1 ? 0xFFFFFFFFu : static_cast<uint32_t>((int64_t{1} << 32) / per_row)};
  return SAREK_HIP_OK;
}
#define SAREK_MX_TRY(expr)                       \
  do {                                           \
    const int st_ = (expr);                      \
    if (st_ != SAREK_HIP_OK) return st_;         \
  } while (0)

}  // namespace
}  // namespace sarek_hip

using namespace sarek_hip;

extern "C" {

int64_t sarek_hip_mx_row_values(int64_t k) { return k <= 0 ? 0 : mx_row_values(k); }

int sarek_hip_mx_quantize(const void *x, int type, int64_t x_stride, unsigned char *codes, unsigned char *scales, int format,
                          int64_t rows, int64_t k, sarek_hip_stream stream) {
  SAREK_MX_TRY(check_matrix("mx_quantize", rows, k));
  if (!known_type(type) || !known_format(format)) return fail(SAREK_HIP_E_INVALID_ARG, "mx_quantize: unknown type %d or format %d", type, format);
  SAREK_MX_TRY(check_stride("mx_quantize", "x", x_stride, k));
  if (rows == 0) return SAREK_HIP_OK;
  if (!x || !codes || !scales) return fail(SAREK_HIP_E_INVALID_ARG, "mx_quantize: NULL pointer");
  if (misaligned(codes, scales)) return fail(SAREK_HIP_E_INVALID_ARG, "mx_quantize: codes start at multiples of 16 bytes, scales of 8");
  const int64_t kp = mx_row_values(k);
  Rows pieces;
  SAREK_MX_TRY(pieces_of("mx_quantize", rows, kp, &pieces));
  return by_type(type, [&]<class T>(T *) {
    const auto run = [&](auto kernel, int at_once) {
      hipLaunchKernelGGL(kernel, grid_of(ceil_div(pieces.count, 8 * at_once)), dim3(256), 0, as_stream(stream), static_cast<const T *>(x), x_stride, codes,
                         scales, pieces, k, kp);
      return check_launch("mx_quantize launch");
    };
    constexpr int kMany = sizeof(T) == 4 ? 2 : 4;
    if (pieces.count < kManyPieces) return format == SAREK_HIP_MX_FP8 ? run(mx_quantize_kernel<T, true, 1>, 1) : run(mx_quantize_kernel<T, false, 1>, 1);
    return format == SAREK_HIP_MX_FP8 ? run(mx_quantize_kernel<T, true, kMany>, kMany) : run(mx_quantize_kernel<T, false, kMany>, kMany);
  });
}

int sarek_hip_mx_dequantize(const unsigned char *codes, const unsigned char *scales, int format, void *out, int type, int64_t out_stride,
                            int64_t rows, int64_t k, sarek_hip_stream stream) {
  SAREK_MX_TRY(check_matrix("mx_dequantize", rows, k));
  if (!known_type(type) || !known_format(format)) return fail(SAREK_HIP_E_INVALID_ARG, "mx_dequantize: unknown type %d or format %d", type, format);
  SAREK_MX_TRY(check_stride("mx_dequantize", "out", out_stride, k));
  if (rows == 0) return SAREK_HIP_OK;
  if (!codes || !scales || !out) return fail(SAREK_HIP_E_INVALID_ARG, "mx_dequantize: NULL pointer");
  if (misaligned(codes, scales)) return fail(SAREK_HIP_E_INVALID_ARG, "mx_dequantize: codes start at multiples of 16 bytes, scales of 8");
  const int64_t kp = mx_row_values(k);
  Rows pieces;
  SAREK_MX_TRY(pieces_of("mx_dequantize", rows, kp, &pieces));
  return by_type(type, [&]<class T>(T *) {
    const auto run = [&](auto kernel, int at_once) {
      hipLaunchKernelGGL(kernel, grid_of(ceil_div(pieces.count, 8 * at_once)), dim3(256), 0, as_stream(stream), codes, scales, static_cast<T *>(out), out_stride,
                         pieces, k, kp);
      return check_launch("mx_dequantize launch");
    };
    if (pieces.count < kManyPieces) return format == SAREK_HIP_MX_FP8 ? run(mx_dequantize_kernel<T, true, 1>, 1) : run(mx_dequantize_kernel<T, false, 1>, 1);
    return format == SAREK_HIP_MX_FP8 ? run(mx_dequantize_kernel<T, true, 4>, 4) : run(mx_dequantize_kernel<T, false, 4>, 4);
  });
}

int sarek_hip_rms_norm_mx(const void *x, int64_t x_stride, const void *residual, int64_t residual_stride, const void *weight, int type,
                          float eps, void *h, int64_t h_stride, unsigned char *codes, unsigned char *scales, float *rstd, int64_t rows,
                          int64_t k, sarek_hip_stream stream) {
  SAREK_MX_TRY(check_matrix("rms_norm_mx", rows, k));
  if (!known_type(type)) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_mx: unknown type %d", type);
  if (!(eps >= 0.f)) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_mx: eps must not be negative");
  SAREK_MX_TRY(check_stride("rms_norm_mx", "x", x_stride, k));
  if (residual) SAREK_MX_TRY(check_stride("rms_norm_mx", "residual", residual_stride, k));
  if (h) SAREK_MX_TRY(check_stride("rms_norm_mx", "h", h_stride, k));
  if (rows == 0) return SAREK_HIP_OK;
  if (!x || !weight || !codes || !scales) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_mx: NULL pointer");
  if (misaligned(codes, scales)) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_mx: codes start at multiples of 16 bytes, scales of 8");
  if (residual && !h) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_mx: a residual is added, but there is no h for the sum");
  const int64_t kp = mx_row_values(k);
  return by_type(type, [&]<class T>(T *) {
    const NormArgs<T> args{static_cast<const T *>(x), static_cast<const T *>(residual), static_cast<const T *>(weight), static_cast<T *>(h),
                           codes, scales, rstd, x_stride, residual_stride, h_stride, rows, k, kp, eps};
    return by_length<T, kNormByThree<T>, kNormByThree<T>>(
        k, many_for_norm(rows),
        [&]<int Threads, int Vectors>(std::integer_sequence<int, Threads, Vectors>) {
          const dim3 grid(static_cast<unsigned>(ceil_div(rows, Threads < 256 ? 256 / Threads : 1)));
          hipLaunchKernelGGL((rms_norm_kernel<T, Threads, Vectors>), grid, dim3(std::max(Threads, 256)), 0, as_stream(stream), args);
          return check_launch("rms_norm_mx launch");
        },
        [&] {
          hipLaunchKernelGGL(rms_norm_long_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(1024), 0, as_stream(stream), args);
          return check_launch("rms_norm_mx launch");
        });
  });
}

int64_t sarek_hip_rms_norm_backward_workspace_floats(int64_t rows, int64_t k) {
  return rows <= 0 || k <= 0 ? 0 : backward_planes(rows, k) * k;
}

int sarek_hip_rms_norm_backward(const void *dy, int64_t dy_stride, const void *h, int64_t h_stride, const void *weight, const float *rstd,
                                const void *dh, int64_t dh_stride, int type, void *dx, int64_t dx_stride, float *dweight, int64_t rows,
                                int64_t k, float *workspace, int64_t workspace_floats, sarek_hip_stream stream) {
  SAREK_MX_TRY(check_matrix("rms_norm_backward", rows, k));
  if (!known_type(type)) return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_backward: unknown type %d", type);
  SAREK_MX_TRY(check_stride("rms_norm_backward", "dy", dy_stride, k));
  SAREK_MX_TRY(check_stride("rms_norm_backward", "h", h_stride, k));
  SAREK_MX_TRY(check_stride("rms_norm_backward", "dx", dx_stride, k));
  if (dh) SAREK_MX_TRY(check_stride("rms_norm_backward", "dh", dh_stride, k));
  if (!dweight || (rows > 0 && (!dy || !h || !weight || !rstd || !dx || !workspace)))
    return fail(SAREK_HIP_E_INVALID_ARG, "rms_norm_backward: NULL pointer");
  if (workspace_floats < sarek_hip_rms_norm_backward_workspace_floats(rows, k))
    return fail(SAREK_HIP_E_WORKSPACE, "rms_norm_backward: a workspace of %lld floats, %lld are needed", static_cast<long long>(workspace_floats),
                static_cast<long long>(sarek_hip_rms_norm_backward_workspace_floats(rows, k)));
  const int planes = rows > 0 ? backward_planes(rows, k) : 0;
  return by_type(type, [&]<class T>(T *) {
    if (planes > 0) {
      const BackwardArgs<T> args{static_cast<const T *>(dy), static_cast<const T *>(h), static_cast<const T *>(weight), static_cast<const T *>(dh),
                                 rstd, static_cast<T *>(dx), workspace, dy_stride, h_stride, dh_stride, dx_stride, rows, k};
      by_length<T, true, false>(
          k, many_for_gradient(rows),
          [&]<int Threads, int Vectors>(std::integer_sequence<int, Threads, Vectors>) {
            hipLaunchKernelGGL((rms_norm_backward_kernel<T, Threads, Vectors>), dim3(planes), dim3(std::max(Threads, 256)), 0, as_stream(stream), args);
            return SAREK_HIP_OK;
          },
          [&] {
            hipLaunchKernelGGL(rms_norm_backward_long_kernel<T>, dim3(planes), dim3(1024), 0, as_stream(stream), args);
            return SAREK_HIP_OK;
          });
      SAREK_MX_TRY(check_launch("rms_norm_backward launch"));
    }
    hipLaunchKernelGGL(rms_norm_planes_kernel, dim3(static_cast<unsigned>(ceil_div(k, 32))), dim3(256), 0, as_stream(stream), workspace,
                       dweight, planes, k);
    return check_launch("rms_norm_backward planes launch");
  });
}

}  // extern "C"
