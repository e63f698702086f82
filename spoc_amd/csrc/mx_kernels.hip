// Rows in microscaled 8- and 4-bit floating point (layout: mx_common.hpp): bringing a matrix to them and back, the root-mean-square
// norm that writes 8-bit rows for the product behind it, and that norm's gradient.  All of them pass over memory once.
#include <algorithm>
#include <type_traits>

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

// One thread to eight values of the padded rows, four threads to a block.
template <class T, bool Fp8>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *__restrict__ x, int64_t stride, uint8_t *__restrict__ codes,
                                                          uint8_t *__restrict__ scales, int64_t rows, int64_t k, int64_t kp) {
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; at < rows * kp; at += static_cast<int64_t>(gridDim.x) * 2048) {
    const int64_t row = at / kp, c = at - row * kp;   // (the threads of a block of 32 stay together, kp being a multiple of 256)
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < k) widen8<T>(load8(x + row * stride + c, k - c), v);
    write_codes<Fp8>(v, codes + row * (Fp8 ? kp : kp / 2), scales + row * (kp / kMxBlock), c);
  }
}

template <class T, bool Fp8>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                            T *__restrict__ out, int64_t stride, int64_t rows, int64_t k, int64_t kp) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8; at < rows * kp; at += static_cast<int64_t>(gridDim.x) * 2048) {
    const int64_t row = at / kp, c = at - row * kp;
    if (c >= k) continue;
    const uint32_t byte = scales[row * (kp / kMxBlock) + c / kMxBlock];
    const float scale = byte == 255 ? __uint_as_float(0x7FC00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
    float v[8];
    auto put = [&](int j, f32x2 pair) { v[j] = pair.x * scale, v[j + 1] = pair.y * scale; };
    if constexpr (Fp8) {
      const u32x2_t q = *reinterpret_cast<const u32x2_t *>(codes + row * kp + c);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        put(4 * w, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[w], 1.f, false));
        put(4 * w + 2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(q[w], 1.f, true));
      }
    } else {
      const uint32_t q = *reinterpret_cast<const uint32_t *>(codes + row * (kp / 2) + c / 2);
      put(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 0));
      put(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 1));
      put(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 2));
      put(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.f, 3));
    }
    store8(out + row * stride + c, k - c, v);
  }
}

// ---- norm --------------------------------------------------------------------------------------------------------------------------

// The sum over the `Threads` threads of a row, in the same order on every run.  `shared`: Threads / 64 floats, not in use by the
// previous sum any more.
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

// h = x + residual rounded to T (h = x without one), r = (mean of h^2 + eps)^-1/2, and the 8-bit form of h r weight.  One workgroup to a
// row, which it goes over twice: what the second turn reads of h, the first one has read or written.
template <class T>
__global__ __launch_bounds__(256) void rms_norm_kernel(const T *x, int64_t x_stride, const T *residual, int64_t residual_stride,
                                                       const T *__restrict__ weight, float eps, T *h, int64_t h_stride,
                                                       uint8_t *__restrict__ codes, uint8_t *__restrict__ scales,
                                                       float *__restrict__ rstd, int64_t rows, int64_t k, int64_t kp) {
  __shared__ float shared[4];
  auto sums = [&](int64_t row, int64_t c, float (&v)[8]) {
    widen8<T>(load8(x + row * x_stride + c, k - c), v);
    if (residual) {
      float w[8];
      widen8<T>(load8(residual + row * residual_stride + c, k - c), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = round_to<T>(v[j] + w[j]);
    }
  };
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < k; c += 256 * 8) {
      float v[8];
      sums(row, c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j] * v[j];
    }
    __syncthreads();
    const float r = 1.f / sqrtf(row_sum<256>(sum, shared) / static_cast<float>(k) + eps);
    if (rstd && threadIdx.x == 0) rstd[row] = r;
    for (int64_t c = threadIdx.x * 8; c < kp; c += 256 * 8) {
      float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (c < k) {
        float w[8];
        sums(row, c, v);
        if (h) store8(h + row * h_stride + c, k - c, v);
        widen8<T>(load8(weight + c, k - c), w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * r * w[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < k ? v[j] : 0.f;   // (0 times an infinite or undefined 1 / rms is not 0)
      write_codes<true>(v, codes + row * kp, scales + row * (kp / kMxBlock), c);
    }
  }
}

// With n = h r and g = weight dy:  dx = r (g - n mean(n g)) + dh,  dweight = sum over the rows of dy n.  A workgroup takes every
// gridDim.x-th row and leaves its rows' share of dweight in a plane of its own; rms_norm_planes_kernel adds the planes up in order.
template <class T>
__global__ __launch_bounds__(256) void rms_norm_backward_kernel(const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ h,
                                                                int64_t h_stride, const T *__restrict__ weight,
                                                                const float *__restrict__ rstd, const T *dh, int64_t dh_stride, T *dx,
                                                                int64_t dx_stride, float *__restrict__ planes, int64_t rows, int64_t k) {
  __shared__ float shared[4];
  float *const plane = planes + blockIdx.x * k;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float r = rstd[row];
    float sum = 0.f;
    for (int64_t c = threadIdx.x * 8; c < k; c += 256 * 8) {
      float d[8], v[8], w[8];
      widen8<T>(load8(dy + row * dy_stride + c, k - c), d);
      widen8<T>(load8(h + row * h_stride + c, k - c), v);
      widen8<T>(load8(weight + c, k - c), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += v[j] * r * (w[j] * d[j]);
    }
    __syncthreads();
    const float mean = row_sum<256>(sum, shared) / static_cast<float>(k);
    for (int64_t c = threadIdx.x * 8; c < k; c += 256 * 8) {
      float d[8], v[8], w[8], e[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      widen8<T>(load8(dy + row * dy_stride + c, k - c), d);
      widen8<T>(load8(h + row * h_stride + c, k - c), v);
      widen8<T>(load8(weight + c, k - c), w);
      if (dh) widen8<T>(load8(dh + row * dh_stride + c, k - c), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float n = v[j] * r;
        if (c + j < k) plane[c + j] = (row == blockIdx.x ? 0.f : plane[c + j]) + d[j] * n;
        e[j] += r * (w[j] * d[j] - n * mean);
      }
      store8(dx + row * dx_stride + c, k - c, e);
    }
  }
}

__global__ __launch_bounds__(256) void rms_norm_planes_kernel(const float *__restrict__ planes, float *__restrict__ dweight, int count,
                                                              int64_t k) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= k) return;
  float sum = 0.f;
  for (int p = 0; p < count; ++p) sum += planes[p * k + c];
  dweight[c] = sum;
}

int backward_planes(int64_t rows) { return static_cast<int>(std::min<int64_t>(rows, 512)); }

int check_matrix(const char *what, int64_t rows, int64_t k) {
  if (rows < 0 || k <= 0) return fail(SAREK_HIP_E_INVALID_ARG, "%s: rows must not be negative and k must be positive (%lld x %lld)", what,
                                      static_cast<long long>(rows), static_cast<long long>(k));
  if (rows > 0x7FFFFFFF || k > 0x7FFFFFFF - kMxRow)
    return fail(SAREK_HIP_E_UNSUPPORTED, "%s: %lld x %lld: rows and k are below 2^31", what, static_cast<long long>(rows), static_cast<long long>(k));
  return SAREK_HIP_OK;
}
// Workgroups for `wanted`, at most 2^21: a launch has below 2^32 threads, the kernels go on from there in turns.
dim3 grid_of(int64_t wanted) { return dim3(static_cast<unsigned>(std::min<int64_t>(wanted, int64_t{1} << 21))); }
int check_stride(const char *what, const char *name, int64_t stride, int64_t k) {
  if (stride < k) return fail(SAREK_HIP_E_INVALID_ARG, "%s: rows of %s are %lld values apart, less than k = %lld", what, name,
                              static_cast<long long>(stride), static_cast<long long>(k));
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
  const dim3 grid = grid_of(ceil_div(rows * (kp / 8), 256));
  return by_type(type, [&]<class T>(T *) {
    if (format == SAREK_HIP_MX_FP8)
      hipLaunchKernelGGL((mx_quantize_kernel<T, true>), grid, dim3(256), 0, as_stream(stream), static_cast<const T *>(x), x_stride, codes, scales, rows, k, kp);
    else
      hipLaunchKernelGGL((mx_quantize_kernel<T, false>), grid, dim3(256), 0, as_stream(stream), static_cast<const T *>(x), x_stride, codes, scales, rows, k, kp);
    return check_launch("mx_quantize launch");
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
  const dim3 grid = grid_of(ceil_div(rows * (kp / 8), 256));
  return by_type(type, [&]<class T>(T *) {
    if (format == SAREK_HIP_MX_FP8)
      hipLaunchKernelGGL((mx_dequantize_kernel<T, true>), grid, dim3(256), 0, as_stream(stream), codes, scales, static_cast<T *>(out), out_stride, rows, k, kp);
    else
      hipLaunchKernelGGL((mx_dequantize_kernel<T, false>), grid, dim3(256), 0, as_stream(stream), codes, scales, static_cast<T *>(out), out_stride, rows, k, kp);
    return check_launch("mx_dequantize launch");
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
    hipLaunchKernelGGL(rms_norm_kernel<T>, grid_of(rows), dim3(256), 0, as_stream(stream), static_cast<const T *>(x),
                       x_stride, static_cast<const T *>(residual), residual_stride, static_cast<const T *>(weight), eps,
                       static_cast<T *>(h), h_stride, codes, scales, rstd, rows, k, kp);
    return check_launch("rms_norm_mx launch");
  });
}

int64_t sarek_hip_rms_norm_backward_workspace_floats(int64_t rows, int64_t k) {
  return rows <= 0 || k <= 0 ? 0 : backward_planes(rows) * k;
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
  const int planes = rows > 0 ? backward_planes(rows) : 0;
  return by_type(type, [&]<class T>(T *) {
    if (planes > 0) {
      hipLaunchKernelGGL(rms_norm_backward_kernel<T>, dim3(planes), dim3(256), 0, as_stream(stream), static_cast<const T *>(dy), dy_stride,
                         static_cast<const T *>(h), h_stride, static_cast<const T *>(weight), rstd, static_cast<const T *>(dh), dh_stride,
                         static_cast<T *>(dx), dx_stride, workspace, rows, k);
      SAREK_MX_TRY(check_launch("rms_norm_backward launch"));
    }
    hipLaunchKernelGGL(rms_norm_planes_kernel, dim3(static_cast<unsigned>(ceil_div(k, 256))), dim3(256), 0, as_stream(stream), workspace,
                       dweight, planes, k);
    return check_launch("rms_norm_backward planes launch");
  });
}

}  // extern "C"
