// Products of microscaled rows with 4-bit weights (layout: mx_common.hpp) on v_mfma_scale_f32_16x16x128_f8f6f4:
//   C[M x N] = A[M x K] . B[N x K]^T (+ bias) (ReLU),  A in e4m3 or e2m1, B in e2m1, sums in float32.
//
// The instruction takes 16 rows of each operand and 128 of k, four blocks of 32, and a scale byte for each row and block: lane l brings
// row l % 16, and the scale of the block in place l / 16.  Of a 4-bit operand lane l's 16 bytes are that block too; of an 8-bit one its 32
// bytes are half (l / 16) % 2 of the blocks in places l / 32 (first 16 bytes) and 2 + l / 32 (second).  (Measured: sums of 4-bit products
// come out exact; 8-bit ones are added on a grid of about 2^-14 of the largest product of the 128.)  Which blocks of a row go to which
// place is free, as long as both operands and the scales agree: of 256 k, step s of two puts block 2 p + s in place p, so that a lane's
// 4-bit codes of both steps are 32 bytes in a row and its scales two.
// The weights are the first operand, so a lane's four results are four columns of one row of C.
#include "mx_common.hpp"

namespace sarek_hip {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

enum { kFormatE4M3 = 0, kFormatE2M1 = 4 };   // the instruction's own numbers

template <bool Fp8, int Step> __device__ __forceinline__ f32x4_t mfma_mx(u32x4_t b, i32x8 a, f32x4_t c, int b_scales, int a_scales) {
  const i32x8 wide = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide, a, c, kFormatE2M1, Fp8 ? kFormatE4M3 : kFormatE2M1, Step, b_scales,
                                                          Step, a_scales);
}

// One wave to a 16 x 16 tile of C, operands straight from memory.
template <bool Fp8, class T>
__global__ __launch_bounds__(64) void gemm_mx_kernel(const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales,
                                                     const uint8_t *__restrict__ b, const uint8_t *__restrict__ b_scales,
                                                     const float *__restrict__ bias, int relu, T *__restrict__ c, int64_t c_stride,
                                                     int64_t m, int64_t n, int64_t kp) {
  const int lane = threadIdx.x, r = lane & 15, place = lane >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 16, n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t arow = min(m0 + r, m - 1), brow = min(n0 + r, n - 1);   // rows past the end are the last one again: not stored
  const uint8_t *const ap = a + arow * (Fp8 ? kp : kp / 2), *const bp = b + brow * (kp / 2);
  const uint8_t *const as = a_scales + arow * (kp / kMxBlock), *const bs = b_scales + brow * (kp / kMxBlock);
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int64_t u = 0; u < kp / kMxRow; ++u) {
    const int sa = *reinterpret_cast<const uint16_t *>(as + u * 8 + 2 * place), sb = *reinterpret_cast<const uint16_t *>(bs + u * 8 + 2 * place);
    u32x4_t bf[2];
    i32x8 af[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf[s] = *reinterpret_cast<const u32x4_t *>(bp + u * 128 + place * 32 + s * 16);
      u32x4_t lo, hi = {0u, 0u, 0u, 0u};
      if constexpr (Fp8) {
        const uint8_t *const p = ap + u * 256 + (2 * (place >> 1) + s) * 32 + (place & 1) * 16;
        lo = *reinterpret_cast<const u32x4_t *>(p);
        hi = *reinterpret_cast<const u32x4_t *>(p + 128);
      } else {
        lo = *reinterpret_cast<const u32x4_t *>(ap + u * 128 + place * 32 + s * 16);
      }
      af[s] = i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
                    static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
    }
    acc = mfma_mx<Fp8, 0>(bf[0], af[0], acc, sb, sa);
    acc = mfma_mx<Fp8, 1>(bf[1], af[1], acc, sb, sa);
  }
  if (m0 + r >= m) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t col = n0 + 4 * place + j;
    if (col >= n) continue;
    float v = acc[j] + (bias ? bias[col] : 0.f);
    if (relu) v = v < 0.f ? 0.f : v;
    store_one(c + (m0 + r) * c_stride + col, v);
  }
}

}  // namespace
}  // namespace sarek_hip

using namespace sarek_hip;

extern "C" int sarek_hip_gemm_mx(const unsigned char *a_codes, const unsigned char *a_scales, int a_format, const unsigned char *b_codes,
                                 const unsigned char *b_scales, const float *bias, int relu, void *c, int c_type, int64_t c_stride,
                                 int64_t m, int64_t n, int64_t k, sarek_hip_stream stream) {
  if (m < 0 || n <= 0 || k <= 0)
    return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: m must not be negative, n and k must be positive (%lld x %lld x %lld)",
                static_cast<long long>(m), static_cast<long long>(n), static_cast<long long>(k));
  if (!known_format(a_format) || !known_type(c_type)) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: unknown format %d or type %d", a_format, c_type);
  if (a_format == SAREK_HIP_MX_FP8 && c_type == SAREK_HIP_TYPE_F32)
    return fail(SAREK_HIP_E_UNSUPPORTED, "gemm_mx: products of 8-bit rows are not exact to float32's last bits: C is bf16 or fp16");
  if (c_stride < n) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: rows of C are %lld values apart, less than n = %lld", static_cast<long long>(c_stride), static_cast<long long>(n));
  if (m > (int64_t{1} << 20) - 1 || n > 0x7FFFFFFF || k > 0x7FFFFFFF - kMxRow)
    return fail(SAREK_HIP_E_UNSUPPORTED, "gemm_mx: m is below 2^20, n and k below 2^31");
  if (m == 0) return SAREK_HIP_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !c) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: NULL pointer");
  if (misaligned(a_codes, a_scales) || misaligned(b_codes, b_scales)) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: codes start at multiples of 16 bytes, scales of 8");
  const int64_t kp = mx_row_values(k);
  const dim3 grid(static_cast<unsigned>(ceil_div(n, 16)), static_cast<unsigned>(ceil_div(m, 16)));
  return by_type(c_type, [&]<class T>(T *) {
    if (a_format == SAREK_HIP_MX_FP8)
      hipLaunchKernelGGL((gemm_mx_kernel<true, T>), grid, dim3(64), 0, as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, relu, static_cast<T *>(c), c_stride, m, n, kp);
    else
      hipLaunchKernelGGL((gemm_mx_kernel<false, T>), grid, dim3(64), 0, as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, relu, static_cast<T *>(c), c_stride, m, n, kp);
    return check_launch("gemm_mx launch");
  });
}
