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
#include <utility>

#include "gemm_common.hpp"
#include "mx_common.hpp"
#include "tunables.hpp"

namespace sarek_hip {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;

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

// ---- 256 x 256 tiles -----------------------------------------------------------------------------------------------------------------

template <class T> __device__ __forceinline__ void store_four(T *p, int64_t count, f32x4_t v) {
  if (count >= 4) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_any *>(p) = v;
    } else {
      typedef u32x2_t u32x2_any __attribute__((aligned(2)));
      *reinterpret_cast<u32x2_any *>(p) = __is_same(T, Bf16) ? u32x2_t{f32_pair_to_bf16(v[0], v[1]), f32_pair_to_bf16(v[2], v[3])}
                                                             : u32x2_t{f32_pair_to_f16(v[0], v[1]), f32_pair_to_f16(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < count) store_one(p + j, v[j]);
}

template <bool Fp8, class T>
__global__ __launch_bounds__(512) void gemm_mx_tile_kernel(const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales,
                                                           const uint8_t *__restrict__ b, const uint8_t *__restrict__ b_scales,
                                                           const float *__restrict__ bias, int relu, T *__restrict__ c, int64_t c_stride,
                                                           int m, int n, int kp, int tiles_m, int tiles_n) {
  constexpr int kStage = Fp8 ? 128 : 256;            // values of k in a stage: 128 bytes of a row of A
  constexpr int kRowB = Fp8 ? 64 : 128;              // bytes of a row of B in a stage
  constexpr int kPerSpan = 512 / kStage;             // stages that 16 scale bytes of a row last
  constexpr int kPeriod = 2 * kPerSpan;
  constexpr int kBytesA = 256 * 128, kBytesB = 256 * kRowB, kBytesS = 256 * 16;
  constexpr int kMovesA = kBytesA / 1024 / 8, kMovesB = kBytesB / 1024 / 8;   // transfers of a wave in a stage
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, place = lane >> 4;
  const int wm = wave >> 1, wn = wave & 1;           // 64 rows of C by 128 columns to a wave
  int tm, tn;
  tile_of_block(tiles_m, tiles_n, 1, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;
  const int pitch_a = Fp8 ? kp : kp / 2, pitch_b = kp / 2, pitch_s = kp / kMxBlock;
  const int rows_a = min(256, m - m0), rows_b = min(256, n - n0);
  // Rows past the end are out of the resources' range and read as zeros.
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(a + static_cast<int64_t>(m0) * pitch_a, static_cast<uint32_t>(rows_a) * pitch_a);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(b + static_cast<int64_t>(n0) * pitch_b, static_cast<uint32_t>(rows_b) * pitch_b);
  const bool of_a = wave < 4;
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(of_a ? a_scales + static_cast<int64_t>(m0) * pitch_s : b_scales + static_cast<int64_t>(n0) * pitch_s,
                                              static_cast<uint32_t>(of_a ? rows_a : rows_b) * pitch_s);
  uint32_t off_a[kMovesA], off_b[kMovesB];
#pragma unroll
  for (int i = 0; i < kMovesA; ++i) {
    const int row = (wave + 8 * i) * 8 + (lane >> 3);
    off_a[i] = static_cast<uint32_t>(row) * pitch_a + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < kMovesB; ++i) {
    constexpr int chunks = kRowB / 16;
    const int row = (wave + 8 * i) * (64 / chunks) + lane / chunks;
    off_b[i] = static_cast<uint32_t>(row) * pitch_b + (((lane % chunks) ^ (Fp8 ? (row >> 2) & 3 : (row >> 1) & 7)) << 4);
  }
  const uint32_t off_s = static_cast<uint32_t>((wave & 3) * 64 + lane) * pitch_s;
  const int stages = kp / kStage, last_span = (stages - 1) / kPerSpan;

  auto issue_codes = [&](char *la, char *lb, int s) {
    const int at = min(s, stages - 1);
#pragma unroll
    for (int i = 0; i < kMovesA; ++i) dma16(ra, off_a[i], at * 128, la + (wave + 8 * i) * 1024);
#pragma unroll
    for (int i = 0; i < kMovesB; ++i) dma16(rb, off_b[i], at * kRowB, lb + (wave + 8 * i) * 1024);
  };
  // A row's last span may be 8 bytes: then the 16 that end with the row are taken.
  auto issue_scales = [&](char *ls, int span) { dma16(rs, off_s, min(min(span, last_span) * 16, pitch_s - 16), ls + wave * 1024); };

  f32x4_t acc[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  int sa[4], sb[8];
  const uint32_t pick = (Fp8 ? static_cast<uint32_t>(place | (4 + place) << 8) : static_cast<uint32_t>(2 * place | (2 * place + 1) << 8)) | 0x0C0C0000u;
  auto scales_of = [&](const char *at, bool short_span) {
    u32x4 d = *reinterpret_cast<const u32x4 *>(at);
    d[0] = short_span ? d[2] : d[0];
    d[1] = short_span ? d[3] : d[1];
    return static_cast<int>(__builtin_amdgcn_perm(d[1], d[0], pick) | __builtin_amdgcn_perm(d[3], d[2], pick) << 16);
  };
  const int a_at = (wm * 64 + r) * 128, b_at = (wn * 128 + r) * kRowB;

  auto stage = [&](auto ic, int s) {
    constexpr int I = decltype(ic)::value, ring = I & 1, span = (I / kPerSpan) & 1, in_span = I % kPerSpan;
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));
    barrier_no_fence();
    if constexpr (in_span == 0) issue_scales(lds_ring<64 + (span ^ 1), 2 * kBytesS>, s / kPerSpan + 1);
    issue_codes(lds_ring<60 + (ring ^ 1), kBytesA>, lds_ring<62 + (ring ^ 1), kBytesB>, s + 1);
    const char *la = lds_ring<60 + ring, kBytesA>, *lb = lds_ring<62 + ring, kBytesB>, *ls = lds_ring<64 + span, 2 * kBytesS>;
    if constexpr (in_span == 0) {
      const bool short_span = s / kPerSpan * 16 + 16 > pitch_s;
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[i] = scales_of(ls + (wm * 64 + i * 16 + r) * 16, short_span);
#pragma unroll
      for (int j = 0; j < 8; ++j) sb[j] = scales_of(ls + kBytesS + (wn * 128 + j * 16 + r) * 16, short_span);
    }
    [&]<int... Steps>(std::integer_sequence<int, Steps...>) {
      (
          [&] {
            constexpr int Step = Steps, sel = Fp8 ? in_span : in_span * 2 + Step;
            i32x8 af[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              u32x4 lo, hi = {0u, 0u, 0u, 0u};
              if constexpr (Fp8) {
                lo = *reinterpret_cast<const u32x4 *>(la + a_at + i * 2048 + ((place ^ (r >> 1)) << 4));
                hi = *reinterpret_cast<const u32x4 *>(la + a_at + i * 2048 + (((4 + place) ^ (r >> 1)) << 4));
              } else {
                lo = *reinterpret_cast<const u32x4 *>(la + a_at + i * 2048 + (((2 * place + Step) ^ (r >> 1)) << 4));
              }
              af[i] = i32x8{static_cast<int>(lo[0]), static_cast<int>(lo[1]), static_cast<int>(lo[2]), static_cast<int>(lo[3]),
                            static_cast<int>(hi[0]), static_cast<int>(hi[1]), static_cast<int>(hi[2]), static_cast<int>(hi[3])};
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int slot = Fp8 ? place ^ (r >> 2) : (2 * place + Step) ^ (r >> 1);
              const u32x4_t bf = *reinterpret_cast<const u32x4_t *>(lb + b_at + j * 16 * kRowB + (slot << 4));
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[i][j] = mfma_mx<Fp8, sel>(bf, af[i], acc[i][j], sb[j], sa[i]);
            }
          }(),
          ...);
    }(std::make_integer_sequence<int, Fp8 ? 1 : 2>{});
  };

  issue_scales(lds_ring<64, 2 * kBytesS>, 0);
  issue_codes(lds_ring<60, kBytesA>, lds_ring<62, kBytesB>, 0);
  const int full = stages - stages % kPeriod;
  for (int s = 0; s < full; s += kPeriod)
    [&]<int... Is>(std::integer_sequence<int, Is...>) {
      (stage(std::integral_constant<int, Is>{}, s + Is), ...);
    }(std::make_integer_sequence<int, kPeriod>{});
  [&]<int... Is>(std::integer_sequence<int, Is...>) {
    ((full + Is < stages ? stage(std::integral_constant<int, Is>{}, full + Is) : void()), ...);
  }(std::make_integer_sequence<int, kPeriod - 1>{});
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // the last, empty transfers, before the LDS is released

#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int col = n0 + wn * 128 + j * 16 + 4 * place;
    f32x4_t add = {0.f, 0.f, 0.f, 0.f};
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) add[e] = bias[min(col + e, n - 1)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = m0 + wm * 64 + i * 16 + r;
      f32x4_t v = acc[i][j] + add;
      if (relu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
      }
      if (row < m && col < n) store_four(c + row * c_stride + col, n - col, v);
    }
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
  const int64_t tiles_m = ceil_div(m, 256), tiles_n = ceil_div(n, 256);
  if (tunable("gemm_mx.tile", m >= 256 && n >= 256 ? 1 : 0) && kp >= 512 && kp <= (1 << 22) && tiles_m * tiles_n < (1 << 22))
    return by_type(c_type, [&]<class T>(T *) {
      const dim3 tiles(static_cast<unsigned>(tiles_m * tiles_n));
      const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, tiles, dim3(512), 0, as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, relu, static_cast<T *>(c),
                           c_stride, static_cast<int>(m), static_cast<int>(n), static_cast<int>(kp), static_cast<int>(tiles_m), static_cast<int>(tiles_n));
        return check_launch("gemm_mx launch");
      };
      return a_format == SAREK_HIP_MX_FP8 ? run(gemm_mx_tile_kernel<true, T>) : run(gemm_mx_tile_kernel<false, T>);
    });
  const dim3 grid(static_cast<unsigned>(ceil_div(n, 16)), static_cast<unsigned>(ceil_div(m, 16)));
  return by_type(c_type, [&]<class T>(T *) {
    if (a_format == SAREK_HIP_MX_FP8)
      hipLaunchKernelGGL((gemm_mx_kernel<true, T>), grid, dim3(64), 0, as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, relu, static_cast<T *>(c), c_stride, m, n, kp);
    else
      hipLaunchKernelGGL((gemm_mx_kernel<false, T>), grid, dim3(64), 0, as_stream(stream), a_codes, a_scales, b_codes, b_scales, bias, relu, static_cast<T *>(c), c_stride, m, n, kp);
    return check_launch("gemm_mx launch");
  });
}
