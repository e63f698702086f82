// Products of microscaled rows with 4-bit weights (layout: mx_common.hpp) on the matrix unit's scaled instructions:
//   C[M x N] = A[M x K] . B[N x K]^T (+ bias) (ReLU),  A in e4m3 or e2m1, B in e2m1, sums in float32.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 rows of each operand and 128 of k, four blocks of 32, and a scale byte for each row and
// block: lane l brings row l % 16, and the scale of block l / 16.  Of a 4-bit operand its 16 bytes are that block too; of an 8-bit one
// its first 16 bytes are values 16 (l / 16) and on, its second 64 + 16 (l / 16) and on.  The weights are the first operand, so a lane's
// results are columns of one row of C, four in a row.
// v_mfma_scale_f32_32x32x64_f8f6f4 is the same for 32 rows and 64 of k, lane l bringing row l % 32 and the scale of block l / 32; of an 8-bit
// operand its first 16 bytes are values 16 (l / 32) and on, its second 32 + 16 (l / 32) and on.
//
// How the instruction adds (measured): products of eight neighbours in k meet on a grid of 2^-13 of what the largest exponents among them
// would give, and what is below is dropped; the eights of a block are then added exactly, and the blocks and C in float32.  4-bit products fit
// the grid, so a block's sum is exact.  8-bit ones do not (2^-9 times 1/2 beside 448 times 6), so 8-bit codes are taken in two parts, of
// magnitudes from 2 on and of those below (split), each with an instruction of its own: the products of either part fit the grid, 2^-3 beside up
// to 2^11.4 and 2^-10 beside up to 2^3.5, and sums are float32 sums of exact products.  In one pass, twice as fast, C was up to 4.7e-5 of the sum
// of the magnitudes off, a half and more of it where large products cancel.
//
// Streams of the instruction alone, random codes: 8-bit with 4-bit rows 4300 TFLOP/s, in two parts with the parting of their codes between
// the instructions 2290 (the codes brought to bf16 and 16-bit instructions: 2050), 4-bit ones 5830, on 32x32x64 6600 (16x16x128 is bound by its
// issue there); the clock falls with the data, zeros reach 9600 in 4 bits.  Of few rows the weights' bytes are the bound, of many the matrix
// unit: gemm_mx_stream_kernel and gemm_mx_tile_kernel.
#include <type_traits>
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

typedef __attribute__((ext_vector_type(16))) float f32x16;
template <bool Fp8, int Scale> __device__ __forceinline__ f32x16 mfma_mx32(u32x4 b, i32x8 a, f32x16 c, int b_scales, int a_scales) {
  const i32x8 wide = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide, a, c, kFormatE2M1, Fp8 ? kFormatE4M3 : kFormatE2M1, Scale, b_scales, Scale,
                                                         a_scales);
}

__device__ __forceinline__ i32x8 join(u32x4 low, u32x4 high) {
  return i32x8{static_cast<int>(low[0]), static_cast<int>(low[1]), static_cast<int>(low[2]), static_cast<int>(low[3]),
               static_cast<int>(high[0]), static_cast<int>(high[1]), static_cast<int>(high[2]), static_cast<int>(high[3])};
}
// Four of a lane's e4m3 codes in two parts, zeros in the place of what is in the other: a magnitude from 2 on has the code's bit 6 set.
__device__ __forceinline__ void split(i32x8 &codes, i32x8 &large, int word) {
  typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
  const uint32_t c = static_cast<uint32_t>(codes[word]);
  const u16x2 whole_bytes = __builtin_bit_cast(u16x2, c >> 6 & 0x01010101u) * u16x2{255, 255};
  large[word] = static_cast<int>(c & __builtin_bit_cast(uint32_t, whole_bytes));
  codes[word] = static_cast<int>(c & ~__builtin_bit_cast(uint32_t, whole_bytes));
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------

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

// Small tiles of C, both operands brought to LDS by transfers, kRing - 1 stages ahead.  Eight waves: WM by WN of them share out the tile of
// C, each MT by NT row and column tiles of 16, and Q of them in each place take every Q-th step of 128 k; a stage is Q steps.  Their sums
// are added in order at the end.
// Few rows are bound by the weights' bytes, and those by how many are under way: rings of 102 to 153 KiB, a workgroup to a compute unit, so that
// even one row of C keeps every one of them loading.  K is split over a workgroup's waves, not over workgroups: their sums
// meet in LDS, with no second launch and no memory for them.  8-bit rows: 1 x 8192 x 8192 8.6 us, 4.2 TB/s; 61 x 11007 x 4095 12.7, its 172
// tiles of 64 x 64 being less than the compute units; 512 x 4096 x 4096 23.5, 1024 x 4096 x 4096 30.3, 1130 TFLOP/s, bound by a start and an
// end that no other workgroup covers (6 us) and by the matrix unit, busy for half of the time.  (LDS conflicts, 11 to 33 % of its cycles, are
// all of the sums' exchange at the end: 1792 clocks of a 64 x 64 tile's workgroup, whatever K is.)
template <bool Fp8, class T, int MT, int NT, int WM, int WN, int kRing>
__global__ __launch_bounds__(512) void gemm_mx_stream_kernel(const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales,
                                                             const uint8_t *__restrict__ b, const uint8_t *__restrict__ b_scales,
                                                             const float *__restrict__ bias, int relu, T *__restrict__ c,
                                                             int64_t c_stride, int m, int n, int kp, int tiles_m, int tiles_n) {
  constexpr int kPlaces = WM * WN, Q = 8 / kPlaces, kStage = Q * 128, kTM = 16 * MT * WM, kTN = 16 * NT * WN;
  constexpr int kRowA = Fp8 ? kStage : kStage / 2, kRowB = kStage / 2;             // bytes of a row in a stage
  constexpr int kBytesA = kTM * kRowA, kBytesB = kTN * kRowB, kWordsA = kTM * Q, kWordsB = kTN * Q;
  constexpr int kBytes = kBytesA + kBytesB + (kWordsA + kWordsB) * 4;
  constexpr int kMovesA = kBytesA / 8192, kMovesB = kBytesB / 8192, kMoves = kMovesA + kMovesB;   // a wave's transfers of a stage's codes
  static_assert(kBytesA % 8192 == 0 && kBytesB % 8192 == 0 && kWordsA % 64 == 0 && kWordsB % 64 == 0 && (kWordsA + kWordsB) / 64 <= 8, "whole transfers");
  static_assert(kRing * kBytes <= 160 * 1024 && (kRing - 2) * kMoves < 64, "LDS, vmcnt");
  constexpr int kChunk = MT * NT * 1024;   // a wave's sums
  static_assert((8 + kRing - 1) / kRing * kChunk <= kBytes, "the waves' sums go into the stages' places");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, place = lane >> 4;
  const int q = wave / kPlaces, wm = wave % kPlaces / WN, wn = wave % WN;           // this wave's step and its part of the tile
  int tm, tn;
  tile_of_block(tiles_m, tiles_n, 1, tm, tn);
  const int m0 = tm * kTM, n0 = tn * kTN;
  const int pitch_a = Fp8 ? kp : kp / 2, pitch_b = kp / 2, pitch_s = kp / kMxBlock, steps = kp / 128, stages = (steps + Q - 1) / Q;
  const uint32_t rows_a = static_cast<uint32_t>(min(m - m0, kTM)), rows_b = static_cast<uint32_t>(min(n - n0, kTN));
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(a + static_cast<int64_t>(m0) * pitch_a, rows_a * pitch_a);
  const __amdgpu_buffer_rsrc_t rb = make_rsrc(b + static_cast<int64_t>(n0) * pitch_b, rows_b * pitch_b);
  // Transfers: lanes past the rows that exist, or past a row's end in the last stage, are sent out of range and bring zeros.  A piece of 16
  // bytes lies at its number in the row with the last bits turned by the row's (its quad's where a row is 128 bytes).
  constexpr uint32_t kOutOfRange = 0x80000000u;   // (a tile's rows end below it, and so does what is added along k)
  auto turn = [](int row, int row_bytes) { return (row_bytes >= 256 ? row & 15 : row >> 1 & 7) << 4; };
  uint32_t off_a[kMovesA], off_b[kMovesB];
  int at_a[kMovesA], at_b[kMovesB];    // where in the row, bytes
#pragma unroll
  for (int i = 0; i < kMovesA; ++i) {
    const int in = (wave + 8 * i) * 1024 + lane * 16, row = in / kRowA;
    at_a[i] = in % kRowA ^ turn(row, kRowA);
    off_a[i] = row < static_cast<int>(rows_a) ? row * pitch_a + at_a[i] : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < kMovesB; ++i) {
    const int in = (wave + 8 * i) * 1024 + lane * 16, row = in / kRowB;
    at_b[i] = in % kRowB ^ turn(row, kRowB);
    off_b[i] = row < static_cast<int>(rows_b) ? row * pitch_b + at_b[i] : kOutOfRange;
  }
  // Scales: a word of four to a row and step, step by step; each of the first waves brings 64 of them.
  const bool scale_a = wave < kWordsA / 64;
  const int word = (scale_a ? wave : wave - kWordsA / 64) * 64 + lane, word_row = word % (scale_a ? kTM : kTN), word_step = word / (scale_a ? kTM : kTN);
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(scale_a ? a_scales + static_cast<int64_t>(m0) * pitch_s : b_scales + static_cast<int64_t>(n0) * pitch_s, (scale_a ? rows_a : rows_b) * pitch_s);
  const uint32_t off_s = word_step < Q && word_row < static_cast<int>(scale_a ? rows_a : rows_b) ? word_row * pitch_s + word_step * 4 : kOutOfRange;
  // Transfer `i` of stage s: its scales, then A's, then B's.
  auto move = [&](char *to, int s, int i) __attribute__((always_inline)) {
    if (i == 0) {
      if (wave < (kWordsA + kWordsB) / 64)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_PTR void *)(to + kBytesA + kBytesB + wave * 256), 4,
                                                 static_cast<int>(s * Q + word_step < steps ? off_s + s * Q * 4 : kOutOfRange), 0, 0, 0);
    } else if (i <= kMovesA) {
      dma16(ra, s * kRowA + at_a[i - 1] < pitch_a ? off_a[i - 1] + s * kRowA : kOutOfRange, 0, to + (wave + 8 * (i - 1)) * 1024);
    } else {
      const int j = i - 1 - kMovesA;
      dma16(rb, s * kRowB + at_b[j] < pitch_b ? off_b[j] + s * kRowB : kOutOfRange, 0, to + kBytesA + (wave + 8 * j) * 1024);
    }
  };
  f32x4_t acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto read = [](const char *p) { return *reinterpret_cast<const u32x4 *>(p); };
  const int row_a = wm * 16 * MT + r, row_b = wn * 16 * NT + r;
  const int a_at = row_a * kRowA + (q * (Fp8 ? 128 : 64) + place * 16 ^ turn(r, kRowA)), b_at = kBytesA + row_b * kRowB + (q * 64 + place * 16 ^ turn(r, kRowB));
  const int a_hi = row_a * kRowA + (q * 128 + 64 + place * 16 ^ turn(r, kRowA));
  const int sa_at = kBytesA + kBytesB + (q * kTM + row_a) * 4 + place, sb_at = kBytesA + kBytesB + (kWordsA + q * kTN + row_b) * 4 + place;
  auto stage = [&]<int I>(std::integral_constant<int, I>, int s) __attribute__((always_inline)) {
    const char *const from = lds_ring<80 + I, kBytes>;
    // What the next stages have in flight may stay there (of a wave with scales to bring, one transfer less).
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((kRing - 2) * kMoves));
    barrier_no_fence();
    // All fragments are asked for before the first MFMA. Where a wave has four MFMA tiles and more, the transfers go one by one between the MFMAs,
    // as all at once keep the waves waiting to issue them (61 x 11007 x 4095 in 8 bits 13.9 us, so 12.9; 512 x 4096 x 4096 25.5, so 23.5; 16 x
    // 11008 x 4096 on 32 x 64 tiles 9.3, so 9.1); below there is too little to hide them behind, and they go first (16 x 4096 x 11008 on 16 x
    // 32 tiles 9.5 us, between the MFMAs 10.0; 1 x 8192 x 8192 on 32 x 32 tiles in 4 bits 9.1 and 9.3).
    constexpr bool kBetween = MT * NT >= 4;
    if constexpr (!kBetween) {
#pragma unroll
      for (int t = 0; t <= kMoves; ++t) move(lds_ring<80 + (I + kRing - 1) % kRing, kBytes>, s + kRing - 1, t);
    }
    u32x4 bf[NT], lo[MT], hi[Fp8 ? MT : 1];
    int sb[NT], sa[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      bf[j] = read(from + b_at + j * 16 * kRowB);
      sb[j] = static_cast<uint8_t>(from[sb_at + j * 64]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      lo[i] = read(from + a_at + i * 16 * kRowA);
      if constexpr (Fp8) hi[i] = read(from + a_hi + i * 16 * kRowA);
      sa[i] = static_cast<uint8_t>(from[sa_at + i * 64]);
    }
    if constexpr (kBetween) __builtin_amdgcn_sched_barrier(0);
    // A fragment's parts: the large one's MFMAs and then the small one's.  The next fragment is parted between them.
    constexpr int kParts = Fp8 ? 2 : 1, kMfmas = kParts * NT, kAll = MT * kMfmas;
    i32x8 af[2], large[2];
    auto take = [&](int i) { af[i & 1] = join(lo[i], Fp8 ? hi[Fp8 ? i : 0] : u32x4{0u, 0u, 0u, 0u}); };
    take(0);
    if constexpr (Fp8) {
#pragma unroll
      for (int w = 0; w < 8; ++w) split(af[0], large[0], w);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (i + 1 < MT) take(i + 1);
#pragma unroll
      for (int t = 0; t < kMfmas; ++t) {
        const int j = t % NT, n = i * kMfmas + t;
        // transfers (kMoves + 1) n / kAll of the n-th MFMA and on
        if constexpr (kBetween) {
#pragma unroll
          for (int u = (kMoves + 1) * n / kAll; u < (kMoves + 1) * (n + 1) / kAll; ++u)
            move(lds_ring<80 + (I + kRing - 1) % kRing, kBytes>, s + kRing - 1, u);
        }
        if constexpr (Fp8) {
#pragma unroll
          for (int w = 8 * t / kMfmas; w < 8 * (t + 1) / kMfmas; ++w)
            if (i + 1 < MT) split(af[(i + 1) & 1], large[(i + 1) & 1], w);
        }
        acc[i][j] = mfma_mx<Fp8, 0>(bf[j], Fp8 && t < NT ? large[i & 1] : af[i & 1], acc[i][j], sb[j], sa[i]);
        if constexpr (kBetween) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  constexpr int kQuads = kTN / 4, kRowsAtOnce = 512 / kQuads;   // of a row of the tile; rows that the threads cover at a time
  const int col4 = threadIdx.x % kQuads, col = n0 + col4 * 4;   // this thread's columns of C
  f32x4_t add = {0.f, 0.f, 0.f, 0.f};
  if (bias) {   // (before the first transfer: loads come in order)
#pragma unroll
    for (int e = 0; e < 4; ++e) add[e] = bias[min(col + e, n - 1)];
  }
  [&]<int... Is>(std::integer_sequence<int, Is...>) {
    (
        [&] {
#pragma unroll
          for (int t = 0; t <= kMoves; ++t) move(lds_ring<80 + Is, kBytes>, Is, t);
        }(),
        ...);
  }(std::make_integer_sequence<int, kRing - 1>{});
  for (int s = 0; s < stages; s += kRing)
    [&]<int... Is>(std::integer_sequence<int, Is...>) {
      ((s + Is < stages ? stage(std::integral_constant<int, Is>{}, s + Is) : void()), ...);
    }(std::make_integer_sequence<int, kRing>{});
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // the last, empty transfers: the stages' places take the sums
  barrier_no_fence();
  // Every wave's sums into LDS, a tile's 16 bytes of row r and column quad p at 4 r + p with the row turned by the column tile's number, then
  // a thread to four columns of a row: its Q sums in order, and C by rows.
  auto chunk = [&](int of) {   // the sums of wave `of`
    char *base = lds_ring<80, kBytes>;
    [&]<int... Is>(std::integer_sequence<int, Is...>) { ((base = of % kRing == Is ? lds_ring<80 + Is, kBytes> : base), ...); }(std::make_integer_sequence<int, kRing>{});
    return reinterpret_cast<f32x4_t *>(base + of / kRing * kChunk);
  };
  f32x4_t *const to = chunk(wave);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) to[(i * NT + j) * 64 + (r ^ (j & 3)) * 4 + place] = acc[i][j];
  wait_lds();
  barrier_no_fence();
  const int tile_j = col4 / 4 % NT, part_n = col4 / 4 / NT;
#pragma unroll
  for (int turn_of = 0; turn_of < (kTM + kRowsAtOnce - 1) / kRowsAtOnce; ++turn_of) {
    const int row_in = turn_of * kRowsAtOnce + threadIdx.x / kQuads, tile_i = row_in / 16 % MT, part_m = row_in / 16 / MT;
    const int row = m0 + row_in;
    if ((kTM % kRowsAtOnce && row_in >= kTM) || row >= m || col >= n) continue;
    const int at = (tile_i * NT + tile_j) * 64 + ((row_in & 15) ^ (tile_j & 3)) * 4 + (col4 & 3);
    f32x4_t v = chunk(part_m * WN + part_n)[at];
#pragma unroll
    for (int w = 1; w < Q; ++w) v += chunk(w * kPlaces + part_m * WN + part_n)[at];
    v += add;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (relu) v[e] = v[e] < 0.f ? 0.f : v[e];
    store_four(c + row * c_stride + col, n - col, v);
  }
}

// ---- 256 x 256 tiles -----------------------------------------------------------------------------------------------------------------

// Eight waves, each with its part of C in registers.  Both operands go through LDS, by transfers that are issued a stage or two ahead and one
// at a time between the MFMAs; before a stage's last step comes the barrier for the next stage, whose first fragments are read in that step.
// 8-bit rows take stages of 128 k, three in LDS, and 64 x 128 of C to a wave: each of A's codes is parted by two waves (of 128 x 64 by
// four), five instructions for four codes.  4-bit ones take 256 k, two, and 128 x 64.
// Measured: 4095 x 11008 x 4096 in 8 bits 235 us, 1570 TFLOP/s, the matrix unit busy for 84 % of the time at 2.0 GHz; 8192^3 in 4 bits, C
// float32, 270 us, 4070 TFLOP/s, busy for 56 % at 1.85 GHz.  What bounds 8-bit rows: the same on zeros takes 197 us, three turns of 66, where
// 2.69 turns of 58 are the matrix unit's rate at 2.4 GHz; a turn's start and end are 8 of it, the clock on real data the rest.  4-bit rows: on
// zeros 173 us, on real data that lies in LDS 219, all of it coming from the L2 249.  Not taken: a workgroup that goes on to its next
// tile, its first stages moved during the last of this one (8192^3 267 to 330 us: the wait for transfers waits for C's stores, too).
template <bool Fp8, class T>
__global__ __launch_bounds__(512) void gemm_mx_tile_kernel(const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales,
                                                           const uint8_t *__restrict__ b, const uint8_t *__restrict__ b_scales,
                                                           const float *__restrict__ bias, int relu, T *__restrict__ c, int64_t c_stride,
                                                           int m, int n, int kp, int tiles_m, int tiles_n, bool past_caches) {
  static_assert(!Fp8 || sizeof(T) == 2, "C of 8-bit rows is 16-bit");
  constexpr int kStage = Fp8 ? 128 : 256;            // values of k in a stage: 128 bytes of a row of A
  constexpr int kRowB = Fp8 ? 64 : 128;              // bytes of a row of B in a stage
  constexpr int kRing = Fp8 ? 3 : 2;                 // stages in LDS
  constexpr int kPerSpan = 512 / kStage;             // stages that 16 scale bytes of a row last
  constexpr int kPeriod = Fp8 ? 12 : 2;              // stages after which places in LDS and in the span repeat
  constexpr int kBytesA = 256 * 128, kBytesB = 256 * kRowB, kBytesS = 256 * 16;
  constexpr int kMovesA = kBytesA / 1024 / 8, kMovesB = kBytesB / 1024 / 8;   // transfers of a wave in a stage
  constexpr int kWavesN = Fp8 ? 2 : 4, kWavesM = 8 / kWavesN;
  constexpr int kWaveRows = 256 / kWavesM, kWaveColumns = 256 / kWavesN;
  constexpr int kTilesA = kWaveRows / 32, kTilesB = kWaveColumns / 32;
  static_assert(kPeriod % kRing == 0 && kPeriod % kPerSpan == 0 && kRing * (kBytesA + kBytesB) + 2 * kBytesS + 1040 <= 160 * 1024, "ring");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 31, place = lane >> 5;
  const int wm = wave / kWavesN, wn = wave % kWavesN;
  int tm, tn;
  tile_of_block(tiles_m, tiles_n, 1, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;
  const int pitch_a = Fp8 ? kp : kp / 2, pitch_b = kp / 2, pitch_s = kp / kMxBlock;
  const int rows_a = min(256, m - m0), rows_b = min(256, n - n0);
  const bool of_a = wave < 4;
  const uint8_t *const a_from = a + static_cast<int64_t>(m0) * pitch_a, *const b_from = b + static_cast<int64_t>(n0) * pitch_b;
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(of_a ? a_scales + static_cast<int64_t>(m0) * pitch_s : b_scales + static_cast<int64_t>(n0) * pitch_s,
                                              static_cast<uint32_t>(of_a ? rows_a : rows_b) * pitch_s);
  // Where piece q (16 bytes) of a row lies in its row of LDS: at q with its last bits turned by the row's, row / 2 % 8 in rows of 128 bytes, row /
  // 8 % 4 in rows of 64.  A ds_read_b128 is served 16 lanes at a time, row quads 0, 3, 5 and 6 of eight and then the others; their pieces
  // meet no bank twice so.  (Of the LDS cycles, which are 15 % of the time in 8 bits and 35 % in 4, 11 and 20 % are conflicts: of the scales' reads,
  // 2 and 8 clocks each, and of C on its way out.  The counter grows with k by just the former.)
  auto turn = [](int row, int row_bytes) { return row_bytes == 64 ? row >> 3 & 3 : row >> 1 & 7; };
  uint32_t off_a[kMovesA], off_b[kMovesB];
#pragma unroll
  for (int i = 0; i < kMovesA; ++i) {
    const int row = (wave + 8 * i) * 8 + (lane >> 3);
    off_a[i] = static_cast<uint32_t>(row) * pitch_a + (((lane & 7) ^ turn(row, 128)) << 4);
  }
#pragma unroll
  for (int i = 0; i < kMovesB; ++i) {
    constexpr int chunks = kRowB / 16;
    const int row = (wave + 8 * i) * (64 / chunks) + lane / chunks;
    off_b[i] = static_cast<uint32_t>(row) * pitch_b + (((lane % chunks) ^ turn(row, kRowB)) << 4);
  }
  const uint32_t off_s = static_cast<uint32_t>((wave & 3) * 64 + lane) * pitch_s;
  const int stages = kp / kStage, last_span = (stages - 1) / kPerSpan;

  // Rows past the end are out of the resources' range and read as zeros; past the last stage the range is empty, and nothing moves.
  auto move_a = [&](char *la, int i, int s) {
    dma16(make_rsrc(a_from, s < stages ? static_cast<uint32_t>(rows_a) * pitch_a : 0u), off_a[i], s * 128, la + (wave + 8 * i) * 1024);
  };
  auto move_b = [&](char *lb, int i, int s) {
    dma16(make_rsrc(b_from, s < stages ? static_cast<uint32_t>(rows_b) * pitch_b : 0u), off_b[i], s * kRowB, lb + (wave + 8 * i) * 1024);
  };
  // A row's last span may be 8 bytes: then the 16 that end with the row are taken.
  char *const ls = lds_ring<68, 2 * kBytesS + 16>;
  auto move_scales = [&](int span) { dma16(rs, off_s, min(min(span, last_span) * 16, pitch_s - 16), ls + wave * 1024); };

  f32x16 acc[kTilesA][kTilesB];
#pragma unroll
  for (int i = 0; i < kTilesA; ++i)
#pragma unroll
    for (int j = 0; j < kTilesB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // Scales: a lane reads the bytes of a row for 256 of k (8-bit; two stages) or 512 (4-bit; two stages too) and keeps those that its place
  // needs, in the order of the steps.
  using Raw = std::conditional_t<Fp8, u32x2_t, u32x4>;
  constexpr int kWords = Fp8 ? 1 : 2;
  int sa[kTilesA][kWords], sb[kTilesB][kWords];
  Raw raw_a[kTilesA], raw_b[kTilesB];
  const uint32_t pick = 0x06040200u + place * 0x01010101u;
  auto keep = [&](int (&to)[kWords], const Raw &d) {
    to[0] = static_cast<int>(__builtin_amdgcn_perm(d[1], d[0], pick));
    if constexpr (!Fp8) to[1] = static_cast<int>(__builtin_amdgcn_perm(d[3], d[2], pick));
  };
  // A lane's 16 bytes of the first row tile; what follows of the row is some bits away: the second half of 8-bit codes (2 pieces on) and
  // their next step (4), the steps of 4-bit ones (2 each).
  int a_at = (wm * kWaveRows + r) * 128 + ((place ^ turn(r, 128)) << 4);
  int b_at = (wn * kWaveColumns + r) * kRowB + ((place ^ turn(r, kRowB)) << 4);
  int sa_at = (wm * kWaveRows + r) * 16, sb_at = kBytesS + (wn * kWaveColumns + r) * 16;
  auto read = [](const char *p) { return *reinterpret_cast<const u32x4 *>(p); };
  // Where in a row's 16 bytes those of stage s begin.  Of a span of 8 bytes they are the second half (which 4-bit rows, that have no second
  // stage then, read first).
  auto raw_at = [&](int s) { return (Fp8 ? (s / 2 & 1) * 8 : 0) + (s / kPerSpan * 16 + 16 > pitch_s ? 8 : 0); };
  auto read_raw = [&](int at) {
    if constexpr (Fp8) {
      return *reinterpret_cast<const u32x2_t *>(ls + at);
    } else {
      typedef u32x4 u32x4_by8 __attribute__((aligned(8)));   // (past the row's 16 bytes: the next row's, not used)
      return static_cast<u32x4>(*reinterpret_cast<const u32x4_by8 *>(ls + at));
    }
  };
  auto read_raw_a = [&](int i, int at) { raw_a[i] = read_raw(sa_at + at + i * 512); };
  auto read_raw_b = [&](int j, int at) { raw_b[j] = read_raw(sb_at + at + j * 512); };

  // Fragments.  B: of this step and the next.  A, 4-bit: the same; 8-bit: one after the other, its large part, and in three turns what is read,
  // what is being parted, and the small part that is left of it.  (A register more than there are, and its traffic waits for the transfers
  // behind it in order.)
  u32x4 bf[2][kTilesB], alo[Fp8 ? 1 : 2 * kTilesA];
  i32x8 af[Fp8 ? 3 : 1], large[Fp8 ? 2 : 1];

  // A stage's MFMAs, and before each what is to be read or moved meanwhile.  During the last step the next stage's first fragments are
  // read, after the barrier that says that it has landed and that this one has been read, and this one's place is filled again.
  auto stage = [&](auto ic, int s) __attribute__((always_inline)) {
    constexpr int I = decltype(ic)::value, ring = I % kRing, next = (I + 1) % kRing;
    constexpr bool first_of_two = I % 2 == 0;
    const char *const la = lds_ring<60 + ring, kBytesA>;
    const char *const lb = lds_ring<64 + ring, kBytesB>;
    const char *const la_next = lds_ring<60 + next, kBytesA>, *const lb_next = lds_ring<64 + next, kBytesB>;
    [[maybe_unused]] const int raw_next = raw_at(s + 1);
    auto landed = [&]() __attribute__((always_inline)) {
      // in flight may be what was asked for after the next stage: the stages behind it
      __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((kRing - 2) * (kMovesA + kMovesB)));
      barrier_no_fence();
    };
    // transfer t of the stage that takes the place of this one
    auto refill = [&](int t) __attribute__((always_inline)) {
      if (t < kMovesA) move_a(lds_ring<60 + ring, kBytesA>, t, s + kRing);
      else if (t < kMovesA + kMovesB) move_b(lds_ring<64 + ring, kBytesB>, t - kMovesA, s + kRing);
    };
    asm volatile("" : "+v"(a_at), "+v"(b_at), "+v"(sa_at), "+v"(sb_at));   // (not one register for each place in LDS across the loop)
    if constexpr (first_of_two) {
#pragma unroll
      for (int j = 0; j < kTilesB; ++j) keep(sb[j], raw_b[j]);
#pragma unroll
      for (int i = 0; i < kTilesA; ++i) keep(sa[i], raw_a[i]);
    }
    if constexpr (Fp8) {
      [&]<int... Steps>(std::integer_sequence<int, Steps...>) {
        (
            [&] {
              constexpr int Step = Steps;
              const char *const from_a = Step == 0 ? la : la_next, *const from_b = Step == 0 ? lb : lb_next;   // of the next step
              if (Step == 1) landed();
#pragma unroll
              for (int t = 0; t < 16; ++t) {
                const int i = t >> 3, part = t >> 2 & 1, j = part == 0 ? t & 3 : 3 - (t & 3), f = 4 * I + 2 * Step + i;   // f: the fragment of A
                const int at = a_at ^ (Step ^ 1) << 6;
                if ((t & 7) < 2) {   // the fragment after the next, half by half
                  const u32x4 half = read(from_a + (at ^ (t & 1) << 5) + i * 4096);
#pragma unroll
                  for (int w = 0; w < 4; ++w) af[(f + 2) % 3][4 * (t & 1) + w] = static_cast<int>(half[w]);
                }
                if (t >= 2 && t < 6) bf[Step ^ 1][t - 2] = read(from_b + (b_at ^ (Step ^ 1) << 5) + (t - 2) * 32 * kRowB);
                // (all of the span's scales have been read before this stage's barrier; the next ones have landed at the next)
                if (Step == 1 && t == 1 && I % kPerSpan == 2) move_scales(s / kPerSpan + 1);
                // one transfer at a time: all of a workgroup's at once keep the path to LDS busy for 768 clocks, and the waves wait to issue them
                if (Step == 1 && t >= 2 && t % 2 == 0) refill(t / 2 - 1);
                if (Step == 1 && !first_of_two && t >= 3 && t % 2 == 1) {
                  if (t < 11) read_raw_b((t - 3) / 2, raw_next);
                  else if (t < 15) read_raw_a((t - 11) / 2, raw_next);
                }
                split(af[(f + 1) % 3], large[(f + 1) % 2], t & 7);
                acc[i][j] = mfma_mx32<true, I % 2 * 2 + Step>(bf[Step][j], part == 0 ? large[f % 2] : af[f % 3], acc[i][j], sb[j][0], sa[i][0]);
                __builtin_amdgcn_sched_barrier(0);
              }
            }(),
            ...);
      }(std::make_integer_sequence<int, 2>{});
    } else {
      [&]<int... Steps>(std::integer_sequence<int, Steps...>) {
        (
            [&] {
              constexpr int Step = Steps, cur = Step & 1, number = I % kPerSpan * 4 + Step;
              const char *const from_a = Step < 3 ? la : la_next, *const from_b = Step < 3 ? lb : lb_next;
              const int bits = (Step + 1) % 4 << 5;
              if (Step == 3) landed();
#pragma unroll
              for (int t = 0; t < 8; ++t) {
                const int i = t >> 1, j = i & 1 ? 1 - (t & 1) : t & 1;
                if (t == 0 || (t >= 3 && t < 6)) alo[(cur ^ 1) * 4 + (t == 0 ? 0 : t - 2)] = read(from_a + (a_at ^ bits) + (t == 0 ? 0 : t - 2) * 4096);
                if (t == 1 || t == 2) bf[cur ^ 1][t - 1] = read(from_b + (b_at ^ bits) + (t - 1) * 4096);
                if (Step == 3) refill(t);
                if (Step == 3 && t == 7 && first_of_two) move_scales(s / kPerSpan + 1);
                if (Step == 3 && !first_of_two && t >= 2) {
                  if (t < 4) read_raw_b(t - 2, raw_next);
                  else read_raw_a(t - 4, raw_next);
                }
                acc[i][j] = mfma_mx32<false, number % 4>(bf[cur][j], join(alo[cur * 4 + i], u32x4{0u, 0u, 0u, 0u}), acc[i][j], sb[j][number / 4], sa[i][number / 4]);
                __builtin_amdgcn_sched_barrier(0);
              }
            }(),
            ...);
      }(std::make_integer_sequence<int, 4>{});
    }
  };

  // The bias comes before the first transfer: loads come in order, and at the end it would be waited for.  4-bit rows have registers for that of
  // a lane's columns; 8-bit ones put the tile's 256 values into LDS, zeros where there are none.
  [[maybe_unused]] f32x4_t add[Fp8 ? 1 : kTilesB][4];
  if constexpr (Fp8) {
    if (of_a)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(bias ? bias + n0 : nullptr, bias ? static_cast<uint32_t>(rows_b) * 4 : 0u),
                                               (LDS_PTR void *)(lds_ring<69, 1024> + wave * 256), 4, threadIdx.x * 4, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < kTilesB; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) add[j][q][e] = bias ? bias[min(n0 + wn * kWaveColumns + j * 32 + 8 * q + 4 * place + e, n - 1)] : 0.f;
  }
  move_scales(0);
  [&]<int... Ss>(std::integer_sequence<int, Ss...>) {
    (
        [&] {
#pragma unroll
          for (int t = 0; t < kMovesA + kMovesB; ++t) {
            if (t < kMovesA) move_a(lds_ring<60 + Ss, kBytesA>, t, Ss);
            else move_b(lds_ring<64 + Ss, kBytesB>, t - kMovesA, Ss);
          }
        }(),
        ...);
  }(std::make_integer_sequence<int, kRing>{});
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((kRing - 1) * (kMovesA + kMovesB)));
  barrier_no_fence();
#pragma unroll
  for (int j = 0; j < kTilesB; ++j) {
    bf[0][j] = read(lds_ring<64, kBytesB> + b_at + j * 32 * kRowB);
    read_raw_b(j, raw_at(0));
  }
#pragma unroll
  for (int i = 0; i < kTilesA; ++i) {
    const u32x4 first = read(lds_ring<60, kBytesA> + a_at + i * 4096);
    if constexpr (Fp8) af[i] = join(first, read(lds_ring<60, kBytesA> + (a_at ^ 32) + i * 4096));
    else alo[i] = first;
    read_raw_a(i, raw_at(0));
  }
  if constexpr (Fp8) {
#pragma unroll
    for (int w = 0; w < 8; ++w) split(af[0], large[0], w);
  }
  __builtin_amdgcn_sched_barrier(0);
  const int full = stages - stages % kPeriod;
  for (int s = 0; s < full; s += kPeriod)
    [&]<int... Is>(std::integer_sequence<int, Is...>) {
      (stage(std::integral_constant<int, Is>{}, s + Is), ...);
    }(std::make_integer_sequence<int, kPeriod>{});
  [&]<int... Is>(std::integer_sequence<int, Is...>) {
    ((full + Is < stages ? stage(std::integral_constant<int, Is>{}, full + Is) : void()), ...);
  }(std::make_integer_sequence<int, kPeriod - 1>{});
  __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));   // the last, empty transfers, before the LDS is released

  // C goes to memory by whole rows of the tile, put together in LDS in turns, 64 KiB of the tile at a time, an equal share of it for the waves
  // that share their rows: piece q (16 bytes) of row r at q ^ (r % 16).  A lane has row r of a row tile, and four columns in a row for every
  // four registers.
  constexpr int kRowC = 256 * sizeof(T), kShare = 65536 / kWavesM, kTurnRows = kShare / kRowC, kTurns = kWaveRows / kTurnRows, kPiece = 16 / sizeof(T);
  static_assert(kTurnRows % 32 == 0 && kWaveRows % kTurnRows == 0, "whole row tiles");
  char *const lc = (wm < kWavesM / 2 ? lds_ring<60, kBytesA> : lds_ring<61, kBytesA>) + wm % (kWavesM / 2) * kShare;
#pragma unroll
  for (int turn_of = 0; turn_of < kTurns; ++turn_of) {
    barrier_no_fence();   // every wave has left the K loop, or has read the turn before
#pragma unroll
    for (int u = 0; u < kTurnRows / 32; ++u) {
      const int i = turn_of * (kTurnRows / 32) + u, row = u * 32 + r;
#pragma unroll
      for (int j = 0; j < kTilesB; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int column = wn * kWaveColumns + j * 32 + 8 * q + 4 * place, at = column * static_cast<int>(sizeof(T));
          f32x4_t v;
          if constexpr (Fp8) v = *reinterpret_cast<const f32x4_t *>(lds_ring<69, 1024> + column * 4);
          else v = add[j][q];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] += acc[i][j][4 * q + e];
            if (relu) v[e] = v[e] < 0.f ? 0.f : v[e];
          }
          store_four(reinterpret_cast<T *>(lc + row * kRowC + (at ^ (row & 15) << 4)), 4, v);
        }
    }
    wait_lds();
    barrier_no_fence();
#pragma unroll
    for (int u = 0; u < kShare / 1024 / kWavesN; ++u) {
      const int row = wn * (kTurnRows / kWavesN) + u * (1024 / kRowC) + lane * 16 / kRowC, at = lane * 16 % kRowC;
      const u32x4 v = read(lc + row * kRowC + (at ^ (row & 15) << 4));
      const int to_row = m0 + wm * kWaveRows + turn_of * kTurnRows + row, col = n0 + lane % (kRowC / 16) * kPiece;
      if (to_row >= m || col >= n) continue;
      T *const to = c + to_row * c_stride + col;
      if (col + kPiece <= n) {
        if (past_caches) __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(to));
        else *reinterpret_cast<u32x4_any *>(to) = v;
      } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
          if (col + e >= n) continue;
          if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t *>(to)[e] = v[e];
          else reinterpret_cast<uint16_t *>(to)[e] = static_cast<uint16_t>(v[e / 2] >> 16 * (e & 1));
        }
      }
    }
  }
}

}  // namespace
}  // namespace sarek_hip

namespace sarek_hip {
namespace {

// The kernels' tiles of C, and the weights that choose one, about us of a workgroup: `once` for its start and its end, a step for 128 of
// k (8-bit and 4-bit rows). They rank the tiles and are no times. Over 48 products of 1 to 8000 rows, each timed with every tile, the choice is
// behind the best by 0.1 % on average in 8 bits and at most 5.5 % (291 x 4798 x 286 9.8 us for 9.3), in 4 bits by 1.5 % and at most 14 % (926 x
// 123 x 251 4.3 us for 3.8).
constexpr int kShapeCount = 7;
struct Shape { int rows, columns; double once, step8, step4; };
constexpr Shape kShapes[kShapeCount] = {{16, 16, 1.9, 0.077, 0.050}, {16, 32, 2.0, 0.110, 0.080},   {32, 32, 2.0, 0.144, 0.097},  {32, 64, 2.0, 0.175, 0.148},
                                        {64, 64, 2.9, 0.248, 0.190}, {128, 128, 6.0, 0.600, 0.360}, {256, 256, 7.5, 2.050, 0.650}};

// The one that the product takes least time on: a workgroup to a compute unit, as many in turn as there are too many.
bool shape_serves(int shape, int64_t m, int64_t n, int64_t kp) {
  if (shape < 0 || shape >= kShapeCount || (shape == kShapeCount - 1 && kp < 512)) return false;   // (its scales come 16 bytes of a row at a time)
  return ceil_div(m, kShapes[shape].rows) * ceil_div(n, kShapes[shape].columns) < int64_t{1} << 22;   // below 2^32 threads
}
int best_shape(bool fp8, int64_t m, int64_t n, int64_t kp) {
  int best = -1;
  double least = 0.0;
  for (int i = 0; i < kShapeCount; ++i) {
    if (!shape_serves(i, m, n, kp)) continue;
    const Shape &s = kShapes[i];
    const int64_t tiles = ceil_div(m, s.rows) * ceil_div(n, s.columns);
    const double us = static_cast<double>(ceil_div(tiles, compute_units())) * (s.once + static_cast<double>(kp / 128) * (fp8 ? s.step8 : s.step4));
    if (best < 0 || us < least) least = us, best = i;
  }
  return best;
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
    return fail(SAREK_HIP_E_UNSUPPORTED, "gemm_mx: C of 8-bit rows is bf16 or fp16");
  if (c_stride < n) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: rows of C are %lld values apart, less than n = %lld", static_cast<long long>(c_stride), static_cast<long long>(n));
  if (m >= int64_t{1} << 20 || n >= int64_t{1} << 24 || k > int64_t{1} << 23)
    return fail(SAREK_HIP_E_UNSUPPORTED, "gemm_mx: m is below 2^20, n below 2^24, k at most 2^23");
  if (m == 0) return SAREK_HIP_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !c) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: NULL pointer");
  if (misaligned(a_codes, a_scales) || misaligned(b_codes, b_scales)) return fail(SAREK_HIP_E_INVALID_ARG, "gemm_mx: codes start at multiples of 16 bytes, scales of 8");
  const int64_t kp = mx_row_values(k);
  const bool fp8 = a_format == SAREK_HIP_MX_FP8;
  const int forced = static_cast<int>(tunable("gemm_mx.shape", -1));
  const int shape = shape_serves(forced, m, n, kp) ? forced : best_shape(fp8, m, n, kp);
  if (shape < 0) return fail(SAREK_HIP_E_UNSUPPORTED, "gemm_mx: %lld x %lld is more than one launch covers", static_cast<long long>(m), static_cast<long long>(n));
  return by_type(c_type, [&]<class T>(T *) {
    const auto run = [&](auto kernel, int tile_m, int tile_n, auto... more) {
      const int64_t tiles_m = ceil_div(m, tile_m), tiles_n = ceil_div(n, tile_n);
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles_m * tiles_n)), dim3(512), 0, as_stream(stream), a_codes, a_scales, b_codes,
                         b_scales, bias, relu, static_cast<T *>(c), c_stride, static_cast<int>(m), static_cast<int>(n), static_cast<int>(kp),
                         static_cast<int>(tiles_m), static_cast<int>(tiles_n), more...);
      return check_launch("gemm_mx launch");
    };
    const bool whole_lines = ((reinterpret_cast<uintptr_t>(c) | static_cast<uintptr_t>(c_stride) * sizeof(T)) & 127) == 0;
    const bool past_caches = whole_lines && m * n * static_cast<int64_t>(sizeof(T)) >= tunable("gemm_mx.past_caches_mib", 200) << 20;
    // (row tiles, column tiles of a wave; waves below and beside each other; stages in LDS.)  8-bit rows: waves below each other, so that
    // every code is parted by one of them.
    using std::integer_sequence;
    const auto small = [&]<int... P8, int... P4>(integer_sequence<int, P8...>, integer_sequence<int, P4...>) {
      if constexpr (sizeof(T) == 2)
        if (fp8) return run(gemm_mx_stream_kernel<true, T, P8...>, kShapes[shape].rows, kShapes[shape].columns);
      return run(gemm_mx_stream_kernel<false, T, P4...>, kShapes[shape].rows, kShapes[shape].columns);
    };
    switch (shape) {
      case 0: return small(integer_sequence<int, 1, 1, 1, 1, 6>{}, integer_sequence<int, 1, 1, 1, 1, 6>{});
      case 1: return small(integer_sequence<int, 1, 2, 1, 1, 4>{}, integer_sequence<int, 1, 2, 1, 1, 6>{});
      case 2: return small(integer_sequence<int, 1, 2, 2, 1, 6>{}, integer_sequence<int, 2, 1, 1, 2, 6>{});
      case 3: return small(integer_sequence<int, 1, 4, 2, 1, 4>{}, integer_sequence<int, 2, 2, 1, 2, 6>{});
      case 4: return small(integer_sequence<int, 2, 4, 2, 1, 3>{}, integer_sequence<int, 4, 2, 1, 2, 4>{});
      case 5: return small(integer_sequence<int, 2, 8, 4, 1, 3>{}, integer_sequence<int, 4, 4, 2, 2, 4>{});
      default:
        if constexpr (sizeof(T) == 2)
          if (fp8) return run(gemm_mx_tile_kernel<true, T>, 256, 256, past_caches);
        return run(gemm_mx_tile_kernel<false, T>, 256, 256, past_caches);
    }
  });
}
