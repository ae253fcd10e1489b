// Device side of the microscaled 4-bit format, shared by its kernels.
//
// Blocks of 32 values along a row: 16 bytes of codes (value 2i in the low half of byte i),
// and one byte of scale, 2^(byte - 127), 255 for a block that is no number.  A code is a sign
// over the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A row of W values has ceil(W / 32) blocks,
// those of its codes back to back (so that every block lies on 16 bytes); values behind W are zero.
#ifndef MX4_H_
#define MX4_H_

#include <type_traits>

#include "sub1_common.h"

namespace mx4 {

constexpr int kBlock = 32;        // values
constexpr int kBlockBytes = 16;   // of codes

__host__ __device__ constexpr int blocks_of(int width) { return (width + kBlock - 1) / kBlock; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The scale as the converting instructions take it: a float of that exponent (its byte 0 and 255
// are read as 2^-127 and as no number; checked for every code under every scale).
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes as bf16: exact, as a code has two bits behind its leading one.
__device__ __forceinline__ bf16x8 expand8(uint32_t codes, float scale) {
  union {
    bf16x2 pair[4];
    bf16x8 all;
  } v;
  v.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  v.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  v.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  v.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return v.all;
}

// Eight 16-bit values from `first` on of a row of `width`; zeros behind its end, whatever
// lies there.  Rows may begin anywhere.  Where the end is inside, the row's last eight are read and
// shifted: one load, as a load for each takes its time eight times over.
__device__ __forceinline__ u32x4 load8(const uint16_t *row, int first, int width) {
  u32x4 v = {0, 0, 0, 0};
  if (first + 8 <= width) {
    __builtin_memcpy(&v, row + first, 16);
  } else if (first < width) {
    unsigned __int128 last = 0;
    if (width >= 8) {
      __builtin_memcpy(&last, row + width - 8, 16);
      last >>= 16 * (first + 8 - width);
    } else {
      for (int i = first; i < width; i++) last |= static_cast<unsigned __int128>(row[i]) << (16 * (i - first));
    }
    v = __builtin_bit_cast(u32x4, last);
  }
  return v;
}

// to nearest, ties to even (one instruction)
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}

// Few tokens: a workgroup of kFewWaves wavefronts multiplies 16 * kRows rows of a matrix with 16 *
// kTokens tokens.  A step is 128 values of a row, four blocks: lane l holds block l / 16 of row l % 16
// in one 16-byte load, and the same block of token l % 16, so that the k-th of four v_mfma_f32_16x16x32_bf16
// takes the k-th eight values of every lane's block (which values of a row meet in an instruction does
// not matter as long as both sides agree).  The wavefronts take the steps in turn, which shares the
// lines of a row among them, and their sums meet in LDS in a fixed order: a token's sum depends on
// the row's length alone, not on the launch.
constexpr int kFewWaves = 8;

template <int kRows, int kTokens>
struct FewSums {
  f32x4 of[kRows][kTokens];
};

// rows: `codes` and `scales` of the first row; `rows` that there are from there on.  x[n] is the row of
// activations of this lane's token of tile n (any row where there is none: tokens do not meet).
template <int kRows, int kTokens>
__device__ __forceinline__ void few_products(FewSums<kRows, kTokens> &sums, const uint8_t *__restrict__ codes,
                                             const uint8_t *__restrict__ scales, int rows, int width,
                                             const uint16_t *const (&x)[kTokens]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4;
  const int blocks = blocks_of(width), steps = (blocks + 3) / 4, whole = width / 128;
  const uint8_t *code_row[kRows], *scale_row[kRows];
#pragma unroll
  for (int r = 0; r < kRows; r++) {
    const int row = min(16 * r + (lane & 15), rows - 1);   // rows that are not there repeat the last
    code_row[r] = codes + static_cast<int64_t>(row) * blocks * kBlockBytes;
    scale_row[r] = scales + static_cast<int64_t>(row) * blocks;
  }
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sums.of[r][n] = f32x4{0, 0, 0, 0};

  auto multiply = [&](const u32x4 (&w)[kRows], const uint32_t (&s)[kRows], const u32x4 (&v)[kTokens][4]) {
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const float scale = scale_of(s[r]);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const bf16x8 a = expand8(w[r][k], scale);
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sums.of[r][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, __builtin_bit_cast(bf16x8, v[n][k]),
                                                                  sums.of[r][n], 0, 0, 0);
      }
    }
  };
  int step = wave;
#pragma unroll 2
  for (; step < whole; step += kFewWaves) {
    const int block = 4 * step + group;
    u32x4 w[kRows], v[kTokens][4];
    uint32_t s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      w[r] = *reinterpret_cast<const u32x4 *>(code_row[r] + static_cast<int64_t>(block) * kBlockBytes);
      s[r] = scale_row[r][block];
    }
#pragma unroll
    for (int n = 0; n < kTokens; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) __builtin_memcpy(&v[n][k], x[n] + block * kBlock + 8 * k, 16);
    multiply(w, s, v);
  }
  if (step < steps) {   // the last, with blocks that end inside it or are not there
    const int block = 4 * step + group;
    u32x4 w[kRows], v[kTokens][4];
    uint32_t s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      w[r] = u32x4{0, 0, 0, 0};
      s[r] = 0;
      if (block < blocks) {
        w[r] = *reinterpret_cast<const u32x4 *>(code_row[r] + static_cast<int64_t>(block) * kBlockBytes);
        s[r] = scale_row[r][block];
      }
    }
#pragma unroll
    for (int n = 0; n < kTokens; n++)
#pragma unroll
      for (int k = 0; k < 4; k++) v[n][k] = load8(x[n], block * kBlock + 8 * k, width);
    multiply(w, s, v);
  }
}

// The wavefronts' sums added up: tile i = r * kTokens + n of the workgroup is given to use(r, n, sum) by
// wavefront i % kFewWaves, where lane l has the sums of rows 4 (l / 16) to + 3 of the tile and token l % 16.
template <int kRows, int kTokens, class Use>
__device__ __forceinline__ void few_join(const FewSums<kRows, kTokens> &sums, f32x4 *lds, Use use) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kTiles = kRows * kTokens;
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) lds[(wave * kTiles + r * kTokens + n) * 64 + lane] = sums.of[r][n];
  __syncthreads();
  for (int i = wave; i < kTiles; i += kFewWaves) {
    f32x4 sum = lds[i * 64 + lane];
#pragma unroll
    for (int other = 1; other < kFewWaves; other++) sum += lds[(other * kTiles + i) * 64 + lane];
    use(i / kTokens, i % kTokens, sum);
  }
}
template <int kRows, int kTokens>
constexpr int kFewLds = kRows *kTokens * 64 * kFewWaves;   // f32x4

// One token: kLanes lanes, a wavefront or half of one, take a whole row, a block a lane at a time: a row's codes are
// read as they lie, 1 KB a load, and so are its scales.  (Few tokens' lanes above read 16 rows' 64 bytes a load, which
// the L1 takes several times as long for, but share them among 16 tokens.)  The token's values wait in LDS, kLanes
// blocks' four parts of 16 bytes each back to back; v_dot2_f32_bf16 multiplies two at a time.  One token
// through 2080 x 6144 3.6 us (by the kernel above 6.1), through 6144 x 2080 3.5 (4.3), of which some 2.3 are a
// launch's; two tokens so 4.4 and 4.6 (by the kernels of a few 5.3, 4.1), four 6.3 and 6.5 (5.4, 4.3).
constexpr int kOneWaves = 8;
constexpr int kOneMostBytes = 128 * 1024;   // of LDS, for the widest row
constexpr int kPlainLds = 64 * 1024;        // what a launch may have without asking (which takes the host 0.4 us)

__host__ __device__ constexpr int one_lds_bytes(int width) { return (blocks_of(width) + 63) / 64 * 4096; }
static_assert(one_lds_bytes(SUB1_MX4_MAX_WIDTH) <= kOneMostBytes, "every width has room");
template <int kLanes>
constexpr int kOneRows = kOneWaves * 64 / kLanes;   // of a workgroup, at once

// Half a wavefront a row where the last turn of a whole one would leave half of it or more idle and rows are many
// enough for a workgroup every other compute unit (one token through 4096 x 1024 2.4 us, by whole ones 2.7; through
// 3001 x 1023 2.5 and 2.8; 26 pairs of a sparse MLP of 1024 x 4096 31.7 and 40).
inline bool halves_pay(int width, int64_t rows) {
  const int over = blocks_of(width) % 64;
  return over > 0 && over <= 32 && rows >= 128 * kOneRows<32>;
}

template <int kLanes>
__device__ __forceinline__ void stage_one(u32x4 *lds, const uint16_t *x, int width) {
  const int parts = (blocks_of(width) + kLanes - 1) / kLanes * kLanes * 4;
  for (int i = threadIdx.x; i < parts; i += 64 * kOneWaves)
    lds[i / (4 * kLanes) * (4 * kLanes) + (i & 3) * kLanes + (i >> 2) % kLanes] = load8(x, 8 * i, width);
}

// Sums over kLanes lanes, in the last of them.
template <int kLanes>
__device__ __forceinline__ float lanes_sum(float v) {
  auto add = [&](auto control, auto rows) {
    v += __int_as_float(sub1::dpp_or_zero<decltype(control)::value, decltype(rows)::value>(__float_as_int(v)));
  };
  add(std::integral_constant<int, sub1::kDppRowShr1>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr2>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr4>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr8>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppBcast15>{}, std::integral_constant<int, 0xa>{});
  if (kLanes == 64) add(std::integral_constant<int, sub1::kDppBcast31>{}, std::integral_constant<int, 0xc>{});
  return v;
}

// What a row's lanes load first: asked for before the token is in LDS, and for all rows that a wavefront takes.
struct OneFirst {
  u32x4 w;
  uint32_t s;
};
__device__ __forceinline__ OneFirst one_block(const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                              int64_t first, int block, int blocks) {
  const int64_t at = first + min(block, blocks - 1);
  return {*reinterpret_cast<const u32x4 *>(codes + at * kBlockBytes), scales[at]};
}

// The product of the row whose blocks begin at `first` with the token in LDS, in the last of its lanes.
template <int kLanes>
__device__ __forceinline__ float one_product(OneFirst v, const uint8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                             int64_t first, int blocks, const u32x4 *lds) {
  const int lane = threadIdx.x % kLanes;
  float sum = 0;
  for (int begin = 0; begin < blocks; begin += kLanes) {
    // behind the last block: nothing (its codes were loaded again, and LDS holds zeros)
    const u32x4 now = begin + lane < blocks ? v.w : u32x4{0, 0, 0, 0};
    const float scale = scale_of(begin + lane < blocks ? v.s : 0);
    if (begin + kLanes < blocks) v = one_block(codes, scales, first, begin + kLanes + lane, blocks);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      union {
        bf16x8 all;
        bf16x2 pair[4];
      } a, x;
      a.all = expand8(now[k], scale);
      x.all = __builtin_bit_cast(bf16x8, lds[begin * 4 + k * kLanes + lane]);
#pragma unroll
      for (int i = 0; i < 4; i++) sum = __builtin_amdgcn_fdot2_f32_bf16(a.pair[i], x.pair[i], sum, false);
    }
  }
  return lanes_sum<kLanes>(sum);
}

}  // namespace mx4

#endif  // MX4_H_
