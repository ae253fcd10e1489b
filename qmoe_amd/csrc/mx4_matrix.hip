// Microscaled 4-bit matrices: values to the format and back, and products with them.
#include "mx4.h"

using namespace mx4;
using sub1::fail;
using sub1::misaligned;

namespace {

// ------------------------------------------------------- to the format and back ---

// Four lanes a block, eight values a lane.  The scale is 2^(floor(log2 largest) - 2), which is read from
// the largest magnitude's exponent and brings it to 4 .. 8 (above 6 is 6); the instruction that packs two
// codes divides by it exactly and rounds to nearest, ties to the even code.
template <class T>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const uint8_t *__restrict__ x, int64_t row_bytes,
                                                           uint32_t rows, int width, uint8_t *__restrict__ codes,
                                                           uint8_t *__restrict__ scales) {
  const uint32_t blocks = blocks_of(width);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, block = at >> 2;   // the caller's rows * blocks * 4 fit
  if (block >= rows * blocks) return;                                    // (all four lanes of a block)
  const uint32_t row = block / blocks;
  Eight<T> v;
  v.load(x + row * row_bytes, static_cast<int>(block - row * blocks) * kBlock + static_cast<int>(at & 3) * 8, width);
  uint32_t largest = 0;   // magnitudes compare as their bits do, and what is no number is above all
#pragma unroll
  for (int i = 0; i < 8; i++) largest = max(largest, __float_as_uint(v.at(i)) & 0x7fffffffu);
  largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 1)));
  largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 2)));
  const uint32_t exponent = largest >> 23;
  const uint32_t byte = exponent == 255 ? 255u : static_cast<uint32_t>(max(static_cast<int>(exponent) - 2, 0));
  uint32_t packed = 0;
  if (exponent != 255) {
    const float scale = byte ? scale_of(byte) : __uint_as_float(0x00400000u);   // 2^-127
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v.at(0), v.at(1), scale, 0);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v.at(2), v.at(3), scale, 1);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v.at(4), v.at(5), scale, 2);
    packed = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(packed, v.at(6), v.at(7), scale, 3);
  }
  reinterpret_cast<uint32_t *>(codes)[at] = packed;
  if ((at & 3) == 0) scales[block] = static_cast<uint8_t>(byte);
}

template <class T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, uint32_t rows,
                                                             int width, uint8_t *__restrict__ out, int64_t row_bytes) {
  const uint32_t blocks = blocks_of(width);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, block = at >> 2;
  if (block >= rows * blocks) return;
  const uint32_t row = block / blocks;
  const uint32_t packed = reinterpret_cast<const uint32_t *>(codes)[at];
  const float scale = scale_of(scales[block]);
  float v[8];
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(packed, scale, 3);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
  Eight<T>::store(out + row * row_bytes, static_cast<int>(block - row * blocks) * kBlock + static_cast<int>(at & 3) * 8,
                  width, v);
}

// ------------------------------------------------------------------- products ---

struct ProductArgs {
  const uint8_t *codes, *scales;
  const uint16_t *x;
  uint16_t *y;
  int64_t ldx, ldy;
  int height, width, tokens;
};

template <int kRows, int kTokens>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_kernel(const ProductArgs p) {
  __shared__ f32x4 lds[kFewLds<kRows, kTokens>];
  const int lane = threadIdx.x & 63;
  const int row0 = blockIdx.x * 16 * kRows, token0 = blockIdx.y * 16 * kTokens;
  const int64_t blocks = blocks_of(p.width);
  const uint16_t *x[kTokens];
#pragma unroll
  for (int n = 0; n < kTokens; n++) {
    const int token = token0 + 16 * n + (lane & 15);
    x[n] = p.x + min(token, p.tokens - 1) * p.ldx;
  }
  FewSums<kRows, kTokens> sums;
  few_products<kRows, kTokens>(sums, p.codes + row0 * blocks * kBlockBytes, p.scales + row0 * blocks, p.height - row0,
                               p.width, x);
  few_join<kRows, kTokens>(sums, lds, [&](int r, int n, f32x4 sum) {
    const int token = token0 + 16 * n + (lane & 15);
    if (token < p.tokens) store_four(p.y + token * p.ldy, row0 + 16 * r + 4 * (lane >> 4), p.height, sum);
  });
}

// The same for rows of a step a wavefront or more: neighbouring lanes read a row's pieces as they lie and hand them
// round through LDS, a part of the wavefront's own, while the next step's are on their way; the lanes that multiply
// are rows apart, and their own loads are pieces of 16 bytes, one by one in the L1.  Sums are added up in the same order.  What bounds it: the
// activations, of which a workgroup reads four times the bytes of its 16 rows, on their way one step ahead.  (Asked for
// two and three steps ahead they measured alike, 13 tokens through 2080 x 6144 8.0 us each, 2 tokens 5.4; that says
// nothing of more on its way: where fetch()'s branches meet, the compiler waits for all loads.)
template <int kRows, int kTokens>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_few_lines_kernel(const ProductArgs p) {
  constexpr int kStage = kRows * 64 + kTokens * 256;   // a wavefront's rows of 64 bytes, tokens of 256
  __shared__ u32x4 lds[kFewWaves * kStage];
  static_assert(kStage >= kRows * kTokens * 64, "the sums take the place of the values");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4;
  const int row0 = blockIdx.x * 16 * kRows, token0 = blockIdx.y * 16 * kTokens;
  const int blocks = blocks_of(p.width), steps = (blocks + 3) / 4, whole = p.width / 128;
  const uint8_t *codes = p.codes + static_cast<int64_t>(row0) * blocks * kBlockBytes;
  const uint8_t *scales = p.scales + static_cast<int64_t>(row0) * blocks;
  FewSums<kRows, kTokens> sums;
  u32x4 *const codes_lds = lds + wave * kStage, *const x_lds = codes_lds + kRows * 64;
  int code_row[kRows], scale_row[kRows];   // rows that are not there repeat the last
  const uint16_t *token[kTokens][4];
#pragma unroll
  for (int r = 0; r < kRows; r++) {
    code_row[r] = min(16 * r + (lane >> 2), p.height - 1 - row0) * blocks;
    scale_row[r] = min(16 * r + (lane & 15), p.height - 1 - row0) * blocks;
  }
#pragma unroll
  for (int n = 0; n < kTokens; n++)
#pragma unroll
    for (int h = 0; h < 4; h++) token[n][h] = p.x + min(token0 + 16 * n + 4 * h + group, p.tokens - 1) * p.ldx;
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sums.of[r][n] = f32x4{0, 0, 0, 0};

  u32x4 next[kRows], next_x[kTokens][4];
  uint32_t next_scales[kRows];
  auto fetch = [&](int step) {
    const int block = min(4 * step + (lane & 3), blocks - 1);
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      next[r] = *reinterpret_cast<const u32x4 *>(codes + (code_row[r] + block) * kBlockBytes);
      if (blocks >= 4)
        __builtin_memcpy(&next_scales[r], scales + scale_row[r] + min(4 * step, blocks - 4), 4);
      else
        next_scales[r] = static_cast<uint32_t>(scales[scale_row[r] + min(group, blocks - 1)]) << 8 * min(group, blocks - 1);
    }
#pragma unroll
    for (int n = 0; n < kTokens; n++)
#pragma unroll
      for (int h = 0; h < 4; h++) {
        if (token0 + 16 * n + 4 * h >= p.tokens) break;   // (what LDS holds there goes nowhere)
        if (step < whole)
          __builtin_memcpy(&next_x[n][h], token[n][h] + 128 * step + 8 * (lane & 15), 16);
        else
          next_x[n][h] = load8(token[n][h], 128 * step + 8 * (lane & 15), p.width);
      }
  };
  if (wave < steps) fetch(wave);
  for (int step = wave; step < steps; step += kFewWaves) {
    const int block = 4 * step + group, from = blocks >= 4 ? min(4 * step, blocks - 4) : 0;
    float scale[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      // behind the last block: its codes, under a scale and with activations that make them nothing
      scale[r] = scale_of(block < blocks ? next_scales[r] >> 8 * (block - from) & 255 : 0);
      codes_lds[r * 64 + (lane & 60) + ((lane & 3) ^ (lane >> 3 & 3))] = next[r];
    }
#pragma unroll
    for (int n = 0; n < kTokens; n++)
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const int i = 4 * h + group;
        if (token0 + 16 * n + 4 * h < p.tokens) x_lds[n * 256 + 16 * i + ((lane & 15) ^ (i & 7))] = next_x[n][h];
      }
    if (step + kFewWaves < steps) fetch(step + kFewWaves);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    u32x4 w[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) w[r] = codes_lds[r * 64 + 4 * (lane & 15) + (group ^ (lane >> 1 & 3))];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      bf16x8 v[kTokens];
#pragma unroll
      for (int n = 0; n < kTokens; n++)
        v[n] = __builtin_bit_cast(bf16x8, x_lds[n * 256 + 16 * (lane & 15) + ((4 * group + k) ^ (lane & 7))]);
#pragma unroll
      for (int r = 0; r < kRows; r++) {
        const bf16x8 a = expand8(w[r][k], scale[r]);
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sums.of[r][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, v[n], sums.of[r][n], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  few_join<kRows, kTokens>(sums, reinterpret_cast<f32x4 *>(lds), [&](int r, int n, f32x4 sum) {
    const int t = token0 + 16 * n + (lane & 15);
    if (t < p.tokens) store_four(p.y + t * p.ldy, row0 + 16 * r + 4 * group, p.height, sum);
  });
}

template <int kLanes>
__global__ __launch_bounds__(64 * kOneWaves) void mx4_one_kernel(const ProductArgs p) {
  extern __shared__ u32x4 one_lds[];
  const int row = blockIdx.x * kOneRows<kLanes> + threadIdx.x / kLanes, blocks = blocks_of(p.width);
  const int64_t first = static_cast<int64_t>(min(row, p.height - 1)) * blocks;   // (all wavefronts fill LDS)
  const OneFirst begin = one_block(p.codes, p.scales, first, threadIdx.x % kLanes, blocks);
  stage_one<kLanes>(one_lds, p.x, p.width);
  __syncthreads();
  const float sum = one_product<kLanes>(begin, p.codes, p.scales, first, blocks, one_lds);
  if (threadIdx.x % kLanes == kLanes - 1 && row < p.height) p.y[row] = static_cast<uint16_t>(two_bf16(sum, 0));
}

template <int kLanes>
int launch_one(const ProductArgs &p, hipStream_t s) {
  if (one_lds_bytes(p.width) > kPlainLds) HIP_TRY(sub1::allow_lds<kOneMostBytes>(mx4_one_kernel<kLanes>));
  mx4_one_kernel<kLanes><<<(p.height + kOneRows<kLanes> - 1) / kOneRows<kLanes>, 64 * kOneWaves, one_lds_bytes(p.width), s>>>(p);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// Many tokens: four wavefronts, two by two, each with 32 kRows rows of the matrix and 32 kTokens tokens, 64
// values of a row a step.  Both sides go through LDS, where two wavefronts read each part.  (A wavefront that
// fetched its 32 rows' 32 bytes of a step straight into its lanes would touch 32 lines for them, and the L1 takes
// longer for that than the matrix cores for the products: 300 tokens through 6144 x 2080 19.0 us, so 18.7 and
// with less in its way below 14.)
// Lane l multiplies block l / 32 of row l % 32 with that of token l % 32: the k-th of a step's four
// v_mfma_f32_32x32x16_bf16 takes the k-th eight values of every lane's block.
template <int kRows, int kTokens>
struct Many {
  static constexpr int rows = 64 * kRows, tokens = 64 * kTokens;   // of a workgroup
};

// The sums of a workgroup's first 256 threads to y, past LDS, so that whole lines of y are written: the lanes
// have four rows of a token each, 8 bytes of a line.  `place` is all of the workgroup's LDS that the tile may take.
template <int kRows, int kTokens, int kPlace>
__device__ __forceinline__ void store_tile(const f32x16 (&sum)[kRows][kTokens], u32x4 (&place)[kPlace], uint16_t *y,
                                           int64_t ldy, int row0, int token0, int height, int tokens) {
  using M = Many<kRows, kTokens>;
  constexpr int kPitch = M::rows + 8;   // 16 bytes further: neighbouring tokens in other banks
  static_assert(M::tokens * kPitch * 2 <= kPlace * 16, "the tile has room");
  uint16_t *const lds = reinterpret_cast<uint16_t *>(place);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, in_tile = lane & 31;
  const bool has_sums = tid < 256;
#pragma unroll
  for (int n = 0; n < kTokens; n++)
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if (!has_sums) break;
        const uint32_t two[2] = {two_bf16(sum[r][n][4 * i], sum[r][n][4 * i + 1]),
                                 two_bf16(sum[r][n][4 * i + 2], sum[r][n][4 * i + 3])};
        __builtin_memcpy(__builtin_assume_aligned(
                             lds + ((wave >> 1) * 32 * kTokens + 32 * n + in_tile) * kPitch +
                                 ((wave & 1) * kRows + r) * 32 + 8 * i + 4 * half, 8),
                         two, 8);
      }
  __syncthreads();
  if (!has_sums) return;
  constexpr int kParts = M::rows / 8, kAtOnce = 256 / kParts;   // parts of 16 bytes of a token, tokens a turn
  const int row = tid % kParts * 8, rows_left = height - row0 - row;
  const uint16_t *from = lds + tid / kParts * kPitch + row;
  uint16_t *to = y + static_cast<int64_t>(token0 + tid / kParts) * ldy + row0 + row;
  const int tokens_left = tokens - token0 - tid / kParts;
  if (rows_left >= 8) {
#pragma unroll 4
    for (int i = 0; i < M::tokens / kAtOnce; i++) {
      u32x4 v;
      __builtin_memcpy(&v, __builtin_assume_aligned(from + i * kAtOnce * kPitch, 16), 16);
      if (i * kAtOnce < tokens_left) __builtin_memcpy(to + i * kAtOnce * ldy, &v, 16);
    }
  } else if (rows_left > 0) {
    for (int i = 0; i * kAtOnce < min(M::tokens, tokens_left); i++)
      for (int k = 0; k < rows_left; k++) to[i * kAtOnce * ldy + k] = from[i * kAtOnce * kPitch + k];
  }
}

// Through registers: the activations a step at a time, the codes 256 values of a row (128 bytes) at a time, in
// four quarters of the rows, one a step.
template <int kRows, int kTokens, int kWaves>
__global__ __launch_bounds__(256, kWaves) void mx4_many_kernel(const ProductArgs p) {
  using M = Many<kRows, kTokens>;
  constexpr int kLoads = M::tokens / 32;                      // of 16 bytes of activations, a thread and step
  constexpr int kQuarter = M::rows / 4;                       // rows
  constexpr int kCodes = (kQuarter + 31) / 32;                // loads of 16 bytes of codes, a thread and step
  // a row's or token's eight parts of 16 bytes, part i at i ^ (row % 8): eight lanes of neighbouring rows
  // that read the same part find it in different banks.  Activations, codes and scales, and the sums of all in their place
  __shared__ u32x4 lds[2 * M::tokens * 8 + 2 * M::rows * 8 + 2 * M::rows / 2];
  u32x4(*const lds_x)[M::tokens * 8] = reinterpret_cast<u32x4(*)[M::tokens * 8]>(lds);
  u32x4(*const lds_w)[M::rows * 8] = reinterpret_cast<u32x4(*)[M::rows * 8]>(lds + 2 * M::tokens * 8);
  uint8_t(*const lds_s)[M::rows * 8] = reinterpret_cast<uint8_t(*)[M::rows * 8]>(lds + 2 * M::tokens * 8 + 2 * M::rows * 8);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, in_tile = lane & 31;
  const int row0 = blockIdx.x * M::rows, token0 = blockIdx.y * M::tokens;
  const int blocks = blocks_of(p.width), steps = (blocks + 1) / 2, whole = p.width / 64;
  const int part = tid & 7, mine = tid >> 3;                  // what this thread fetches: a part of every 32nd row
  const bool codes_too = kQuarter >= 32 || mine < kQuarter;   // (by whole wavefronts)

  const uint16_t *x_row[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; i++) x_row[i] = p.x + min(token0 + mine + 32 * i, p.tokens - 1) * p.ldx + part * 8;

  struct Step {
    u32x4 x[kLoads], w[kCodes];
    uint8_t s[kCodes];
  };
  auto load_x = [&](Step &t, int step) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) __builtin_memcpy(&t.x[i], x_row[i] + step * 64, 16);
  };
  // Quarter j % 4 of the rows' eight blocks from 8 (j / 4) on; blocks behind the last repeat it.
  auto load_w = [&](Step &t, int j) {
    if (codes_too) {
      const int block = min(8 * (j >> 2) + part, blocks - 1);
#pragma unroll
      for (int i = 0; i < kCodes; i++) {
        const int64_t row = min(row0 + (j & 3) * kQuarter + mine + 32 * i, p.height - 1);
        t.w[i] = *reinterpret_cast<const u32x4 *>(p.codes + (row * blocks + block) * kBlockBytes);
        t.s[i] = p.scales[row * blocks + block];
      }
    }
  };
  auto put_x = [&](const Step &t, int side) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) lds_x[side][(mine + 32 * i) * 8 + (part ^ (mine >> 1 & 7))] = t.x[i];
  };
  auto put_w = [&](const Step &t, int j) {
    if (codes_too) {
      const int side = (j >> 2) & 1;
#pragma unroll
      for (int i = 0; i < kCodes; i++) {
        const int row = (j & 3) * kQuarter + mine + 32 * i;
        lds_w[side][row * 8 + (part ^ (row >> 1 & 7))] = t.w[i];
        // behind the last block nothing: zeros, with whatever scale its repeated codes had
        lds_s[side][row * 8 + part] = 8 * (j >> 2) + part < blocks ? t.s[i] : static_cast<uint8_t>(0);
      }
    }
  };
  f32x16 sum[kRows][kTokens];
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sum[r][n] = f32x16{0};

  auto multiply = [&](int step) {
    const int side = (step >> 2) & 1, block = 2 * (step & 3) + half;
    const u32x4 *from = lds_x[step & 1] + ((wave >> 1) * 32 * kTokens + in_tile) * 8;
    u32x4 w[kRows];
    float scale[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const int row = ((wave & 1) * kRows + r) * 32 + in_tile;
      w[r] = lds_w[side][row * 8 + (block ^ (row >> 1 & 7))];
      scale[r] = scale_of(lds_s[side][row * 8 + block]);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      bf16x8 a[kRows], b[kTokens];
#pragma unroll
      for (int n = 0; n < kTokens; n++)
        b[n] = __builtin_bit_cast(bf16x8, from[n * 32 * 8 + ((4 * half + k) ^ (in_tile >> 1 & 7))]);
#pragma unroll
      for (int r = 0; r < kRows; r++) a[r] = expand8(w[r][k], scale[r]);
#pragma unroll
      for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sum[r][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[r], b[n], sum[r][n], 0, 0, 0);
    }
  };
  // In turn `step` are asked for the activations of step + 2 and quarter step + 5 of the codes, and what was asked
  // for in the turn before goes to LDS behind the products: the activations of step + 1, where nobody has read
  // since the turn before, and quarter step + 4, whose side was last read in the turn before its first quarter.
  // (Behind the last whole step that one is asked for again: a branch's end would wait for what is on its way.)
  auto turn = [&](Step &now, Step &next, int step) {
    load_x(now, min(step + 2, whole - 1));
    load_w(now, step + 5);
    __builtin_amdgcn_sched_barrier(0);   // (asked for here, not where the compiler has them needed)
    multiply(step);
    __builtin_amdgcn_sched_barrier(0);
    put_x(next, (step + 1) & 1);
    put_w(next, step + 4);
    __syncthreads();
  };
  Step even, odd;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    load_w(even, j);
    load_w(odd, j + 1);
    put_w(even, j);
    put_w(odd, j + 1);
  }
  if (whole > 0) {
    load_x(even, 0);
    load_x(odd, min(1, whole - 1));
    load_w(odd, 4);
    put_x(even, 0);
  }
  __syncthreads();
  if (whole > 0) {
    int step = 0;
    for (; step + 2 <= whole; step += 2) {
      turn(even, odd, step);
      turn(odd, even, step + 1);
    }
    if (step < whole) turn(even, odd, step);
  }
  if (whole < steps) {   // the last step, where the row ends inside it: its codes are there
#pragma unroll
    for (int i = 0; i < kLoads; i++)
      lds_x[whole & 1][(mine + 32 * i) * 8 + (part ^ (mine >> 1 & 7))] =
          load8(p.x + min(token0 + mine + 32 * i, p.tokens - 1) * p.ldx, whole * 64 + part * 8, p.width);
    __syncthreads();
    multiply(whole);
  }
  __syncthreads();
  store_tile<kRows, kTokens>(sum, lds, p.y, p.ldy, row0, token0, p.height, p.tokens);
}

// Straight into LDS, three steps of activations and three pairs of steps of codes and scales, each asked for two
// steps or more ahead: no registers hold what is on its way, and a wavefront's turn is its reads of LDS and its
// products (a 128 x 128 tile's turn 0.47 us, through registers 0.67; its MFMAs alone take 0.21).  Nothing is busy all
// the time with two workgroups a compute unit (2272 tokens through 6144 x 2080, by counters: the matrix cores for 39 % of
// the launch, L1 33, LDS 19, VALU 20): the wavefronts meet once a step, and 864 tiles fill a second round of 512 by
// two thirds (4096 x 4096 x 4096 121 us, 1.1 PFLOP/s; of 1.4 that a library product in bf16 reaches at twice that size).
// kParts groups of four wavefronts share a tile's steps, where tiles alone would leave compute units idle.
template <int kRows, int kTokens, int kParts, int kWaves>
__global__ __launch_bounds__(256 * kParts, kWaves) void mx4_many_direct_kernel(const ProductArgs p) {
  using M = Many<kRows, kTokens>;
  constexpr int kLoads = M::tokens / 32;    // fetches of activations, a wavefront and step
  constexpr int kStepBytes = M::tokens * 128, kPairBytes = M::rows * 64, kCodes = 3 * kStepBytes,
                kScaleBytes = M::rows * 16, kScales = kCodes + 3 * kPairBytes,
                kPartBytes = kScales + 3 * kScaleBytes;
  // three steps of activations: a token's eight parts of 16 bytes, part i at i ^ (token / 2 % 8); three pairs of
  // steps of codes: a row's four parts, part i at i ^ (row / 4 % 4); and of scales, 32 bits each
  __shared__ u32x4 all_lds[kParts * kPartBytes / 16];
  const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int which_part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  u32x4 *const lds = all_lds + which_part * (kPartBytes / 16);
  const int half = lane >> 5, in_tile = lane & 31;
  const int row0 = blockIdx.x * M::rows, token0 = blockIdx.y * M::tokens;
  const int blocks = blocks_of(p.width), steps = (blocks + 1) / 2, whole = p.width / 64;

  // the part's steps: as many turns for each part, those behind the last step without products
  const int turns = kParts == 1 ? whole : (whole + 2 * kParts - 1) / (2 * kParts) * 2;
  const int first_step = which_part * turns, my_steps = kParts == 1 ? whole : min(turns, whole - first_step);

  // what this lane fetches, from the tile's first token and row on: a tile's activations span less than 4 GB
  const uint16_t *x_tile = p.x + token0 * p.ldx;
  const uint8_t *code_tile = p.codes + static_cast<int64_t>(row0) * blocks * kBlockBytes;
  const uint8_t *scale_tile = p.scales + static_cast<int64_t>(row0) * blocks;
  uint32_t x_at[kLoads], block_at[kRows];
#pragma unroll
  for (int i = 0; i < kLoads; i++)
    x_at[i] = static_cast<uint32_t>(min((i * 4 + wave) * 8 + (lane >> 3), p.tokens - 1 - token0)) *
                  static_cast<uint32_t>(p.ldx * 2) + ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) * 16;
  const int code_part = (lane & 3) ^ (lane >> 4);
#pragma unroll
  for (int q = 0; q < kRows; q++) block_at[q] = min((q * 4 + wave) * 16 + (lane >> 2), p.height - 1 - row0) * blocks;
  const uint32_t lds_at = lds_address(lds);
  auto fetch_x = [&](int side, int step) {
#pragma unroll
    for (int i = 0; i < kLoads; i++) fetch(x_tile + step * 64, x_at[i], lds_at + side * kStepBytes + (i * 4 + wave) * 1024);
  };
  // 64 rows, those of `q`, of the four blocks from 4 pair on; blocks behind the last repeat it
  auto fetch_w = [&](int side, int pair, int q) {
    fetch(code_tile, (block_at[q] + min(4 * pair + code_part, blocks - 1)) * kBlockBytes,
          lds_at + kCodes + side * kPairBytes + (q * 4 + wave) * 1024);
    fetch_byte(scale_tile, block_at[q] + min(4 * pair + (lane & 3), blocks - 1),
               lds_at + kScales + side * kScaleBytes + (q * 4 + wave) * 256);
  };

  f32x16 sum[kRows][kTokens];
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sum[r][n] = f32x16{0};

  auto multiply = [&](int x_side, int w_side, int q) {
    const u32x4 *x = lds + (x_side * kStepBytes + (wave >> 1) * kTokens * 4096 + in_tile * 128) / 16;
    const u32x4 *codes = lds + (kCodes + w_side * kPairBytes + (wave & 1) * kRows * 2048 + in_tile * 64) / 16;
    const uint32_t *scales = reinterpret_cast<const uint32_t *>(lds) +
                             (kScales + w_side * kScaleBytes + (wave & 1) * kRows * 512 + in_tile * 16) / 4;
    u32x4 w[kRows];
    float scale[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      w[r] = codes[r * 128 + ((2 * q + half) ^ (in_tile >> 2 & 3))];
      scale[r] = scale_of(scales[r * 128 + 2 * q + half]);
    }
    bf16x8 b[2][kTokens];
    auto read = [&](int k) {
#pragma unroll
      for (int n = 0; n < kTokens; n++)
        b[k & 1][n] = __builtin_bit_cast(bf16x8, x[n * 256 + ((4 * half + k) ^ (in_tile >> 1 & 7))]);
    };
    read(0);
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (k < 3) read(k + 1);   // ahead of the products before it, where the compiler would not put it
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 a[kRows];
#pragma unroll
      for (int r = 0; r < kRows; r++) a[r] = expand8(w[r][k], scale[r]);
#pragma unroll
      for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sum[r][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[r], b[k & 1][n], sum[r][n], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Turn `step` asks for the activations of step + 2, whose place was read in the turn before, and for 64 rows'
  // codes of the pair after the next, whose place was read in the pair before; it waits for all that was
  // asked for before the last turn, its own step among it.
  auto turn = [&](auto number, int step) {
    constexpr int kTurn = decltype(number)::value, q = kTurn & 1;
    meet<kLoads + ((q ^ 1) < kRows ? 2 : 0)>();   // but for what the last turn asked for
    if (q < kRows) fetch_w((kTurn / 2 + 2) % 3, ((first_step + step) >> 1) + 2, q);
    fetch_x((kTurn + 2) % 3, min(first_step + step + 2, whole - 1));
    if (kParts == 1 || step < my_steps) multiply(kTurn % 3, kTurn / 2 % 3, q);
  };
#pragma unroll
  for (int q = 0; q < kRows; q++) {
    fetch_w(0, first_step >> 1, q);
    fetch_w(1, (first_step >> 1) + 1, q);
  }
  fetch_x(0, min(first_step, whole - 1));
  fetch_x(1, min(first_step + 1, whole - 1));
  meet<0>();
  int step = 0;
  for (;;) {
    turn(std::integral_constant<int, 0>{}, step);
    if (++step == turns) break;
    turn(std::integral_constant<int, 1>{}, step);
    if (++step == turns) break;
    turn(std::integral_constant<int, 2>{}, step);
    if (++step == turns) break;
    turn(std::integral_constant<int, 3>{}, step);
    if (++step == turns) break;
    turn(std::integral_constant<int, 4>{}, step);
    if (++step == turns) break;
    turn(std::integral_constant<int, 5>{}, step);
    if (++step == turns) break;
  }
  meet<0>();   // nothing is on its way into LDS any more
  if (whole < steps) {   // the last step, where the row ends inside it: its activations go where step 0's were
    const int part = tid & 7, mine = tid >> 3;
    for (int i = 0; i < kLoads; i++)
      lds[(mine + 32 * i) * 8 + (part ^ (mine >> 1 & 7))] =
          load8(p.x + min(token0 + mine + 32 * i, p.tokens - 1) * p.ldx, whole * 64 + part * 8, p.width);
    // and its codes and scales, both blocks, where the first pair's were
    if (tid < M::rows) {
      const int64_t row = min(row0 + tid, p.height - 1) * static_cast<int64_t>(blocks);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const bool there = 2 * whole + i < blocks;
        const int64_t block = row + min(2 * whole + i, blocks - 1);
        lds[(kCodes + tid * 64) / 16 + (i ^ (tid >> 2 & 3))] = *reinterpret_cast<const u32x4 *>(p.codes + block * kBlockBytes);
        reinterpret_cast<uint32_t *>(lds)[(kScales + tid * 16) / 4 + i] = there ? p.scales[block] : 0;
      }
    }
    __syncthreads();
    if (kParts == 1 || which_part == kParts - 1) multiply(0, 0, 0);
  }
  __syncthreads();
  if constexpr (kParts > 1) {   // the parts' sums, added in their order
    f32x4 *sums = reinterpret_cast<f32x4 *>(all_lds);
    constexpr int kFours = 4 * kRows * kTokens;
    if (which_part) {
#pragma unroll
      for (int i = 0; i < kFours; i++) {
        const f32x16 &v = sum[i / 4 / kTokens][i / 4 % kTokens];
        sums[((which_part - 1) * kFours + i) * 256 + tid] =
            f32x4{v[i % 4 * 4], v[i % 4 * 4 + 1], v[i % 4 * 4 + 2], v[i % 4 * 4 + 3]};
      }
    }
    __syncthreads();
    if (which_part == 0) {
#pragma unroll
      for (int other = 0; other < kParts - 1; other++)
#pragma unroll
        for (int i = 0; i < kFours; i++) {
          const f32x4 v = sums[(other * kFours + i) * 256 + tid];
#pragma unroll
          for (int k = 0; k < 4; k++) sum[i / 4 / kTokens][i / 4 % kTokens][i % 4 * 4 + k] += v[k];
        }
    }
    __syncthreads();
  }
  store_tile<kRows, kTokens>(sum, all_lds, p.y, p.ldy, row0, token0, p.height, p.tokens);
}

template <int kRows, int kTokens, int kParts, int kWaves>
void launch_direct(const ProductArgs &p, hipStream_t s) {
  using M = Many<kRows, kTokens>;
  mx4_many_direct_kernel<kRows, kTokens, kParts, kWaves>
      <<<dim3((p.height + M::rows - 1) / M::rows, (p.tokens + M::tokens - 1) / M::tokens), 256 * kParts, 0, s>>>(p);
}

template <int kRows, int kTokens, int kWaves>
void launch_many(const ProductArgs &p, hipStream_t s) {
  using M = Many<kRows, kTokens>;
  mx4_many_kernel<kRows, kTokens, kWaves><<<dim3((p.height + M::rows - 1) / M::rows, (p.tokens + M::tokens - 1) / M::tokens),
                                    256, 0, s>>>(p);
}

struct QuantizedArgs {
  const uint8_t *codes, *scales, *x_codes, *x_scales;
  uint16_t *y;
  int64_t ldy;
  int height, width, tokens;
};

// Both sides in the format, many tokens: kRowSides by kTokenSides wavefronts, each with 32 kRows rows of the matrix and
// 32 kTokens tokens, 128 values of a row a step, as mx4_many_direct_kernel fetches them;
// v_mfma_scale_f32_32x32x64_f8f6f4 takes a lane's block of 32 values as it is, and one byte of a register for its scale.  The scales come through registers, a
// row's eight at a time: of one byte each they would be too many fetches, and of four they do not lie on four.
// That load's wait is the compiler's, which knows nothing of the fetches and waits for all of them, every second step; with
// the scales it costs an eighth of the time (8192 x 8192 x 8192 293 to 302 us, 3.7 of the 8.8 PFLOP/s that the matrix cores
// reach alone; without scales 256).  At 17 steps a tile, 8192 tokens through 6144 x 2080, the matrix cores are busy for 29 %
// of the launch, L1 for 35, LDS for 21: a compute unit holds one workgroup, whose first fetches and last stores
// overlap with nobody's products.
template <int kRows, int kTokens, int kRowSides, int kTokenSides>
__global__ __launch_bounds__(64 * kRowSides * kTokenSides, 2) void mx4_both_kernel(const QuantizedArgs p) {
  constexpr int kBothRows = 32 * kRows * kRowSides, kBothTokens = 32 * kTokens * kTokenSides;
  constexpr int kWaves = kRowSides * kTokenSides, kThreads = 64 * kWaves;
  constexpr int kWFetches = kBothRows / 16 / kWaves, kXFetches = kBothTokens / 16 / kWaves, kScaleRows = kBothRows + kBothTokens;
  constexpr int kStepBytes = (kBothRows + kBothTokens) * 64, kScales = 3 * kStepBytes,
                kScaleBytes = (kBothRows + kBothTokens) * 8;
  // three steps of codes, rows first, then tokens: four parts of 16 bytes, part i at i ^ (row / 4 % 4); two
  // pairs of steps of scales, eight bytes a row
  __shared__ u32x4 lds[(kScales + 2 * kScaleBytes) / 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, in_tile = lane & 31, row_side = wave % kRowSides, token_side = wave / kRowSides;
  const int row0 = blockIdx.x * kBothRows, token0 = blockIdx.y * kBothTokens;
  const int blocks = blocks_of(p.width), steps = (blocks + 3) / 4;
  const uint8_t *code_tile = p.codes + static_cast<int64_t>(row0) * blocks * kBlockBytes;
  const uint8_t *x_tile = p.x_codes + static_cast<int64_t>(token0) * blocks * kBlockBytes;
  const uint32_t lds_at = lds_address(lds);

  // what this lane fetches of a step: 16 rows' 64 bytes a fetch
  const int part = (lane & 3) ^ (lane >> 4);
  uint32_t w_at[kWFetches], x_at[kXFetches];
#pragma unroll
  for (int i = 0; i < kWFetches; i++) w_at[i] = min((i * kWaves + wave) * 16 + (lane >> 2), p.height - 1 - row0) * blocks;
#pragma unroll
  for (int i = 0; i < kXFetches; i++)
    x_at[i] = min((i * kWaves + wave) * 16 + (lane >> 2), p.tokens - 1 - token0) * blocks;
  auto fetch_step = [&](int side, int step) {
    const int block = min(4 * step + part, blocks - 1);
#pragma unroll
    for (int i = 0; i < kWFetches; i++)
      fetch(code_tile, (w_at[i] + block) * kBlockBytes, lds_at + side * kStepBytes + (i * kWaves + wave) * 1024);
#pragma unroll
    for (int i = 0; i < kXFetches; i++)
      fetch(x_tile, (x_at[i] + block) * kBlockBytes, lds_at + side * kStepBytes + kBothRows * 64 + (i * kWaves + wave) * 1024);
  };
  // this thread's row's or token's scales of eight blocks, or of its last eight (the caller's width has as many);
  // threads that are left over repeat the last token
  static_assert(kScaleRows <= kThreads, "a row or token a thread");
  const int scale_row = min(tid, kScaleRows - 1);
  const uint8_t *my_scales =
      scale_row < kBothRows ? p.scales + static_cast<int64_t>(min(row0 + scale_row, p.height - 1)) * blocks
                            : p.x_scales + static_cast<int64_t>(min(token0 + scale_row - kBothRows, p.tokens - 1)) * blocks;
  auto load_scales = [&](int pair) {
    uint64_t eight;
    __builtin_memcpy(&eight, my_scales + min(8 * pair, blocks - 8), 8);
    return eight;
  };
  auto put_scales = [&](int side, int pair, uint64_t eight) {   // zeros behind the last
    reinterpret_cast<uint64_t *>(lds)[(kScales + side * kScaleBytes) / 8 + scale_row] =
        eight >> min(8 * max(8 * pair + 8 - blocks, 0), 63);
  };

  f32x16 sum[kRows][kTokens];
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sum[r][n] = f32x16{0};

  auto multiply = [&](int side, int scale_side, auto which) {
    constexpr int q = decltype(which)::value;   // the step's place in its pair
    const u32x4 *w = lds + (side * kStepBytes + row_side * kRows * 32 * 64 + in_tile * 64) / 16;
    const u32x4 *x = lds + (side * kStepBytes + kBothRows * 64 + token_side * kTokens * 32 * 64 + in_tile * 64) / 16;
    const uint64_t *scales = reinterpret_cast<const uint64_t *>(lds) + (kScales + scale_side * kScaleBytes) / 8 + in_tile;
    uint32_t ws[kRows], xs[kTokens];   // of this half's blocks: bytes 0 and 2
#pragma unroll
    for (int r = 0; r < kRows; r++) ws[r] = static_cast<uint32_t>(scales[(row_side * kRows + r) * 32] >> (32 * q)) >> (8 * half);
#pragma unroll
    for (int n = 0; n < kTokens; n++)
      xs[n] = static_cast<uint32_t>(scales[kBothRows + (token_side * kTokens + n) * 32] >> (32 * q)) >> (8 * half);
    u32x4 a[2][kRows], b[2][kTokens];
    auto read = [&](int k) {
      const int at = (2 * k + half) ^ (in_tile >> 2 & 3);
#pragma unroll
      for (int r = 0; r < kRows; r++) a[k][r] = w[r * 128 + at];
#pragma unroll
      for (int n = 0; n < kTokens; n++) b[k][n] = x[n * 128 + at];
    };
    read(0);
    __builtin_amdgcn_sched_barrier(0);
    read(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
      for (int n = 0; n < kTokens; n++)
        sum[r][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a[0][r]), wide(b[0][n]), sum[r][n], 4, 4, 0,
                                                                    ws[r], 0, xs[n]);
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
      for (int n = 0; n < kTokens; n++)
        sum[r][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(a[1][r]), wide(b[1][n]), sum[r][n], 4, 4, 2,
                                                                    ws[r], 2, xs[n]);
    __builtin_amdgcn_sched_barrier(0);
  };
  uint64_t scales = load_scales(0);
  fetch_step(0, 0);
  fetch_step(1, min(1, steps - 1));
  put_scales(0, 0, scales);
  __syncthreads();
  // Turn `step` asks for step + 2's codes, whose place was read in the turn before, and the first of a pair for the
  // next pair's scales, which the second puts where the pair before had its own.
  auto turn = [&](auto number, int step) {
    constexpr int kTurn = decltype(number)::value, q = kTurn & 1;
    meet<kWFetches + kXFetches>();   // but for the codes that the last turn asked for
    if (q == 0) scales = load_scales((step >> 1) + 1);
    fetch_step((kTurn + 2) % 3, min(step + 2, steps - 1));
    __builtin_amdgcn_sched_barrier(0);
    multiply(kTurn % 3, step >> 1 & 1, std::integral_constant<int, q>{});
    if (q == 1) put_scales(((step >> 1) + 1) & 1, (step >> 1) + 1, scales);
  };
  int step = 0;
  for (;;) {
    turn(std::integral_constant<int, 0>{}, step);
    if (++step == steps) break;
    turn(std::integral_constant<int, 1>{}, step);
    if (++step == steps) break;
    turn(std::integral_constant<int, 2>{}, step);
    if (++step == steps) break;
    turn(std::integral_constant<int, 3>{}, step);
    if (++step == steps) break;
    turn(std::integral_constant<int, 4>{}, step);
    if (++step == steps) break;
    turn(std::integral_constant<int, 5>{}, step);
    if (++step == steps) break;
  }
  meet<0>();   // nothing is on its way into LDS any more
  // to y past LDS, half of the tokens at a time
  uint16_t *out = reinterpret_cast<uint16_t *>(lds);
  constexpr int kPitch = kBothRows + 8, kPieces = kBothRows / 8, kAtOnce = kThreads / kPieces, kHalf = kBothTokens / 2;
  static_assert(kHalf * kPitch * 2 <= sizeof(lds), "the tile has room");
#pragma unroll
  for (int side = 0; side < 2; side++) {
    if (token_side / (kTokenSides / 2) == side) {
#pragma unroll
      for (int n = 0; n < kTokens; n++)
#pragma unroll
        for (int r = 0; r < kRows; r++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t two[2] = {two_bf16(sum[r][n][4 * i], sum[r][n][4 * i + 1]),
                                     two_bf16(sum[r][n][4 * i + 2], sum[r][n][4 * i + 3])};
            __builtin_memcpy(__builtin_assume_aligned(out + ((token_side % (kTokenSides / 2) * kTokens + n) * 32 + in_tile) * kPitch +
                                                          (row_side * kRows + r) * 32 + 8 * i + 4 * half, 8),
                             two, 8);
          }
    }
    __syncthreads();
    const int row = tid % kPieces * 8, rows_left = p.height - row0 - row, token = tid / kPieces;
    const int tokens_left = p.tokens - token0 - kHalf * side - token;
    const uint16_t *from = out + token * kPitch + row;
    uint16_t *to = p.y + static_cast<int64_t>(token0 + kHalf * side + token) * p.ldy + row0 + row;
    if (rows_left >= 8) {
#pragma unroll 4
      for (int i = 0; i < kHalf / kAtOnce; i++) {
        u32x4 v;
        __builtin_memcpy(&v, __builtin_assume_aligned(from + i * kAtOnce * kPitch, 16), 16);
        if (i * kAtOnce < tokens_left) __builtin_memcpy(to + i * kAtOnce * p.ldy, &v, 16);
      }
    } else if (rows_left > 0) {
      for (int i = 0; i * kAtOnce < min(kHalf, tokens_left); i++)
        for (int k = 0; k < rows_left; k++) to[i * kAtOnce * p.ldy + k] = from[i * kAtOnce * kPitch + k];
    }
    __syncthreads();
  }
}

template <int kRows, int kTokens, int kRowSides, int kTokenSides>
void launch_both_tiles(const QuantizedArgs &p, hipStream_t s) {
  constexpr int kBothRows = 32 * kRows * kRowSides, kBothTokens = 32 * kTokens * kTokenSides;
  mx4_both_kernel<kRows, kTokens, kRowSides, kTokenSides>
      <<<dim3((p.height + kBothRows - 1) / kBothRows, (p.tokens + kBothTokens - 1) / kBothTokens),
         64 * kRowSides * kTokenSides, 0, s>>>(p);
}

// Few tokens of both sides: eight wavefronts a workgroup take eight blocks of its rows and tokens in turn, and
// v_mfma_scale_f32_16x16x128_f8f6f4 a lane's block of a row and of a token as they are.  Eight lanes read a row's
// whole line and hand the blocks round through LDS, a part of the wavefront's own: the lanes that multiply are 16 rows
// apart, and their own loads would be pieces of 16 bytes, one by one in the L1 (61 tokens through 2080 x 6144 12.8 us
// with blocks four at a time and a byte of scale each, 9.3 with eight and eight bytes, through LDS 6.0).
// The next blocks are on their way meanwhile.  What bounds it: three turns' trips to memory, and a launch.
template <int kRows, int kTokens>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_both_few_kernel(const QuantizedArgs p) {
  constexpr int kSides = kRows + kTokens;   // 16 rows or tokens of eight blocks each: 2 KB
  __shared__ u32x4 lds[kFewWaves * kSides * 128];
  static_assert(kSides * 128 * kFewWaves >= kFewLds<kRows, kTokens>, "the sums take the place of the codes");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4;
  const int row0 = blockIdx.x * 16 * kRows, token0 = blockIdx.y * 16 * kTokens;
  const int blocks = blocks_of(p.width), units = (blocks + 7) / 8;
  u32x4 *const mine = lds + wave * kSides * 128;
  const uint8_t *codes[2] = {p.codes + static_cast<int64_t>(row0) * blocks * kBlockBytes,
                             p.x_codes + static_cast<int64_t>(token0) * blocks * kBlockBytes};
  const uint8_t *scales[2] = {p.scales + static_cast<int64_t>(row0) * blocks, p.x_scales + static_cast<int64_t>(token0) * blocks};
  const int last[2] = {p.height - 1 - row0, p.tokens - 1 - token0};
  uint32_t first[kSides][2], scale_first[kSides];
#pragma unroll
  for (int i = 0; i < kSides; i++) {
    const int side = i >= kRows, at = 16 * (side ? i - kRows : i);
#pragma unroll
    for (int h = 0; h < 2; h++) first[i][h] = min(at + 8 * h + (lane >> 3), last[side]) * blocks;
    scale_first[i] = min(at + (lane & 15), last[side]) * blocks;
  }
  FewSums<kRows, kTokens> sums;
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sums.of[r][n] = f32x4{0, 0, 0, 0};

  u32x4 next[kSides][2];
  uint64_t next_scales[kSides];
  auto scales_from = [&](int unit) { return max(min(8 * unit, blocks - 8), 0); };
  auto fetch_unit = [&](int unit) {
    const int block = min(8 * unit + (lane & 7), blocks - 1);
#pragma unroll
    for (int i = 0; i < kSides; i++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        next[i][h] = *reinterpret_cast<const u32x4 *>(codes[i >= kRows] + (first[i][h] + block) * kBlockBytes);
#pragma unroll
    for (int i = 0; i < kSides; i++) {
      const uint8_t *from = scales[i >= kRows] + scale_first[i];
      if (blocks >= 8) {
        __builtin_memcpy(&next_scales[i], from + scales_from(unit), 8);
      } else {
        const int one = min(group, blocks - 1), two = min(4 + group, blocks - 1);
        next_scales[i] = static_cast<uint64_t>(from[one]) << (8 * one) | static_cast<uint64_t>(from[two]) << (8 * two);
      }
    }
  };
  if (wave < units) fetch_unit(wave);
  for (int unit = wave; unit < units; unit += kFewWaves) {
    uint64_t now[kSides];
#pragma unroll
    for (int i = 0; i < kSides; i++) {
      now[i] = next_scales[i];
#pragma unroll
      for (int h = 0; h < 2; h++) mine[i * 128 + h * 64 + (lane & 56) + ((lane & 7) ^ (lane >> 3))] = next[i][h];
    }
    if (unit + kFewWaves < units) fetch_unit(unit + kFewWaves);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int from = scales_from(unit);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int block = 8 * unit + 4 * i + group;
      const bool there = block < blocks;   // behind the last block: its codes, under scales that make them nothing
      const int by = 8 * (min(block, blocks - 1) - from);
      u32x4 v[kSides];
      int s[kSides];
#pragma unroll
      for (int j = 0; j < kSides; j++) {
        v[j] = mine[j * 128 + (lane & 15) * 8 + ((4 * i + group) ^ (lane & 7))];
        s[j] = there ? static_cast<int>(now[j] >> by) & 255 : 0;
      }
#pragma unroll
      for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sums.of[r][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(v[r]), wide(v[kRows + n]), sums.of[r][n], 4, 4, 0,
                                                                           s[r], 0, s[kRows + n]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  few_join<kRows, kTokens>(sums, reinterpret_cast<f32x4 *>(lds), [&](int r, int n, f32x4 sum) {
    const int t = token0 + 16 * n + (lane & 15);
    if (t < p.tokens) store_four(p.y + t * p.ldy, row0 + 16 * r + 4 * group, p.height, sum);
  });
}

template <int kRows, int kTokens>
void launch_both_few(const QuantizedArgs &p, hipStream_t s) {
  const dim3 grid((p.height + 16 * kRows - 1) / (16 * kRows), (p.tokens + 16 * kTokens - 1) / (16 * kTokens));
  mx4_both_few_kernel<kRows, kTokens><<<grid, 64 * kFewWaves, 0, s>>>(p);
}

// Which kernel (us, measured as below): wavefronts that take rows and all their blocks, in the smallest tiles that are no
// more than the compute units (2080 x 6144: 61 tokens by 16 x 16, 16 x 32, 32 x 32, 32 x 64 7.3, 6.9, 6.0, 7.9, and
// through LDS 12; 32 tokens 5.2, 5.0, 5.8, 7.8; 192 tokens 14.0, 12.8, 12.3, 8.6 and 12.5; 6144 x 2080: 61 tokens
// 7.7, 6.9, 7.0, 5.8; 128 tokens, 384 of the largest, 10.2 and 6.8; 64 tokens through 1024 x 4096 3.9, 4.7, 5.5, 7.3).
// Beyond that tiles of 128 x 64 through LDS, to one
// a compute unit (568 through 2080 x 6144, 153 of them: 20.1, of 128 x 128 23.8), of 128 x 128 (1136 through 2080 x
// 6144, 306 small ones: 25.6, small 30.9), and of 256 x 256 where they are enough (2272 through 6144 x 2080, 216
// of them: 25.6, of 128 x 128 35.5; 1136, 120: 20.7 and 19.1); not for up to 64 tokens or rows of less than a step.
void launch_both(const QuantizedArgs &p, hipStream_t s) {
  auto tiles = [&](int rows, int tokens) {
    return static_cast<int64_t>((p.height + rows - 1) / rows) * ((p.tokens + tokens - 1) / tokens);
  };
  const int64_t small_tiles = tiles(128, 64), large_tiles = tiles(256, 256);
  if (p.tokens <= 64 || tiles(32, 64) <= 256 || blocks_of(p.width) < 8) {
    sub1::note_kernel("mx4_both_few_kernel");
    if (p.tokens <= 16 || tiles(16, 16) <= 256)
      launch_both_few<1, 1>(p, s);
    else if (tiles(16, 32) <= 256)
      launch_both_few<1, 2>(p, s);
    else if (tiles(32, 32) <= 256)
      launch_both_few<2, 2>(p, s);
    else
      launch_both_few<2, 4>(p, s);
  } else if (small_tiles <= 256) {
    sub1::note_kernel("mx4_both_kernel<2, 1>");
    launch_both_tiles<2, 1, 2, 2>(p, s);
  } else if (large_tiles < 180) {
    sub1::note_kernel("mx4_both_kernel<2, 2>");
    launch_both_tiles<2, 2, 2, 2>(p, s);
  } else {
    sub1::note_kernel("mx4_both_kernel<4, 2>");
    launch_both_tiles<4, 2, 2, 4>(p, s);
  }
}

template <int kRows, int kTokens>
dim3 few_grid(const ProductArgs &p) {
  return dim3((p.height + 16 * kRows - 1) / (16 * kRows), (p.tokens + 16 * kTokens - 1) / (16 * kTokens));
}
template <int kRows, int kTokens>
void launch_few(const ProductArgs &p, hipStream_t s) {
  sub1::note_kernel("mx4_few_kernel");
  mx4_few_kernel<kRows, kTokens><<<few_grid<kRows, kTokens>(p), 64 * kFewWaves, 0, s>>>(p);
}
template <int kRows, int kTokens>
void launch_few_lines(const ProductArgs &p, hipStream_t s) {
  sub1::note_kernel("mx4_few_lines_kernel");
  mx4_few_lines_kernel<kRows, kTokens><<<few_grid<kRows, kTokens>(p), 64 * kFewWaves, 0, s>>>(p);
}

// Which kernel, by what was measured on matrices of 500 x 500 to 6144 x 2080 (us, one after the other in a graph):
// a token alone by whole rows.  Up to 32 tokens, and more where tiles of 32 x 16 are no more than the compute units,
// wavefronts that take rows and all their values: with pieces handed round through LDS (13 tokens through 2080 x 6144
// 7.7 us, without 8.9; 32 through 1024 x 4096 6.0 and 10.8; 13 through 3001 x 1023 4.3 and 5.2; 16 rows a workgroup to
// one a compute unit, then 32: 48 tokens through 2080 x 6144 11.7 and 10.5, through tiles shared as below 13.3), but
// not in rows of less than a step a wavefront (5 through 768 x 768 3.1, without 2.7) nor for 17 to 32 tokens and
// rows enough for two tiles each way (32 through 6144 x 2080 7.4 and 6.6).  Then tiles of 64 x 64, as there are few of
// them shared by four, two or one group of four wavefronts (70 through 2080 x 6144, 66 tiles: 13.7, 15.7, 20.5; 200
// through 4096 x 1024, 256 tiles: 5.9, 5.5, 5.9; 568, 576 tiles: 14.3, 10.9, 8.9), and of 128 x 128 from four
// of the small ones a compute unit on (2272 through 6144 x 2080, 3456 tiles: 65, small ones 90; 1136, 1728: 34 and 47).
// Activations whose rows do not lie on 16 bytes cannot be fetched into LDS without registers
// (2272 through 6144 x 2080 77, 568 through 4096 x 1024 12.3), by tiles that no groups share: wavefronts that take rows
// then pay to three tiles of 32 x 16 a compute unit (200 through 2080 x 6143, 845: 37 us, through registers 57; 50
// through 6144 x 2079, 768: 13.4 and 15.3; 100 through 3756 x 1036, 826: 10.0 and 9.5; 400 through 2080 x 6143, 1625:
// 68 and 58).
int launch_product(const ProductArgs &p, hipStream_t s) {
  auto tiles = [&](int rows, int tokens) {
    return static_cast<int64_t>((p.height + rows - 1) / rows) * ((p.tokens + tokens - 1) / tokens);
  };
  const int64_t small_tiles = tiles(64, 64);
  const bool in_lines = !misaligned(p.x, 16) && p.ldx % 8 == 0 && p.ldx < 1 << 23;   // fetch() takes them
  if (p.tokens == 1) {
    sub1::note_kernel("mx4_one_kernel");
    return halves_pay(p.width, p.height) ? launch_one<32>(p, s) : launch_one<64>(p, s);
  } else if (p.tokens <= 32 || p.width < 64 || tiles(32, 16) <= (in_lines ? 256 : 768)) {
    const int64_t rows = tiles(16, 1 << 20);
    if (p.width < 64 || (p.tokens > 16 && p.tokens <= 32 && rows > 256))
      launch_few<2, 2>(p, s);
    else if (p.tokens <= 16 && blocks_of(p.width) < 32)
      launch_few<1, 1>(p, s);
    else if (p.tokens <= 16 || tiles(16, 16) <= 256)
      launch_few_lines<1, 1>(p, s);
    else
      launch_few_lines<2, 1>(p, s);
  } else if (!in_lines) {
    sub1::note_kernel("mx4_many_kernel");
    if (small_tiles < 1024)
      launch_many<1, 1, 4>(p, s);
    else
      launch_many<2, 2, 2>(p, s);
  } else {
    sub1::note_kernel("mx4_many_direct_kernel");
    if (small_tiles <= 96)
      launch_direct<1, 1, 4, 4>(p, s);
    else if (small_tiles <= 320)
      launch_direct<1, 1, 2, 4>(p, s);
    else if (small_tiles < 1024)
      launch_direct<1, 1, 1, 4>(p, s);
    else
      launch_direct<2, 2, 1, 2>(p, s);
  }
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// ------------------------------------------------------------------- launching ---

constexpr int kTypes = 3;
constexpr int64_t kTypeBytes[kTypes] = {2, 2, 4};

int check_values(const char *who, const void *x, const void *codes, const void *scales, int type, int64_t rows,
                 int width, int64_t ld) {
  if (type < 0 || type >= kTypes) return fail(SUB1_ERR_SHAPE, "%s: type %d (SUB1_MX4_BF16, _FP16 or _FP32)", who, type);
  if (rows < 0 || width < 1 || width > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "%s: %lld rows of width %d (1..%d)", who, static_cast<long long>(rows), width,
                SUB1_MX4_MAX_WIDTH);
  if (rows == 0) return SUB1_OK;
  if (!x || !codes || !scales) return fail(SUB1_ERR_NULL, "%s: NULL argument", who);
  if (rows > 1 && ld < width) return fail(SUB1_ERR_SHAPE, "%s: row stride smaller than the rows", who);
  if (misaligned(x, kTypeBytes[type]) || misaligned(codes, 16)) return fail(SUB1_ERR_ALIGN, "%s: misaligned pointer", who);
  return SUB1_OK;
}

// Rows in parts whose threads a 32-bit count holds: launch(first row, rows, workgroups).
template <class Launch>
int in_parts(int64_t rows, int width, Launch launch) {
  const int64_t threads = 4 * static_cast<int64_t>(blocks_of(width)), most = (int64_t{1} << 31) / threads;
  for (int64_t first = 0; first < rows; first += most) {
    const int64_t n = rows - first < most ? rows - first : most;
    launch(first, static_cast<uint32_t>(n), static_cast<unsigned>((n * threads + 255) / 256));
    HIP_TRY(hipGetLastError());
  }
  return SUB1_OK;
}

int check_product(const char *who, const void *codes, const void *scales, int height, int width, const void *x,
                  int64_t ldx, const void *y, int64_t ldy, int tokens) {
  if (tokens < 0 || tokens > SUB1_MX4_MAX_TOKENS)
    return fail(SUB1_ERR_SHAPE, "%s: tokens %d outside 0..%d", who, tokens, SUB1_MX4_MAX_TOKENS);
  if (height < 1 || width < 1 || width > SUB1_MX4_MAX_WIDTH || height > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "%s: height %d width %d (1..%d)", who, height, width, SUB1_MX4_MAX_WIDTH);
  if (tokens == 0) return SUB1_OK;
  if (!codes || !scales || !x || !y) return fail(SUB1_ERR_NULL, "%s: NULL argument", who);
  if (tokens > 1 && (ldx < width || ldy < height))
    return fail(SUB1_ERR_SHAPE, "%s: row strides smaller than the rows", who);
  if (misaligned(codes, 16) || misaligned(y, 2)) return fail(SUB1_ERR_ALIGN, "%s: misaligned pointer", who);
  return SUB1_OK;
}

}  // namespace

// ================================================================ C ABI =====

extern "C" int sub1_mx4_quantize(const void *x, int type, int64_t ldx, int64_t rows, int width, uint8_t *codes,
                                 uint8_t *scales, void *stream) {
  const int rc = check_values("sub1_mx4_quantize", x, codes, scales, type, rows, width, ldx);
  if (rc || rows == 0) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = ldx * kTypeBytes[type], blocks = blocks_of(width);
  return in_parts(rows, width, [&](int64_t first, uint32_t n, unsigned grid) {
    const uint8_t *from = static_cast<const uint8_t *>(x) + first * row_bytes;
    uint8_t *c = codes + first * blocks * kBlockBytes, *sc = scales + first * blocks;
    if (type == SUB1_MX4_BF16)
      mx4_quantize_kernel<__bf16><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
    else if (type == SUB1_MX4_FP16)
      mx4_quantize_kernel<_Float16><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
    else
      mx4_quantize_kernel<float><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
  });
}

extern "C" int sub1_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int width, void *out,
                                   int type, int64_t ldo, void *stream) {
  const int rc = check_values("sub1_mx4_dequantize", out, codes, scales, type, rows, width, ldo);
  if (rc || rows == 0) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = ldo * kTypeBytes[type], blocks = blocks_of(width);
  return in_parts(rows, width, [&](int64_t first, uint32_t n, unsigned grid) {
    uint8_t *to = static_cast<uint8_t *>(out) + first * row_bytes;
    const uint8_t *c = codes + first * blocks * kBlockBytes, *sc = scales + first * blocks;
    if (type == SUB1_MX4_BF16)
      mx4_dequantize_kernel<__bf16><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
    else if (type == SUB1_MX4_FP16)
      mx4_dequantize_kernel<_Float16><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
    else
      mx4_dequantize_kernel<float><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
  });
}

extern "C" int sub1_mx4_product(const uint8_t *codes, const uint8_t *scales, int height, int width, const void *x,
                                int64_t ldx, void *y, int64_t ldy, int tokens, void *stream) {
  const int rc = check_product("sub1_mx4_product", codes, scales, height, width, x, ldx, y, ldy, tokens);
  if (rc || tokens == 0) return rc;
  if (misaligned(x, 2)) return fail(SUB1_ERR_ALIGN, "sub1_mx4_product: misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const ProductArgs p{codes, scales, static_cast<const uint16_t *>(x), static_cast<uint16_t *>(y), ldx, ldy, height,
                      width, tokens};
  return launch_product(p, s);
}

extern "C" int sub1_mx4_product_quantized(const uint8_t *codes, const uint8_t *scales, int height, int width,
                                          const uint8_t *x_codes, const uint8_t *x_scales, void *y, int64_t ldy,
                                          int tokens, void *stream) {
  const int rc = check_product("sub1_mx4_product_quantized", codes, scales, height, width, x_codes, width, y, ldy, tokens);
  if (rc || tokens == 0) return rc;
  if (!x_scales) return fail(SUB1_ERR_NULL, "sub1_mx4_product_quantized: NULL argument");
  if (misaligned(x_codes, 16)) return fail(SUB1_ERR_ALIGN, "sub1_mx4_product_quantized: misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const QuantizedArgs p{codes, scales, x_codes, x_scales, static_cast<uint16_t *>(y), ldy, height, width, tokens};
  launch_both(p, s);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}
