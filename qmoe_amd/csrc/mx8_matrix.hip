// Activations in microscaled 8 bits: values to the format and back, and their products with matrices
// in microscaled 4 bits.
#include "mx8.h"

using namespace mx8;
using mx4::bf16x2;
using mx4::bf16x8;
using mx4::Eight;
using mx4::f32x4;
using mx4::FewSums;
using mx4::i32x8;
using mx4::kBlockBytes;
using mx4::kFewWaves;
using sub1::fail;
using sub1::misaligned;

namespace {

// ------------------------------------------------------- to the format and back ---

// Four lanes a block, eight values a lane.
template <class T>
__global__ __launch_bounds__(256) void mx8_quantize_kernel(const uint8_t *__restrict__ x, int64_t row_bytes, uint32_t rows,
                                                           int width, uint8_t *__restrict__ codes,
                                                           uint8_t *__restrict__ scales) {
  const uint32_t blocks = blocks_of(width);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, block = at >> 2;   // the caller's rows * blocks * 4 fit
  if (block >= rows * blocks) return;                                    // (all four lanes of a block)
  const uint32_t row = block / blocks;
  Eight<T> e;
  e.load(x + row * row_bytes, static_cast<int>(block - row * blocks) * kBlock + static_cast<int>(at & 3) * 8, width);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = e.at(i);
  store_block(v, codes, scales, at, true);
}

template <class T>
__global__ __launch_bounds__(256) void mx8_dequantize_kernel(const uint8_t *__restrict__ codes,
                                                             const uint8_t *__restrict__ scales, uint32_t rows, int width,
                                                             uint8_t *__restrict__ out, int64_t row_bytes) {
  const uint32_t blocks = blocks_of(width);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x, block = at >> 2;
  if (block >= rows * blocks) return;
  const uint32_t row = block / blocks;
  const u32x2 packed = reinterpret_cast<const u32x2 *>(codes)[at];
  const float scale = mx4::scale_of(scales[block]);
  float v[8];
  unpack4(packed[0], scale, v);
  unpack4(packed[1], scale, v + 4);
  round8<T>(out + row * row_bytes, static_cast<int>(block - row * blocks) * kBlock + static_cast<int>(at & 3) * 8, width, v);
}

// ------------------------------------------------------------------- products ---

struct Product8Args {
  const uint8_t *codes, *scales, *x_codes, *x_scales;
  uint16_t *y;
  uint8_t *y_codes, *y_scales;   // in place of y
  int64_t ldy;
  int height, width, tokens, relu;
};

__device__ __forceinline__ float bent(float v, int relu) { return relu && v < 0 ? 0.0f : v; }   // (what is no number stays so)

// An operand of the scaled MFMAs: 16 bytes in 4 bits, or 32 bytes in 8 bits.
__device__ __forceinline__ i32x8 operand(u32x4 a, u32x4 b) {
  return i32x8{static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]),
               static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3])};
}

// Few tokens: eight wavefronts a workgroup take eight blocks of its rows and tokens in turn; whole lines are read and the
// blocks handed round through LDS, a part of the wavefront's own, the next ones on their way meanwhile.
// v_mfma_scale_f32_16x16x128_f8f6f4 takes lane l's block l / 16 of row l % 16 as it is; of token l % 16 it takes in
// lane l the 16 values from 16 (l / 16) on and the 16 from 64 + 16 (l / 16) on, but its scale for block l / 16.
template <int kRows, int kTokens>
__global__ __launch_bounds__(64 * kFewWaves) void mx8_few_kernel(const Product8Args p) {
  constexpr int kStage = kRows * 128 + kTokens * 256;   // of 16 bytes: 16 rows of 128, 16 tokens of 256
  __shared__ u32x4 lds[kFewWaves * kStage];
  static_assert(kStage * kFewWaves >= mx4::kFewLds<kRows, kTokens>, "the sums take the place of the codes");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4;
  const int row0 = blockIdx.x * 16 * kRows, token0 = blockIdx.y * 16 * kTokens;
  const int blocks = blocks_of(p.width), units = (blocks + 7) / 8;
  u32x4 *const w_lds = lds + wave * kStage, *const x_lds = w_lds + kRows * 128;
  const uint8_t *codes = p.codes + static_cast<int64_t>(row0) * blocks * kBlockBytes;
  const uint8_t *x_codes = p.x_codes + static_cast<int64_t>(token0) * blocks * kBlock;
  const uint8_t *scales = p.scales + static_cast<int64_t>(row0) * blocks, *x_scales = p.x_scales + static_cast<int64_t>(token0) * blocks;
  const int last_row = p.height - 1 - row0, last_token = p.tokens - 1 - token0;
  // rows and tokens that are not there repeat the last
  uint32_t w_first[kRows][2], x_first[kTokens][4], ws_first[kRows], xs_first[kTokens];
#pragma unroll
  for (int r = 0; r < kRows; r++) {
#pragma unroll
    for (int h = 0; h < 2; h++) w_first[r][h] = min(16 * r + 8 * h + (lane >> 3), last_row) * blocks;
    ws_first[r] = min(16 * r + (lane & 15), last_row) * blocks;
  }
#pragma unroll
  for (int n = 0; n < kTokens; n++) {
#pragma unroll
    for (int h = 0; h < 4; h++) x_first[n][h] = min(16 * n + 4 * h + group, last_token) * blocks;
    xs_first[n] = min(16 * n + (lane & 15), last_token) * blocks;
  }
  FewSums<kRows, kTokens> sums;
#pragma unroll
  for (int r = 0; r < kRows; r++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sums.of[r][n] = f32x4{0, 0, 0, 0};

  u32x4 next_w[kRows][2], next_x[kTokens][4];
  uint64_t next_ws[kRows], next_xs[kTokens];
  const auto scales_from = [&](int unit) { return max(min(8 * unit, blocks - 8), 0); };
  auto eight_scales = [&](const uint8_t *from, int unit) -> uint64_t {
    uint64_t eight;
    if (blocks >= 8) {
      __builtin_memcpy(&eight, from + scales_from(unit), 8);
    } else {
      const int one = min(group, blocks - 1), two = min(4 + group, blocks - 1);
      eight = static_cast<uint64_t>(from[one]) << (8 * one) | static_cast<uint64_t>(from[two]) << (8 * two);
    }
    return eight;
  };
  auto fetch_unit = [&](int unit) {
    const int block = min(8 * unit + (lane & 7), blocks - 1), x_block = min(8 * unit + (lane >> 1 & 7), blocks - 1);
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
      for (int h = 0; h < 2; h++)
        next_w[r][h] = *reinterpret_cast<const u32x4 *>(codes + (w_first[r][h] + block) * kBlockBytes);
#pragma unroll
    for (int n = 0; n < kTokens; n++)
#pragma unroll
      for (int h = 0; h < 4; h++)
        next_x[n][h] = *reinterpret_cast<const u32x4 *>(x_codes + (x_first[n][h] + x_block) * kBlock + 16 * (lane & 1));
#pragma unroll
    for (int r = 0; r < kRows; r++) next_ws[r] = eight_scales(scales + ws_first[r], unit);
#pragma unroll
    for (int n = 0; n < kTokens; n++) next_xs[n] = eight_scales(x_scales + xs_first[n], unit);
  };
  if (wave < units) fetch_unit(wave);
  for (int unit = wave; unit < units; unit += kFewWaves) {
    uint64_t now_ws[kRows], now_xs[kTokens];
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      now_ws[r] = next_ws[r];
#pragma unroll
      for (int h = 0; h < 2; h++) w_lds[r * 128 + h * 64 + (lane & 56) + ((lane & 7) ^ (lane >> 3))] = next_w[r][h];
    }
#pragma unroll
    for (int n = 0; n < kTokens; n++) {
      now_xs[n] = next_xs[n];
#pragma unroll
      for (int h = 0; h < 4; h++) {
        const int i = 4 * h + group;   // its token
        x_lds[n * 256 + 16 * i + ((lane & 15) ^ i)] = next_x[n][h];
      }
    }
    if (unit + kFewWaves < units) fetch_unit(unit + kFewWaves);
    sub1::wave_lds_fence();
    const int from = scales_from(unit);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int block = 8 * unit + 4 * i + group;
      const bool there = block < blocks;   // behind the last block: its codes, under scales that make them nothing
      const int by = 8 * (min(block, blocks - 1) - from);
      i32x8 a[kRows], b[kTokens];
      int as[kRows], bs[kTokens];
#pragma unroll
      for (int r = 0; r < kRows; r++) {
        a[r] = mx4::wide(w_lds[r * 128 + (lane & 15) * 8 + ((4 * i + group) ^ (lane & 7))]);
        as[r] = there ? static_cast<int>(now_ws[r] >> by) & 255 : 0;
      }
#pragma unroll
      for (int n = 0; n < kTokens; n++) {
        const u32x4 *token = x_lds + n * 256 + 16 * (lane & 15);
        b[n] = operand(token[(8 * i + group) ^ (lane & 15)], token[(8 * i + 4 + group) ^ (lane & 15)]);
        bs[n] = there ? static_cast<int>(now_xs[n] >> by) & 255 : 0;
      }
#pragma unroll
      for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sums.of[r][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[r], b[n], sums.of[r][n], 4, 0, 0, as[r], 0, bs[n]);
    }
    sub1::wave_lds_fence();
  }
  __syncthreads();
  if (!p.y_codes) {
    mx4::few_join<kRows, kTokens>(sums, reinterpret_cast<f32x4 *>(lds), [&](int r, int n, f32x4 sum) {
      const int t = token0 + 16 * n + (lane & 15);
#pragma unroll
      for (int k = 0; k < 4; k++) sum[k] = bent(sum[k], p.relu);
      if (t < p.tokens) mx4::store_four(p.y + t * p.ldy, row0 + 16 * r + 4 * group, p.height, sum);
    });
  } else if constexpr (kRows == 2) {   // both tiles of a token's 32 rows are a block
    f32x4 *const all = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int n = 0; n < kTokens; n++) all[(wave * 2 * kTokens + r * kTokens + n) * 64 + lane] = sums.of[r][n];
    __syncthreads();
    for (int n = wave; n < kTokens; n += kFewWaves) {
      float v[8];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        f32x4 sum = all[(r * kTokens + n) * 64 + lane];
        for (int other = 1; other < kFewWaves; other++) sum += all[((other * 2 + r) * kTokens + n) * 64 + lane];
#pragma unroll
        for (int k = 0; k < 4; k++) v[4 * r + k] = row0 + 16 * r + 4 * group + k < p.height ? bent(sum[k], p.relu) : 0.0f;
      }
      uint32_t largest = largest_of(v);
      largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 16)));
      largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 32)));
      const uint32_t byte = scale_byte(largest);
      const u32x2 packed = pack8(v, byte);
      const int t = token0 + 16 * n + (lane & 15);
      if (t < p.tokens) {
        const int64_t block = static_cast<int64_t>(t) * blocks_of(p.height) + blockIdx.x;
        reinterpret_cast<uint32_t *>(p.y_codes + block * kBlock)[group] = packed[0];
        reinterpret_cast<uint32_t *>(p.y_codes + block * kBlock)[4 + group] = packed[1];
        if (group == 0) p.y_scales[block] = static_cast<uint8_t>(byte);
      }
    }
  }
}

template <int kRows, int kTokens>
void launch_few(const Product8Args &p, hipStream_t s) {
  const dim3 grid((p.height + 16 * kRows - 1) / (16 * kRows), (p.tokens + 16 * kTokens - 1) / (16 * kTokens));
  mx8_few_kernel<kRows, kTokens><<<grid, 64 * kFewWaves, 0, s>>>(p);
}

int launch_product(const Product8Args &p, hipStream_t s) {
  sub1::note_kernel("mx8_few_kernel");
  if (p.tokens <= 16)
    launch_few<2, 1>(p, s);
  else
    launch_few<2, 2>(p, s);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// ------------------------------------------------------------------- launching ---

int check_values(const char *who, const void *x, const void *codes, const void *scales, int type, int64_t rows, int width,
                 int64_t ld) {
  if (type < 0 || type >= kTypes) return fail(SUB1_ERR_SHAPE, "%s: type %d (SUB1_MX4_BF16, _FP16 or _FP32)", who, type);
  if (rows < 0 || width < 1 || width > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "%s: %lld rows of width %d (1..%d)", who, static_cast<long long>(rows), width, SUB1_MX4_MAX_WIDTH);
  if (rows == 0) return SUB1_OK;
  if (!x || !codes || !scales) return fail(SUB1_ERR_NULL, "%s: NULL argument", who);
  if (rows > 1 && ld < width) return fail(SUB1_ERR_SHAPE, "%s: row stride smaller than the rows", who);
  if (misaligned(x, kTypeBytes[type]) || misaligned(codes, 16)) return fail(SUB1_ERR_ALIGN, "%s: misaligned pointer", who);
  return SUB1_OK;
}

// Rows in parts of at most 2^31 threads: launch(first row, rows, workgroups).
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

}  // namespace

// ================================================================ C ABI =====

extern "C" int sub1_mx8_quantize(const void *x, int type, int64_t ldx, int64_t rows, int width, uint8_t *codes, uint8_t *scales,
                                 void *stream) {
  const int rc = check_values("sub1_mx8_quantize", x, codes, scales, type, rows, width, ldx);
  if (rc || rows == 0) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = ldx * kTypeBytes[type], blocks = blocks_of(width);
  return in_parts(rows, width, [&](int64_t first, uint32_t n, unsigned grid) {
    const uint8_t *from = static_cast<const uint8_t *>(x) + first * row_bytes;
    uint8_t *c = codes + first * blocks * kBlock, *sc = scales + first * blocks;
    if (type == SUB1_MX4_BF16)
      mx8_quantize_kernel<__bf16><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
    else if (type == SUB1_MX4_FP16)
      mx8_quantize_kernel<_Float16><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
    else
      mx8_quantize_kernel<float><<<grid, 256, 0, s>>>(from, row_bytes, n, width, c, sc);
  });
}

extern "C" int sub1_mx8_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t rows, int width, void *out, int type,
                                   int64_t ldo, void *stream) {
  const int rc = check_values("sub1_mx8_dequantize", out, codes, scales, type, rows, width, ldo);
  if (rc || rows == 0) return rc;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t row_bytes = ldo * kTypeBytes[type], blocks = blocks_of(width);
  return in_parts(rows, width, [&](int64_t first, uint32_t n, unsigned grid) {
    uint8_t *to = static_cast<uint8_t *>(out) + first * row_bytes;
    const uint8_t *c = codes + first * blocks * kBlock, *sc = scales + first * blocks;
    if (type == SUB1_MX4_BF16)
      mx8_dequantize_kernel<__bf16><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
    else if (type == SUB1_MX4_FP16)
      mx8_dequantize_kernel<_Float16><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
    else
      mx8_dequantize_kernel<float><<<grid, 256, 0, s>>>(c, sc, n, width, to, row_bytes);
  });
}

extern "C" int sub1_mx8_product(const uint8_t *codes, const uint8_t *scales, int height, int width, const uint8_t *x_codes,
                                const uint8_t *x_scales, int relu, void *y, int64_t ldy, uint8_t *y_codes, uint8_t *y_scales,
                                int tokens, void *stream) {
  if (tokens < 0 || tokens > SUB1_MX4_MAX_TOKENS)
    return fail(SUB1_ERR_SHAPE, "sub1_mx8_product: tokens %d outside 0..%d", tokens, SUB1_MX4_MAX_TOKENS);
  if (height < 1 || width < 1 || width > SUB1_MX4_MAX_WIDTH || height > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "sub1_mx8_product: height %d width %d (1..%d)", height, width, SUB1_MX4_MAX_WIDTH);
  if (tokens == 0) return SUB1_OK;
  if (!codes || !scales || !x_codes || !x_scales || !y == !y_codes || !y_codes != !y_scales)
    return fail(SUB1_ERR_NULL, "sub1_mx8_product: both sides' codes and scales, y or its codes and scales");
  if (y && tokens > 1 && ldy < height) return fail(SUB1_ERR_SHAPE, "sub1_mx8_product: row stride smaller than the rows");
  if (misaligned(codes, 16) || misaligned(x_codes, 16) || misaligned(y, 2) || misaligned(y_codes, 16))
    return fail(SUB1_ERR_ALIGN, "sub1_mx8_product: misaligned pointer");
  const Product8Args p{codes, scales, x_codes, x_scales, static_cast<uint16_t *>(y), y_codes, y_scales, ldy, height, width, tokens,
                       relu != 0};
  return launch_product(p, static_cast<hipStream_t>(stream));
}
