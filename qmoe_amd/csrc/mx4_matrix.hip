// Microscaled 4-bit matrices: values to the format and back, and products with them.
#include "mx4.h"

using namespace mx4;
using sub1::fail;
using sub1::misaligned;

namespace {

// ------------------------------------------------------- to the format and back ---

// The type of the values that a kernel reads or writes, as eight of them at once.
template <class T>
struct Eight;
template <>
struct Eight<__bf16> {
  u32x4 raw;
  __device__ __forceinline__ void load(const uint8_t *row, int first, int width) {
    raw = load8(reinterpret_cast<const uint16_t *>(row), first, width);
  }
  __device__ __forceinline__ float at(int i) const {
    return __uint_as_float(i & 1 ? raw[i / 2] & 0xffff0000u : raw[i / 2] << 16);
  }
  static __device__ __forceinline__ void store(uint8_t *row, int first, int width, const float (&v)[8]) {
    uint16_t *p = reinterpret_cast<uint16_t *>(row) + first;
    uint32_t two[4];   // exact: a bf16 has room for a code under any scale
#pragma unroll
    for (int i = 0; i < 4; i++) two[i] = __float_as_uint(v[2 * i]) >> 16 | (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
    if (first + 8 <= width) {
      __builtin_memcpy(p, two, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (first + i < width) p[i] = static_cast<uint16_t>(two[i / 2] >> (16 * (i & 1)));
    }
  }
};
template <>
struct Eight<_Float16> {
  u32x4 raw;
  __device__ __forceinline__ void load(const uint8_t *row, int first, int width) {
    raw = load8(reinterpret_cast<const uint16_t *>(row), first, width);
  }
  __device__ __forceinline__ float at(int i) const {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(raw[i / 2] >> (16 * (i & 1)))));
  }
  static __device__ __forceinline__ void store(uint8_t *row, int first, int width, const float (&v)[8]) {
    _Float16 *p = reinterpret_cast<_Float16 *>(row) + first;
    _Float16 half[8];   // to nearest: large scales leave this type's range, small ones its steps
#pragma unroll
    for (int i = 0; i < 8; i++) half[i] = static_cast<_Float16>(v[i]);
    if (first + 8 <= width) {
      __builtin_memcpy(p, half, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (first + i < width) p[i] = half[i];
    }
  }
};
template <>
struct Eight<float> {
  float raw[8];
  __device__ __forceinline__ void load(const uint8_t *row, int first, int width) {
    const float *p = reinterpret_cast<const float *>(row) + first;
    if (first + 8 <= width) {
      __builtin_memcpy(raw, p, 32);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) raw[i] = first + i < width ? p[i] : 0.0f;
    }
  }
  __device__ __forceinline__ float at(int i) const { return raw[i]; }
  static __device__ __forceinline__ void store(uint8_t *row, int first, int width, const float (&v)[8]) {
    float *p = reinterpret_cast<float *>(row) + first;
    if (first + 8 <= width) {
      __builtin_memcpy(p, v, 32);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (first + i < width) p[i] = v[i];
    }
  }
};

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

// Four rows of one token's y, from `row` on.
__device__ __forceinline__ void store_four(uint16_t *y, int row, int height, f32x4 sum) {
  const uint32_t two[2] = {two_bf16(sum[0], sum[1]), two_bf16(sum[2], sum[3])};
  if (row + 4 <= height) {
    __builtin_memcpy(y + row, two, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (row + i < height) y[row + i] = static_cast<uint16_t>(two[i / 2] >> (16 * (i & 1)));
  }
}

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
    x[n] = token < p.tokens ? p.x + token * p.ldx : nullptr;
  }
  FewSums<kRows, kTokens> sums;
  few_products<kRows, kTokens>(sums, p.codes + row0 * blocks * kBlockBytes, p.scales + row0 * blocks, p.height - row0,
                               p.width, x);
  few_join<kRows, kTokens>(sums, lds, [&](int r, int n, f32x4 sum) {
    const int token = token0 + 16 * n + (lane & 15);
    if (token < p.tokens) store_four(p.y + token * p.ldy, row0 + 16 * r + 4 * (lane >> 4), p.height, sum);
  });
}

struct QuantizedArgs {
  const uint8_t *codes, *scales, *x_codes, *x_scales;
  uint16_t *y;
  int64_t ldy;
  int height, width, tokens;
};

// Both sides in the format: a wavefront takes 16 rows and 16 tokens, 128 values of each a step, which the
// matrix core multiplies from the codes as they are, each lane's block under its own scale.
__global__ __launch_bounds__(256) void mx4_quantized_kernel(const QuantizedArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = lane >> 4;
  const int row0 = blockIdx.x * 16, token0 = blockIdx.y * 64 + 16 * wave;
  if (token0 >= p.tokens) return;
  const int blocks = blocks_of(p.width);
  const int64_t row = min(row0 + (lane & 15), p.height - 1), token = min(token0 + (lane & 15), p.tokens - 1);
  f32x4 sum = {0, 0, 0, 0};
  for (int block = group; block < (blocks + 3) / 4 * 4; block += 4) {
    i32x8 a = {0, 0, 0, 0, 0, 0, 0, 0}, b = {0, 0, 0, 0, 0, 0, 0, 0};
    int sa = 0, sb = 0;
    if (block < blocks) {
      const u32x4 va = *reinterpret_cast<const u32x4 *>(p.codes + (row * blocks + block) * kBlockBytes);
      const u32x4 vb = *reinterpret_cast<const u32x4 *>(p.x_codes + (token * blocks + block) * kBlockBytes);
#pragma unroll
      for (int i = 0; i < 4; i++) a[i] = va[i], b[i] = vb[i];
      sa = p.scales[row * blocks + block];
      sb = p.x_scales[token * blocks + block];
    }
    sum = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, sum, 4, 4, 0, sa, 0, sb);
  }
  const int t = token0 + (lane & 15);
  if (t < p.tokens) store_four(p.y + t * p.ldy, row0 + 4 * group, p.height, sum);
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
  const unsigned rows = (height + 15) / 16;
  sub1::note_kernel("mx4_few_kernel");
  if (tokens <= 16)
    mx4_few_kernel<1, 1><<<dim3(rows, 1), 64 * kFewWaves, 0, s>>>(p);
  else
    mx4_few_kernel<1, 2><<<dim3(rows, (tokens + 31) / 32), 64 * kFewWaves, 0, s>>>(p);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
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
  sub1::note_kernel("mx4_quantized_kernel");
  mx4_quantized_kernel<<<dim3((height + 15) / 16, (tokens + 63) / 64), 256, 0, s>>>(p);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}
