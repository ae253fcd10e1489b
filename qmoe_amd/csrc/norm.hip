// Root-mean-square norm of rows, the residual's addition before it, the result in the input's type or in
// microscaled 8 bits:
//   s = x + r, rounded to r's type; y = s / sqrt(mean(s^2) + eps) * w
#include "mx8.h"

using namespace mx8;
using mx4::Eight;
using sub1::fail;
using sub1::misaligned;

namespace {

struct NormArgs {
  const uint8_t *x, *residual, *weight;
  uint8_t *total, *y, *codes, *scales;
  int64_t x_bytes, residual_bytes, total_bytes, y_bytes;   // from a row to the next
  int64_t rows;
  double eps, inverse_width;
  int width, weight_fp32;
};

template <class R>
__device__ __forceinline__ float rounded_to(float v) {
  return static_cast<float>(static_cast<R>(v));
}

// 1 / sqrt(mean + eps).  Of rows so large that it would leave fp32's normal range, values are brought down first.
struct Factor {
  float before, by;
  __device__ __forceinline__ float times(float v) const { return v * before * by; }
};
__device__ __forceinline__ Factor factor_of(const NormArgs &a, double sum) {
  const double factor = rsqrt(sum * a.inverse_width + a.eps);
  const bool large = factor < 0x1p-100;
  return {large ? 0x1p-64f : 1.0f, static_cast<float>(large ? factor * 0x1p64 : factor)};
}

// A row's values stay in registers, kPer eights a thread: one read of x and r, one write of s and y.  The sum of
// squares is held in 64 bits: no square of an fp32 value overflows there and the order of the sum does not count; the
// vector units add and multiply 64 bits as fast as 32.  kLanes: 16 or 64 lanes a row, where nothing waits for another
// wavefront; 0: a workgroup a row. Bound by HBM: 16384 x 2080 in bf16 with a residual, to 8 bits, 48 us in a graph, 5.0
// TB/s (a copy: 4.95 to 5.4); 16384 x 1023 in fp16, whose rows do not lie on 16 bytes, 3.7 TB/s.  Loads and stores that
// pass the caches by measured alike.
template <class T, class R, bool kResidual, int kLanes, int kPer>
__global__ __launch_bounds__(kLanes ? 256 : 1024) void rms_norm_kernel(const NormArgs a) {
  __shared__ double parts[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kRows = kLanes ? 256 / kLanes : 1;
  const int64_t mine = kLanes ? blockIdx.x * int64_t{kRows} + threadIdx.x / (kLanes ? kLanes : 1) : blockIdx.x;
  if (kLanes != 0 && mine - lane / (kLanes ? kLanes : 1) >= a.rows) return;   // (a whole wavefront)
  const int64_t row = kLanes == 16 && mine >= a.rows ? a.rows - 1 : mine;     // what is not there repeats the wavefront's last row
  const int me = kLanes ? threadIdx.x % (kLanes ? kLanes : 1) : threadIdx.x, lanes = kLanes ? kLanes : static_cast<int>(blockDim.x);
  float v[kPer][8], w[kPer][8];
  {
    const uint8_t *from = a.x + row * a.x_bytes, *other = a.residual + row * a.residual_bytes;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
      const int first = 8 * (me + i * lanes);
      Eight<T> x;
      x.load(from, first, a.width);
      if constexpr (kResidual) {
        Eight<R> r;
        r.load(other, first, a.width);
#pragma unroll
        for (int k = 0; k < 8; k++) v[i][k] = rounded_to<R>(x.at(k) + r.at(k));
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[i][k] = x.at(k);
      }
    }
  }
  auto weights = [&](int i) {
    if (a.weight_fp32) {
      Eight<float> e;
      e.load(a.weight, 8 * (me + i * lanes), a.width);
#pragma unroll
      for (int k = 0; k < 8; k++) w[i][k] = e.at(k);
    } else {
      Eight<T> e;
      e.load(a.weight, 8 * (me + i * lanes), a.width);
#pragma unroll
      for (int k = 0; k < 8; k++) w[i][k] = e.at(k);
    }
  };
  constexpr bool kEarly = kPer <= 2;   // asked for with the values, where registers are left
  if (kEarly) {
#pragma unroll
    for (int i = 0; i < kPer; i++) weights(i);
  }
  if constexpr (kResidual) {
#pragma unroll
    for (int i = 0; i < kPer; i++) round8<R>(a.total + row * a.total_bytes, 8 * (me + i * lanes), a.width, v[i]);
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; i++)
#pragma unroll
    for (int k = 0; k < 8; k++) sum = fma(static_cast<double>(v[i][k]), static_cast<double>(v[i][k]), sum);
  if constexpr (kLanes != 0) {
    sum = sum_over<kLanes>(sum);
  } else {
    sum = mx4::wave_sum(sum);
    if (lane == 63) parts[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int i = 0; i < lanes / 64; i++) sum += parts[i];
  }
  const Factor f = factor_of(a, sum);
#pragma unroll
  for (int i = 0; i < kPer; i++) {
    const int first = 8 * (me + i * lanes);
    float y[8];
    if (!kEarly) weights(i);
#pragma unroll
    for (int k = 0; k < 8; k++) y[k] = f.times(v[i][k]) * w[i][k];
    if (a.codes)
      store_block(y, a.codes, a.scales, row * blocks_of(a.width) * 4 + first / 8, first < blocks_of(a.width) * kBlock);
    else
      round8<T>(a.y + row * a.y_bytes, first, a.width, y);
  }
}

// Rows too wide for registers, a workgroup each: they are read a second time, what was added from `total`, where each thread
// reads what it has written.  1024 x 40000 in bf16 with a residual, to 8 bits, 62 us in a graph, without one to bf16 36: 4.6
// TB/s of what has to be moved; 64 rows 10 and 7.5, one of 65536 12.5 and 9.
template <class T, class R, bool kResidual>
__global__ __launch_bounds__(1024) void rms_norm_wide_kernel(const NormArgs a) {
  __shared__ double parts[16];
  const int64_t row = blockIdx.x;
  const int end = blocks_of(a.width) * kBlock;
  const uint8_t *from = a.x + row * a.x_bytes;
  double sum = 0;
  for (int first = 8 * threadIdx.x; first < end; first += 8 * 1024) {
    Eight<T> x;
    x.load(from, first, a.width);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = x.at(k);
    if constexpr (kResidual) {
      Eight<R> r;
      r.load(a.residual + row * a.residual_bytes, first, a.width);
#pragma unroll
      for (int k = 0; k < 8; k++) v[k] = rounded_to<R>(v[k] + r.at(k));
      round8<R>(a.total + row * a.total_bytes, first, a.width, v);
    }
#pragma unroll
    for (int k = 0; k < 8; k++) sum = fma(static_cast<double>(v[k]), static_cast<double>(v[k]), sum);
  }
  sum = mx4::wave_sum(sum);
  if ((threadIdx.x & 63) == 63) parts[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0;
  for (int i = 0; i < 16; i++) sum += parts[i];
  const Factor f = factor_of(a, sum);
  for (int first = 8 * threadIdx.x; first < end; first += 8 * 1024) {   // (a block's four lanes together)
    float v[8], w[8];
    auto take = [&](auto type, const uint8_t *row_of, float (&to)[8]) {
      Eight<decltype(type)> e;
      e.load(row_of, first, a.width);
#pragma unroll
      for (int k = 0; k < 8; k++) to[k] = e.at(k);
    };
    if constexpr (kResidual)
      take(R(), a.total + row * a.total_bytes, v);
    else
      take(T(), from, v);
    if (a.weight_fp32)
      take(float(), a.weight, w);
    else
      take(T(), a.weight, w);
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] = f.times(v[k]) * w[k];
    if (a.codes)
      store_block(v, a.codes, a.scales, row * blocks_of(a.width) * 4 + first / 8, true);
    else
      round8<T>(a.y + row * a.y_bytes, first, a.width, v);
  }
}

template <class T, class R, bool kResidual, int kLanes, int kPer>
void launch_lanes(const NormArgs &a, hipStream_t s) {
  constexpr int kRows = 256 / kLanes;
  rms_norm_kernel<T, R, kResidual, kLanes, kPer><<<static_cast<unsigned>((a.rows + kRows - 1) / kRows), 256, 0, s>>>(a);
}

// Which form (us, in a graph).  Few rows: a workgroup each, an eight a thread as far as 1024 threads go (1000 x 2080,
// residual, to 8 bits 6.1, by a wavefront each 7.2; 4000 14.2 and 15.3), and rows of fp32 that a wavefront's registers
// hold barely (4096 x 4096, residual 43 and 50).  Many: a wavefront each (16384 x 2080 48 and 53; without residual 26
// and 36).  Many narrow ones: a quarter of one (16384 x 100 5.8 and 11, 16000 x 300 11.3 and 12.8; 1000 x 300 by a
// workgroup each 3.9, by quarters 4.7).
template <class T, class R, bool kResidual>
int launch_rows(const NormArgs &a, hipStream_t s) {
  const int eights = blocks_of(a.width) * 4;
  const bool in_fp32 = sizeof(T) == 4 || (kResidual && sizeof(R) == 4);
  if (eights <= 64 && a.rows > 2048) {
    sub1::note_kernel("rms_norm_kernel, 16 lanes a row");
    if (eights <= 16) launch_lanes<T, R, kResidual, 16, 1>(a, s);
    else if (eights <= 32) launch_lanes<T, R, kResidual, 16, 2>(a, s);
    else if (eights <= 48) launch_lanes<T, R, kResidual, 16, 3>(a, s);
    else launch_lanes<T, R, kResidual, 16, 4>(a, s);
  } else if (a.rows > 4096 && eights <= (in_fp32 ? 4 : 8) * 64) {
    sub1::note_kernel("rms_norm_kernel, a wavefront a row");
    const int per = (eights + 63) / 64;   // (narrower rows took quarters)
    if (per == 2) launch_lanes<T, R, kResidual, 64, 2>(a, s);
    else if (per == 3) launch_lanes<T, R, kResidual, 64, 3>(a, s);
    else if (per == 4) launch_lanes<T, R, kResidual, 64, 4>(a, s);
    else if constexpr (sizeof(T) == 2 && sizeof(R) == 2) {
      if (per == 5) launch_lanes<T, R, kResidual, 64, 5>(a, s);
      else if (per == 6) launch_lanes<T, R, kResidual, 64, 6>(a, s);
      else launch_lanes<T, R, kResidual, 64, 8>(a, s);
    }
  } else {
    sub1::note_kernel(eights <= 4096 ? "rms_norm_kernel, a workgroup a row" : "rms_norm_wide_kernel, a workgroup a row");
    const unsigned grid = static_cast<unsigned>(a.rows);
    if (eights <= 1024) rms_norm_kernel<T, R, kResidual, 0, 1><<<grid, (eights + 63) / 64 * 64, 0, s>>>(a);
    else if (eights <= 2048) rms_norm_kernel<T, R, kResidual, 0, 2><<<grid, 1024, 0, s>>>(a);
    else if (eights <= 4096) rms_norm_kernel<T, R, kResidual, 0, 4><<<grid, 1024, 0, s>>>(a);
    else rms_norm_wide_kernel<T, R, kResidual><<<grid, 1024, 0, s>>>(a);
  }
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// In launches of at most 2^31 threads.
template <class T, class R>
int launch(const NormArgs &all, hipStream_t s) {
  constexpr int64_t kMost = int64_t{1} << 21;
  for (int64_t first = 0; first < all.rows; first += kMost) {
    NormArgs a = all;
    const int64_t blocks = blocks_of(a.width);
    a.rows = all.rows - first < kMost ? all.rows - first : kMost;
    a.x += first * a.x_bytes;
    if (a.residual) a.residual += first * a.residual_bytes, a.total += first * a.total_bytes;
    if (a.codes) a.codes += first * blocks * kBlock, a.scales += first * blocks;
    else a.y += first * a.y_bytes;
    const int rc = all.residual ? launch_rows<T, R, true>(a, s) : launch_rows<T, T, false>(a, s);
    if (rc) return rc;
  }
  return SUB1_OK;
}

}  // namespace

// ================================================================ C ABI =====

extern "C" int sub1_rms_norm(const sub1_norm *norm, const void *x, int64_t ldx, const void *residual, int64_t ldr, void *total,
                             int64_t ldt, void *y, int64_t ldy, uint8_t *codes, uint8_t *scales, int64_t rows, void *stream) {
  if (!norm) return fail(SUB1_ERR_NULL, "sub1_rms_norm: NULL argument");
  const int width = norm->width, type = norm->type, rtype = norm->residual_type;
  auto type_fits = [&](int t) { return t == type || t == SUB1_MX4_FP32; };
  if (type < 0 || type >= kTypes || !type_fits(rtype) || !type_fits(norm->weight_type))
    return fail(SUB1_ERR_SHAPE, "sub1_rms_norm: types %d, residual %d, weight %d (SUB1_MX4_BF16, _FP16 or _FP32; the others x's or _FP32)",
                type, rtype, norm->weight_type);
  if (rows < 0 || rows > SUB1_NORM_MAX_ROWS || width < 1 || width > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "sub1_rms_norm: %lld rows of width %d (1..%d)", static_cast<long long>(rows), width, SUB1_MX4_MAX_WIDTH);
  if (!(norm->eps >= SUB1_NORM_LEAST_EPS && norm->eps <= 1e30))
    return fail(SUB1_ERR_SHAPE, "sub1_rms_norm: eps %g outside %g..1e30", norm->eps, SUB1_NORM_LEAST_EPS);
  if (rows == 0) return SUB1_OK;
  if (!x || !norm->weight || !residual != !total || !codes != !scales || !y == !codes)
    return fail(SUB1_ERR_NULL, "sub1_rms_norm: x and weight, residual and total or neither, y or codes and scales");
  if (rows > 1 && (ldx < width || (residual && (ldr < width || ldt < width)) || (y && ldy < width)))
    return fail(SUB1_ERR_SHAPE, "sub1_rms_norm: row strides smaller than the rows");
  const int64_t size = kTypeBytes[type], rsize = kTypeBytes[rtype];
  if (misaligned(x, size) || misaligned(norm->weight, kTypeBytes[norm->weight_type]) || misaligned(residual, rsize) ||
      misaligned(total, rsize) || misaligned(y, size) || misaligned(codes, 16))
    return fail(SUB1_ERR_ALIGN, "sub1_rms_norm: misaligned pointer");
  const NormArgs a{static_cast<const uint8_t *>(x), static_cast<const uint8_t *>(residual),
                   static_cast<const uint8_t *>(norm->weight), static_cast<uint8_t *>(total), static_cast<uint8_t *>(y), codes, scales,
                   ldx * size, ldr * rsize, ldt * rsize, ldy * size, rows, norm->eps, 1.0 / width, width,
                   norm->weight_type == SUB1_MX4_FP32};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (type == SUB1_MX4_FP32) return launch<float, float>(a, s);
  if (type == SUB1_MX4_BF16) return rtype == type ? launch<__bf16, __bf16>(a, s) : launch<__bf16, float>(a, s);
  return rtype == type ? launch<_Float16, _Float16>(a, s) : launch<_Float16, float>(a, s);
}
