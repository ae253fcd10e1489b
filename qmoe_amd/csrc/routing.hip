// Which experts a token goes to, from its router's logits, and the weighted sum of what they put out.
//
//   s = softmax(l) or 1 / (1 + exp(-l)), over all experts; c = s + bias
//   a group's mark: the sum of its group_mark (1 or 2) best c; the top_groups groups with the largest
//   in those the top_k experts with the largest c; their shares s, over their sum if wanted, times a factor
//
// Scores that decide are compared as they are in 64 bits, equal ones by the lower index; without a bias experts
// are in the order of their logits, which scores keep.  What is no number comes last.
#include "mx8.h"

using namespace mx8;
using mx4::Eight;
using sub1::fail;
using sub1::misaligned;

namespace {

struct RouteArgs {
  const uint8_t *logits;
  const float *bias;
  float *shares;
  void *index;
  int64_t row_bytes, tokens;
  int experts, top_k, groups, top_groups, group_mark, sigmoid, normalize, wide_index;
  float scale;
};

constexpr int kMaxGroups = 64;   // a lane each

template <class T>
__device__ __forceinline__ float logit_at(const uint8_t *row, int e);
template <>
__device__ __forceinline__ float logit_at<__bf16>(const uint8_t *row, int e) {
  return sub1::bf16_to_f32(reinterpret_cast<const uint16_t *>(row)[e]);
}
template <>
__device__ __forceinline__ float logit_at<_Float16>(const uint8_t *row, int e) {
  return static_cast<float>(reinterpret_cast<const _Float16 *>(row)[e]);
}
template <>
__device__ __forceinline__ float logit_at<float>(const uint8_t *row, int e) {
  return reinterpret_cast<const float *>(row)[e];
}

// Larger values first as whole numbers; what is no number is 0, below all others.
__device__ __forceinline__ uint64_t rank_of(double v) {
  const uint64_t bits = __double_as_longlong(v + 0.0);   // -0 is 0
  return v != v ? 0 : bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
}
__device__ __forceinline__ double value_of(uint64_t rank) {
  return rank == 0 ? __longlong_as_double(0x7ff8000000000000ull)
                   : __longlong_as_double(rank >> 63 ? rank & 0x7fffffffffffffffull : ~rank);
}

template <class Combine>
__device__ __forceinline__ uint32_t wave_all(uint32_t v, Combine combine) {   // zeros from beyond the lanes do no harm
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppRowShr1, 0xf>(static_cast<int>(v))));
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppRowShr2, 0xf>(static_cast<int>(v))));
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppRowShr4, 0xf>(static_cast<int>(v))));
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppRowShr8, 0xf>(static_cast<int>(v))));
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppBcast15, 0xa>(static_cast<int>(v))));
  v = combine(v, static_cast<uint32_t>(sub1::dpp_or_zero<sub1::kDppBcast31, 0xc>(static_cast<int>(v))));
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  return wave_all(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
  const uint32_t high = wave_largest(static_cast<uint32_t>(v >> 32));
  return static_cast<uint64_t>(high) << 32 | wave_largest(static_cast<uint32_t>(v >> 32) == high ? static_cast<uint32_t>(v) : 0u);
}
__device__ __forceinline__ double wave_total(double v) {
  const uint64_t u = __double_as_longlong(mx4::wave_sum(v));
  return __longlong_as_double(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), 63))) << 32 |
                              static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), 63)));
}

struct Best {
  uint64_t rank;
  int at;   // -1: none
};
// The lanes' best, of equal ranks the lowest `at`.
__device__ __forceinline__ Best wave_best(Best b) {
  const uint64_t rank = wave_largest(b.at < 0 ? 0 : b.rank);
  const uint32_t at = wave_largest(b.at >= 0 && b.rank == rank ? ~static_cast<uint32_t>(b.at) : 0u);
  return {rank, at ? static_cast<int>(~at) : -1};
}

// A wavefront's token, everything computed again in 64 bits wherever it is asked for: right for every case.
template <class T>
__device__ __forceinline__ void route_exactly(const RouteArgs &a, int64_t token) {
  const int lane = threadIdx.x & 63, size = a.experts / a.groups;
  const uint8_t *row = a.logits + token * a.row_bytes;
  double most = 0, under = 1;
  if (!a.sigmoid) {
    uint64_t largest = 0;
    for (int e = lane; e < a.experts; e += 64) largest = max(largest, rank_of(logit_at<T>(row, e)));
    most = value_of(wave_largest(largest));
    if (most == -INFINITY) {
      most = 0;   // all of them masked: scores of zero
    } else {
      double sum = 0;
      for (int e = lane; e < a.experts; e += 64) sum += exp(logit_at<T>(row, e) - most);
      under = wave_total(sum);
    }
  }
  auto score = [&](int e) {
    const double l = logit_at<T>(row, e);
    return a.sigmoid ? 1 / (1 + exp(-l)) : exp(l - most) / under;
  };
  auto biased = [&](int e) { return score(e) + (a.bias ? static_cast<double>(a.bias[e]) : 0.0); };
  auto key = [&](int e) { return rank_of(a.bias ? biased(e) : static_cast<double>(logit_at<T>(row, e))); };
  // this lane's best of an allowed group's, behind `last`
  auto look = [&](Best &best, Best last, int first, int end) {
    for (int e = first + lane; e < end; e += 64) {
      const uint64_t rank = key(e);
      const bool left = rank < last.rank || (rank == last.rank && e > last.at);
      if (left && (best.at < 0 || rank > best.rank)) best = {rank, e};
    }
  };
  constexpr Best kNone = {~uint64_t{0}, -1};   // before the first (nothing has this rank)

  uint64_t allowed = ~uint64_t{0};
  if (a.top_groups < a.groups) {
    uint64_t mark = 0;   // of lane g: that of group g
    for (int g = 0; g < a.groups; g++) {
      Best one = {0, -1}, two = {0, -1};
      look(one, kNone, g * size, g * size + size);
      one = wave_best(one);
      uint64_t rank = one.rank;
      if (a.group_mark == 2) {
        look(two, one, g * size, g * size + size);
        two = wave_best(two);
        rank = rank_of(biased(one.at) + (two.at < 0 ? 0.0 : biased(two.at)));
      }
      if (lane == g) mark = rank;
    }
    allowed = 0;
    Best last = kNone;
    for (int i = 0; i < a.top_groups; i++) {
      const bool left = lane < a.groups && (mark < last.rank || (mark == last.rank && lane > last.at));
      last = wave_best(left ? Best{mark, lane} : Best{0, -1});
      allowed |= uint64_t{1} << last.at;
    }
  }

  Best last = kNone;
  int mine = 0;
  for (int j = 0; j < a.top_k; j++) {
    Best best = {0, -1};
    if (a.groups == 1) {
      look(best, last, 0, a.experts);
    } else {
      for (int g = 0; g < a.groups; g++)
        if (allowed >> g & 1) look(best, last, g * size, g * size + size);
    }
    last = wave_best(best);
    if (lane == j) mine = last.at;
  }
  const bool has = lane < a.top_k;
  double share = has ? score(mine) : 0.0;
  if (a.normalize) {
    const double total = wave_total(share);
    if (total != 0) share /= total;
  }
  if (has) {
    const int64_t at = token * a.top_k + lane;
    a.shares[at] = static_cast<float>(share * a.scale);
    if (a.wide_index)
      static_cast<int64_t *>(a.index)[at] = mine;
    else
      static_cast<int32_t *>(a.index)[at] = mine;
  }
}

template <class T>
__global__ __launch_bounds__(256) void route_kernel(const RouteArgs a) {
  const int64_t token = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (token < a.tokens) route_exactly<T>(a, token);
}

template <class T>
int launch_route(const RouteArgs &a, hipStream_t s) {
  sub1::note_kernel("route_kernel");
  route_kernel<T><<<static_cast<unsigned>((a.tokens + 3) / 4), 256, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// -------------------------------------------------------------- the weighted sum ---

struct CombineArgs {
  const uint8_t *outputs, *residual;
  const float *shares;
  uint8_t *y;
  uint32_t tokens;
  int top_k, width;
};

// Eight values of a token a thread; fp32 sums, in the order of the token's places, the residual last.
template <class T>
__global__ __launch_bounds__(256) void combine_kernel(const CombineArgs a) {
  const uint32_t eights = (a.width + 7) / 8, at = blockIdx.x * 256 + threadIdx.x, token = at / eights;
  if (token >= a.tokens) return;
  const int first = static_cast<int>(at - token * eights) * 8;
  const int64_t row_bytes = static_cast<int64_t>(a.width) * sizeof(T);
  const uint8_t *from = a.outputs + token * a.top_k * row_bytes;
  const float *shares = a.shares + static_cast<int64_t>(token) * a.top_k;
  float sum[8] = {};
  for (int j = 0; j < a.top_k; j++) {
    Eight<T> v;
    v.load(from + j * row_bytes, first, a.width);
    const float share = shares[j];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = fmaf(share, v.at(i), sum[i]);
  }
  if (a.residual) {
    Eight<T> v;
    v.load(a.residual + token * row_bytes, first, a.width);
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] += v.at(i);
  }
  round8<T>(a.y + token * row_bytes, first, a.width, sum);
}

}  // namespace

// ================================================================ C ABI =====

extern "C" int sub1_route(const sub1_router *router, const void *logits, int type, int64_t ldl, int64_t tokens, float *shares,
                          void *index, int index_bytes, void *stream) {
  if (!router) return fail(SUB1_ERR_NULL, "sub1_route: NULL argument");
  const sub1_router &r = *router;
  if (type < 0 || type >= kTypes) return fail(SUB1_ERR_SHAPE, "sub1_route: type %d (SUB1_MX4_BF16, _FP16 or _FP32)", type);
  if (r.experts < 1 || r.experts > SUB1_ROUTE_MAX_EXPERTS || r.groups < 1 || r.groups > kMaxGroups || r.experts % r.groups)
    return fail(SUB1_ERR_SHAPE, "sub1_route: %d experts (1..%d) in %d groups (1..%d, of one size)", r.experts, SUB1_ROUTE_MAX_EXPERTS,
                r.groups, kMaxGroups);
  if (r.top_groups < 1 || r.top_groups > r.groups || (r.group_mark != 1 && r.group_mark != 2))
    return fail(SUB1_ERR_SHAPE, "sub1_route: %d of %d groups by their %d best", r.top_groups, r.groups, r.group_mark);
  if (r.top_k < 1 || r.top_k > SUB1_ROUTE_MAX_TOP_K || r.top_k > r.experts / r.groups * r.top_groups)
    return fail(SUB1_ERR_SHAPE, "sub1_route: %d experts a token of %d (at most %d)", r.top_k, r.experts / r.groups * r.top_groups,
                SUB1_ROUTE_MAX_TOP_K);
  if ((r.scores != SUB1_ROUTE_SOFTMAX && r.scores != SUB1_ROUTE_SIGMOID) || !(r.scale - r.scale == 0))
    return fail(SUB1_ERR_SHAPE, "sub1_route: scores %d, factor %g", r.scores, static_cast<double>(r.scale));
  if (index_bytes != 4 && index_bytes != 8) return fail(SUB1_ERR_SHAPE, "sub1_route: an index of %d bytes (4 or 8)", index_bytes);
  if (tokens < 0 || tokens > SUB1_ROUTE_MAX_TOKENS)
    return fail(SUB1_ERR_SHAPE, "sub1_route: tokens %lld outside 0..%d", static_cast<long long>(tokens), SUB1_ROUTE_MAX_TOKENS);
  if (tokens == 0) return SUB1_OK;
  if (!logits || !shares || !index) return fail(SUB1_ERR_NULL, "sub1_route: NULL argument");
  if (tokens > 1 && ldl < r.experts) return fail(SUB1_ERR_SHAPE, "sub1_route: row stride smaller than the rows");
  if (misaligned(logits, kTypeBytes[type]) || misaligned(shares, 4) || misaligned(index, index_bytes) || misaligned(r.bias, 4))
    return fail(SUB1_ERR_ALIGN, "sub1_route: misaligned pointer");
  const RouteArgs a{static_cast<const uint8_t *>(logits), r.bias, shares, index, ldl * kTypeBytes[type], tokens, r.experts, r.top_k,
                    r.groups, r.top_groups, r.group_mark, r.scores == SUB1_ROUTE_SIGMOID, r.normalize != 0, index_bytes == 8, r.scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (type == SUB1_MX4_BF16) return launch_route<__bf16>(a, s);
  if (type == SUB1_MX4_FP16) return launch_route<_Float16>(a, s);
  return launch_route<float>(a, s);
}

extern "C" int sub1_combine(const void *outputs, int type, const float *shares, const void *residual, int64_t tokens, int top_k,
                            int width, void *y, void *stream) {
  if (type < 0 || type >= kTypes) return fail(SUB1_ERR_SHAPE, "sub1_combine: type %d (SUB1_MX4_BF16, _FP16 or _FP32)", type);
  if (tokens < 0 || tokens > SUB1_ROUTE_MAX_TOKENS || top_k < 1 || top_k > SUB1_ROUTE_MAX_TOP_K || width < 1 || width > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "sub1_combine: %lld tokens (0..%d) of %d outputs (1..%d) of width %d (1..%d)",
                static_cast<long long>(tokens), SUB1_ROUTE_MAX_TOKENS, top_k, SUB1_ROUTE_MAX_TOP_K, width, SUB1_MX4_MAX_WIDTH);
  if (tokens == 0) return SUB1_OK;
  if (!outputs || !shares || !y) return fail(SUB1_ERR_NULL, "sub1_combine: NULL argument");
  const int64_t size = kTypeBytes[type];
  if (misaligned(outputs, size) || misaligned(residual, size) || misaligned(y, size) || misaligned(shares, 4))
    return fail(SUB1_ERR_ALIGN, "sub1_combine: misaligned pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t eights = (width + 7) / 8, most = (int64_t{1} << 31) / eights, row_bytes = width * size;
  for (int64_t first = 0; first < tokens; first += most) {   // in launches of at most 2^31 threads
    const int64_t n = tokens - first < most ? tokens - first : most;
    const CombineArgs a{static_cast<const uint8_t *>(outputs) + first * top_k * row_bytes,
                        residual ? static_cast<const uint8_t *>(residual) + first * row_bytes : nullptr, shares + first * top_k,
                        static_cast<uint8_t *>(y) + first * row_bytes, static_cast<uint32_t>(n), top_k, width};
    const unsigned grid = static_cast<unsigned>((n * eights + 255) / 256);
    if (type == SUB1_MX4_BF16)
      combine_kernel<__bf16><<<grid, 256, 0, s>>>(a);
    else if (type == SUB1_MX4_FP16)
      combine_kernel<_Float16><<<grid, 256, 0, s>>>(a);
    else
      combine_kernel<float><<<grid, 256, 0, s>>>(a);
    HIP_TRY(hipGetLastError());
  }
  return SUB1_OK;
}
