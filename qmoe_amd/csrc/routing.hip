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
  int experts, top_k, groups, top_groups, group_mark, sigmoid, normalize, wide_index, group_bits;   // 2^group_bits: groups and more
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

template <int kLanes>
__device__ __forceinline__ uint32_t largest_over(uint32_t v) {
  return over_lanes<kLanes>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int kLanes>
__device__ __forceinline__ uint32_t smallest_over(uint32_t v) {
  return over_lanes<kLanes>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int kLanes>
__device__ __forceinline__ uint64_t largest_over(uint64_t v) {
  const uint32_t high = largest_over<kLanes>(static_cast<uint32_t>(v >> 32));
  return static_cast<uint64_t>(high) << 32 | largest_over<kLanes>(static_cast<uint32_t>(v >> 32) == high ? static_cast<uint32_t>(v) : 0u);
}
struct Best {
  uint64_t rank;
  int at;   // -1: none
};
// The lanes' best, of equal ranks the lowest `at`.
__device__ __forceinline__ Best wave_best(Best b) {
  const uint64_t rank = largest_over<64>(b.at < 0 ? uint64_t{0} : b.rank);
  const uint32_t at = largest_over<64>(b.at >= 0 && b.rank == rank ? ~static_cast<uint32_t>(b.at) : 0u);
  return {rank, at ? static_cast<int>(~at) : -1};
}

__device__ __forceinline__ void store_choice(const RouteArgs &a, int64_t token, int place, double share, int expert) {
  const int64_t at = token * a.top_k + place;
  a.shares[at] = static_cast<float>(share * a.scale);
  if (a.wide_index)
    static_cast<int64_t *>(a.index)[at] = expert;
  else
    static_cast<int32_t *>(a.index)[at] = expert;
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
    most = value_of(largest_over<64>(largest));
    if (most == -INFINITY) {
      most = 0;   // all of them masked: scores of zero
    } else {
      double sum = 0;
      for (int e = lane; e < a.experts; e += 64) sum += exp(logit_at<T>(row, e) - most);
      under = sum_over<64>(sum);
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
    const double total = sum_over<64>(share);
    if (total != 0) share /= total;
  }
  if (has) store_choice(a, token, lane, share, mine);
}

template <class T>
__global__ __launch_bounds__(256) void route_exact_kernel(const RouteArgs a) {
  const int64_t token = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
  if (token < a.tokens) route_exactly<T>(a, token);
}

// ---------------------------------------------------------------- the quick form ---

__device__ __forceinline__ uint32_t rank32(float v) {   // as rank_of; of numbers alone
  const int32_t bits = __float_as_int(v + 0.0f);
  return static_cast<uint32_t>(bits ^ (bits >> 31 | static_cast<int32_t>(0x80000000)));
}
__device__ __forceinline__ float value32(uint32_t rank) {
  return __uint_as_float(rank >> 31 ? rank & 0x7fffffffu : ~rank);
}

// kLanes lanes a token, kPer experts a lane; one read of the logits.  Bound by its instructions' latency (VALU busy for 20 % or
// more, two wavefronts a SIMD), not by memory: 8192 tokens' 8 of 256 in groups, with a bias, 8.0 us a call (9.2 MB would take 2), of which the choice of
// groups takes 1.9, the eight choices 1.4, the bias and its scores 1.6, the rest a launch, the logits' trip and a look
// at the chosen ones'; one token's kernel 2.0.  A kernel for each kind of scores, with and without a bias: 9.7 in a
// graph, 11.6 where both were asked for at run time.  Scores are computed in 32 bits, which places all experts but
// those next to each other; from there are taken the top_k and on as long as the next may be one of them for all that
// is known, and of those alone the order is found in 64 bits; where they are equal to the last bit (padding, coarse
// logits) the lower indexes are the answer, and no more are looked at.  Groups' marks too close to tell are computed
// again in 64 bits, of the experts that may be in them. What is still open (more near the last than there are lanes)
// and what is no number goes to the exact form.  A lane has experts of one group, as many together as 16 bytes of
// logits hold, then those behind the group's other lanes', kPer in all.  An expert's key is its rank with j in the last
// bits, so that the largest key says which it is.
template <class T, int kLanes, int kPer, bool kSigmoid, bool kBias>
__device__ __forceinline__ bool route_quickly(const RouteArgs &a, int64_t token) {
  __shared__ uint16_t all_places[256];
  uint16_t *const places = all_places + (threadIdx.x & ~(kLanes - 1));   // of this token
  constexpr uint32_t kIndex = kPer - 1;
  constexpr float kLog2e = 1.44269504f;
  const int lane = threadIdx.x & (kLanes - 1), size = a.experts / a.groups, group_lanes = kLanes >> a.group_bits;
  const int group = lane / group_lanes, sub = lane & (group_lanes - 1), base = group * size;
  const bool in_group = group < a.groups;
  const uint8_t *row = a.logits + token * a.row_bytes;
  constexpr int kTogether = kPer < 16 / static_cast<int>(sizeof(T)) ? kPer : 16 / static_cast<int>(sizeof(T));
  auto at_of = [&](int j) { return kTogether * (sub + group_lanes * (j / kTogether)) + j % kTogether; };   // in its group
  float v[kPer], b[kPer];
  const T *const logits = reinterpret_cast<const T *>(row) + base;
#pragma unroll
  for (int j = 0; j < kPer; j += kTogether) {
    T some[kTogether] = {};
    if (in_group && at_of(j) + kTogether <= size) {
      __builtin_memcpy(some, logits + at_of(j), sizeof(some));
    } else {
#pragma unroll
      for (int i = 0; i < kTogether; i++)
        if (in_group && at_of(j + i) < size) some[i] = logits[at_of(j + i)];
    }
#pragma unroll
    for (int i = 0; i < kTogether; i++) v[j + i] = static_cast<float>(some[i]);
  }
  if constexpr (kBias) {
#pragma unroll
    for (int j = 0; j < kPer; j += kTogether) {
      float some[kTogether] = {};
      if (in_group && at_of(j) + kTogether <= size) {
        __builtin_memcpy(some, a.bias + base + at_of(j), sizeof(some));
      } else {
#pragma unroll
        for (int i = 0; i < kTogether; i++)
          if (in_group && at_of(j + i) < size) some[i] = a.bias[base + at_of(j + i)];
      }
#pragma unroll
      for (int i = 0; i < kTogether; i++) b[j + i] = some[i];
    }
  }
  bool odd = false;   // something that the exact form has to look at
  float most = 0, largest_score = 1;
  double under = 1;
  constexpr bool approximate = kBias;
  const int limit = in_group ? size : 0;
  auto there = [&](int j) { return at_of(j) < limit; };
  if (!kSigmoid) {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPer; j++) m = there(j) ? fmaxf(m, v[j]) : m;
    most = value32(largest_over<kLanes>(rank32(m)));
    double sum[4] = {0, 0, 0, 0};   // (four chains: one of 64-bit sums takes its time)
#pragma unroll
    for (int j = 0; j < kPer; j++)
      sum[j % 4] += static_cast<double>(there(j) ? __builtin_amdgcn_exp2f((v[j] - most) * kLog2e) : 0.0f);
    under = sum_over<kLanes>((sum[0] + sum[1]) + (sum[2] + sum[3]));
    if (most == -INFINITY) most = 0, under = 1;   // all of them masked: scores of zero
    largest_score = static_cast<float>(1 / under);
    odd |= !(fabsf(most) < INFINITY);
  }
  const float over = largest_score;
  auto score32 = [&](float l) {
    return kSigmoid ? __builtin_amdgcn_rcpf(1 + __builtin_amdgcn_exp2f(-l * kLog2e)) : __builtin_amdgcn_exp2f((l - most) * kLog2e) * over;
  };
  // How far apart two sums of scores and biases near `c` may be taken for when they are not.  A sigmoid is off by less
  // than 2^-22 (its argument's rounding, at most 1.5 |l| 2^-24 s (1 - s), the exponential's and the quotient's steps),
  // a share by less than 2^-20 of the largest (|l - most| e^(l - most) is at most 0.37; a sum over 4096 is off by 2^-20
  // of itself); a sum's steps are 2^-24 c.
  auto tolerance = [&](float c) { return (kSigmoid ? 0x1p-20f : 0x1p-18f * largest_score) + 0x1p-21f * fabsf(c); };
  auto exact_score = [&](float l) {
    return kSigmoid ? 1 / (1 + exp(-static_cast<double>(l))) : exp(static_cast<double>(l) - most) / under;
  };
  auto sum_exactly = [&] {
    double sum = 0;
#pragma unroll 1   // (seldom, and long)
    for (int j = 0; j < kPer; j++)
      if (there(j)) sum += exp(static_cast<double>(logit_at<T>(row, base + at_of(j))) - most);
    sum = sum_over<kLanes>(sum);
    under = sum == 0 ? 1 : sum;
  };
  float one = -INFINITY, two = -INFINITY;   // the lane's best of its group, for the group's mark
  const bool by_marks = a.top_groups < a.groups, marks_of_scores = approximate || a.group_mark == 2;
  uint32_t key[kPer];
#pragma unroll
  for (int j = 0; j < kPer; j++) {
    if (approximate) v[j] = score32(v[j]) + b[j];
    odd |= there(j) && (approximate ? !(fabsf(v[j]) < INFINITY) : v[j] != v[j]);
    key[j] = there(j) ? (rank32(v[j]) & ~kIndex) | (kIndex - j) : 0;
  }
  if (by_marks) {
    if (!approximate && marks_of_scores) {
#pragma unroll
      for (int j = 0; j < kPer; j++) v[j] = score32(v[j]);
    }
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const float c = there(j) ? v[j] : -INFINITY;
      two = fmaxf(two, fminf(one, c));
      one = fmaxf(one, c);
    }
    for (int by = 1; by < group_lanes; by *= 2) {
      const float other_one = __shfl_xor(one, by, kLanes), other_two = __shfl_xor(two, by, kLanes);
      two = fmaxf(fmaxf(two, other_two), fminf(one, other_one));
      one = fmaxf(one, other_one);
    }
    const bool of_two = a.group_mark == 2 && size > 1;
    const float mark = of_two ? one + two : one;
    odd |= in_group && marks_of_scores && !(fabsf(mark) < INFINITY);
    const uint32_t rank = in_group ? rank32(mark) : 0;
    bool taken = false;
    auto pick = [&](auto from) {   // the groups with the largest marks, of equal ones the lower
      taken = false;
      for (int i = 0; i < a.top_groups; i++) {
        const auto most_of = largest_over<kLanes>(taken ? decltype(from)(0) : from);
        taken |= static_cast<uint32_t>(group) == smallest_over<kLanes>(!taken && from == most_of ? static_cast<uint32_t>(group) : ~0u);
      }
    };
    pick(rank);
    if (marks_of_scores) {
      // A mark is off by what its addends are, which may be larger than it (two scores' errors, two sums' roundings, that
      // of their own sum and one of what follows here): no group taken may be below one not taken.
      const float off = 0.5f * tolerance(0) + 0x1p-22f * (of_two ? fabsf(one) + fabsf(two) : fabsf(one));
      const uint32_t kept = smallest_over<kLanes>(taken && in_group ? rank32(mark - off) : ~0u);
      const uint32_t next = largest_over<kLanes>(!taken && in_group ? rank32(mark + off) : 0);
      if (__ballot(!odd && !(next < kept))) {   // too close: marks in 64 bits, of the experts that may be in them
        if (!kSigmoid) sum_exactly();
        const float least = of_two ? two : one;
        const float from = least - tolerance(least);
        uint64_t look = 0;
#pragma unroll
        for (int j = 0; j < kPer; j++) look |= static_cast<uint64_t>(there(j) && v[j] >= from) << j;
        double exact_one = -INFINITY, exact_two = -INFINITY;
        while (__ballot(look != 0)) {
          if (look) {
            const int e = base + at_of(__ffsll(static_cast<unsigned long long>(look)) - 1);
            const double c = exact_score(logit_at<T>(row, e)) + (approximate ? static_cast<double>(a.bias[e]) : 0.0);
            exact_two = fmax(exact_two, fmin(exact_one, c));
            exact_one = fmax(exact_one, c);
            look &= look - 1;
          }
        }
        for (int by = 1; by < group_lanes; by *= 2) {
          const double other_one = __shfl_xor(exact_one, by, kLanes), other_two = __shfl_xor(exact_two, by, kLanes);
          exact_two = fmax(fmax(exact_two, other_two), fmin(exact_one, other_one));
          exact_one = fmax(exact_one, other_one);
        }
        pick(in_group ? rank_of(of_two ? exact_one + exact_two : exact_one) : uint64_t{0});
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; j++) key[j] = taken ? key[j] : 0;
  }

  // The lane's largest keys, the largest first: a choice takes one off, and only a lane that has given all of them goes
  // through its experts again.
  constexpr int kTop = kPer < 3 ? kPer : 3;
  uint32_t top[kTop];
  auto look = [&](auto all, uint32_t below) {   // of all keys, or those below
#pragma unroll
    for (int i = 0; i < kTop; i++) top[i] = 0;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const uint32_t k = decltype(all)::value || key[j] < below ? key[j] : 0;
#pragma unroll
      for (int i = kTop - 1; i > 0; i--) top[i] = max(min(top[i - 1], top[i]), min(max(top[i - 1], top[i]), k));   // the one in the middle
      top[0] = max(top[0], k);
    }
  };
  look(std::true_type(), 0);
  auto slack = [&](float c) { return tolerance(c) + kPer * 0x1p-22f * fabsf(c); };   // with what the keys leave out
  // Whether those of a rank are equal, not only near each other: of equal logits and biases, and all others clear of them.
  auto equal_ones = [&](uint32_t rank) {
    uint64_t left = 0;
    uint32_t below = 0, above = ~0u;
#pragma unroll
    for (int j = 0; j < kPer; j++) {
      const uint32_t k = key[j] & ~kIndex;
      left |= static_cast<uint64_t>(k == rank) << j;
      if (approximate) {
        below = max(below, k < rank ? k : 0u);
        above = min(above, k > rank ? k : ~0u);
      }
    }
    uint32_t most_l = 0, least_l = ~0u, most_b = 0, least_b = ~0u;
    while (__ballot(left != 0)) {
      if (left) {
        const int e = base + at_of(__ffsll(static_cast<unsigned long long>(left)) - 1);
        const uint32_t l = rank32(logit_at<T>(row, e)), c = approximate ? rank32(a.bias[e]) : 0;
        most_l = max(most_l, l), least_l = min(least_l, l);
        most_b = max(most_b, c), least_b = min(least_b, c);
        left &= left - 1;
      }
    }
    bool equal = largest_over<kLanes>(most_l) == smallest_over<kLanes>(least_l);
    if (approximate) {
      const float kept = value32(rank), far = slack(kept);
      below = largest_over<kLanes>(below), above = smallest_over<kLanes>(above);
      equal &= (below == 0 || value32(below) < kept - far) && (above == ~0u || value32(above) > kept + far);
      most_b = largest_over<kLanes>(most_b), least_b = smallest_over<kLanes>(least_b);
      equal &= most_b == least_b;
    }
    return equal;
  };
  // places[i] is the i-th found, of a rank the lower first; behind top_k as long as the next may belong before it
  int given = 0;
  auto take = [&](int i, uint32_t m, bool more) {
    const uint32_t best = top[0], e = static_cast<uint32_t>(base + at_of(static_cast<int>(kIndex - (best & kIndex))));
    bool mine = (best ^ m) <= kIndex;   // (of a token that has none left all of them)
    if (__popcll(__ballot(mine)) != 64 / kLanes) {
      const uint32_t lowest = smallest_over<kLanes>(mine ? e : ~0u);
      mine &= e == lowest;
    }
    if (mine) {
      if (more) places[i] = static_cast<uint16_t>(e);
#pragma unroll
      for (int k = 0; k < kTop; k++) top[k] = k + 1 < kTop ? top[k + 1] : 0;
      given++;
    }
    if (kTop < kPer && __ballot(mine && given == kTop)) {
      if (mine && given == kTop) {
        look(std::false_type(), best);
        given = 0;
      }
    }
  };
  uint32_t m = 0;
#pragma unroll 1
  for (int i = 0; i < a.top_k; i++) {
    m = largest_over<kLanes>(top[0]);
    take(i, m, true);
  }
  int found = a.top_k;
  const uint32_t least = m & ~kIndex;
  const float near = value32(least) - slack(value32(least));
  auto may_belong = [&] { return m != 0 && (approximate ? !(value32(m & ~kIndex) < near) : (m & ~kIndex) == least); };
  m = largest_over<kLanes>(top[0]);
  if (__ballot(may_belong())) {
    const bool settled = equal_ones(least);
#pragma unroll 1
    for (int i = a.top_k; i < kLanes; i++) {
      const bool more = !settled && may_belong();
      if (!__ballot(more)) break;
      take(i, m, more);
      if (more) found = i + 1;
      odd |= i == kLanes - 1;
      m = largest_over<kLanes>(top[0]);
    }
  }
  sub1::wave_lds_fence();

  // in 64 bits: scores of those found, their order
  const bool has = lane < found;
  const int mine = has ? min(static_cast<int>(places[lane]), a.experts - 1) : 0;   // (where there is something odd nothing may be found)
  const float l = logit_at<T>(row, mine);
  double score = exact_score(l);
  int place = 0;
  for (int again = 0; again < 2; again++) {
    const double c = approximate ? score + a.bias[mine] : static_cast<double>(l);
    // they are in order but where they were told apart by less than the keys hold
    const double after = __shfl(c, lane + 1, kLanes);
    const int index_after = __shfl(mine, lane + 1, kLanes);
    bool close = lane + 1 < found && fabs(c - after) < 0x1p-20 * largest_score;   // (the sum under the scores is of those in 32 bits)
    place = lane;
    if (__ballot(lane + 1 < found && !(c > after || (c == after && mine < index_after)))) {
      place = 0;
      for (int i = 0; i < kLanes; i++) {
        if (!__ballot(i < found)) break;
        const double other = __shfl(c, i, kLanes);
        const int at = __shfl(mine, i, kLanes);
        if (i < found && i != lane) {
          place += other > c || (other == c && at < mine);
          close |= has && fabs(other - c) < 0x1p-20 * largest_score;
        }
      }
    }
    if (again || kSigmoid || !approximate || !__ballot(close && !odd)) break;
    sum_exactly();
    score = exact_score(l);
  }
  const uint64_t odds = __ballot(odd) >> (threadIdx.x & (64 - kLanes));   // of this token's lanes, from bit 0 on
  if (kLanes == 64 ? odds != 0 : (odds & 0xffff) != 0) return false;
  const bool kept = has && place < a.top_k;
  double share = kept ? score : 0.0;
  if (a.normalize) {
    const double total = sum_over<kLanes>(share);
    if (total != 0) share /= total;
  }
  if (kept) store_choice(a, token, place, share, mine);
  return true;
}

template <class T, int kLanes, int kPer, bool kSigmoid, bool kBias>
__global__ __launch_bounds__(256) void route_quick_kernel(const RouteArgs a) {
  constexpr int kTokens = 64 / kLanes;   // of a wavefront
  const int64_t first = (blockIdx.x * int64_t{4} + (threadIdx.x >> 6)) * kTokens;
  if (first >= a.tokens) return;
  const int64_t token = first + (threadIdx.x & 63) / kLanes;
  // tokens that are not there repeat the last
  const uint64_t done = __ballot(route_quickly<T, kLanes, kPer, kSigmoid, kBias>(a, token < a.tokens ? token : a.tokens - 1));
  if (done == ~uint64_t{0}) return;
  for (int i = 0; i < kTokens && first + i < a.tokens; i++)
    if (!(done >> (i * kLanes) & 1)) route_exactly<T>(a, first + i);
}

template <class T, int kLanes, int kPer>
void launch_quick(const RouteArgs &a, hipStream_t s) {
  constexpr int kTokens = 4 * 64 / kLanes;
  const unsigned grid = static_cast<unsigned>((a.tokens + kTokens - 1) / kTokens);
  if (a.sigmoid) {
    if (a.bias) route_quick_kernel<T, kLanes, kPer, true, true><<<grid, 256, 0, s>>>(a);
    else route_quick_kernel<T, kLanes, kPer, true, false><<<grid, 256, 0, s>>>(a);
  } else {
    if (a.bias) route_quick_kernel<T, kLanes, kPer, false, true><<<grid, 256, 0, s>>>(a);
    else route_quick_kernel<T, kLanes, kPer, false, false><<<grid, 256, 0, s>>>(a);
  }
}

template <class T>
int launch_route(RouteArgs a, hipStream_t s) {
  a.group_bits = 0;
  while (1 << a.group_bits < a.groups) a.group_bits++;
  // experts a lane, with 16 or 64 lanes a token
  auto per = [&](int lanes) {
    const int of_group = lanes >> a.group_bits;
    return of_group ? (a.experts / a.groups + of_group - 1) / of_group : 1 << 30;
  };
  // A wavefront for four tokens where there are several for every SIMD, else for one (us in a graph: 8192 tokens' 8 of
  // 256 in groups, a bias, 9.1 and 12.3; 8 of 512, softmax 8.9 and 10.8; 1 of 128 4.1 and 5.6; 3000 tokens 7.3 and 7.4,
  // 7.2 and 6.2, 3.7 and 4.0; 4096 tokens' 8 of 512 7.5 both; 2048 tokens' 7.1 and 6.0, 7.2 and 5.4, 3.7 and 3.6).
  const int per16 = per(16), per64 = per(64);
  if (a.tokens > (per16 <= 16 ? 2500 : 4096) && per16 <= 32 && a.top_k <= 12) {
    sub1::note_kernel("route_quick_kernel, 16 lanes a token");
    if (per16 <= 1) launch_quick<T, 16, 1>(a, s);
    else if (per16 <= 2) launch_quick<T, 16, 2>(a, s);
    else if (per16 <= 4) launch_quick<T, 16, 4>(a, s);
    else if (per16 <= 8) launch_quick<T, 16, 8>(a, s);
    else if (per16 <= 16) launch_quick<T, 16, 16>(a, s);
    else launch_quick<T, 16, 32>(a, s);
  } else if (per64 <= 64 && a.top_k <= 56) {
    sub1::note_kernel("route_quick_kernel, 64 lanes a token");
    if (per64 <= 1) launch_quick<T, 64, 1>(a, s);
    else if (per64 <= 2) launch_quick<T, 64, 2>(a, s);
    else if (per64 <= 4) launch_quick<T, 64, 4>(a, s);
    else if (per64 <= 8) launch_quick<T, 64, 8>(a, s);
    else if (per64 <= 16) launch_quick<T, 64, 16>(a, s);
    else if (per64 <= 32) launch_quick<T, 64, 32>(a, s);
    else launch_quick<T, 64, 64>(a, s);
  } else {
    sub1::note_kernel("route_exact_kernel");
    route_exact_kernel<T><<<static_cast<unsigned>((a.tokens + 3) / 4), 256, 0, s>>>(a);
  }
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

// Eight values of a token a thread; fp32 sums, in the order of the token's places, the residual last.  Bound by HBM:
// 8192 tokens' four of 2080 in bf16 with a residual 36.5 us, 5.6 TB/s.
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
                    r.groups, r.top_groups, r.group_mark, r.scores == SUB1_ROUTE_SIGMOID, r.normalize != 0, index_bytes == 8, 0, r.scale};
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
