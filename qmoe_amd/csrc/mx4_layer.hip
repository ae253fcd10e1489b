// A whole sparse MLP for a few tokens, its experts' matrices in the microscaled 4-bit format:
//   logits = x R^T, the top_k experts of each token, p = softmax over all experts at those,
//   h = bf16(relu(wi_e x)), y = sum over them of p wo_e h.
#include "mx4.h"

using namespace mx4;
using sub1::fail;
using sub1::misaligned;

namespace {

constexpr int kTile = 16;   // tokens of an expert that its rows are multiplied with at once

struct LayerArgs {
  const void *router;
  const uint8_t *wi_codes, *wi_scales, *wo_codes, *wo_scales;
  const uint16_t *x;
  uint16_t *y;
  float *logits;
  int64_t *index;
  int tokens, length, experts, d_model, d_ff, top_k, normalize, capacity;
  // the scratch memory's parts
  int32_t *tiles;      // [0]: how many; from 4 on (expert, first pair, pairs, 0) of each
  int32_t *pairs;      // token * top_k + place, in the order of their experts, those that no expert takes left out
  int32_t *chosen;     // the experts of the tokens' places
  float *p;            // [tokens * top_k], their shares, negative where the token keeps its input
  uint16_t *h;         // bf16 [tokens * top_k, d_ff up to a whole block]
  float *out;          // [tokens * top_k, d_model]
};

// ----------------------------------------------------------------- the router ---

__device__ __forceinline__ void load4(const float *row, int first, int width, float (&v)[4]) {
  if (first + 4 <= width) {
    __builtin_memcpy(v, row + first, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = first + i < width ? row[first + i] : 0.0f;
  }
}
__device__ __forceinline__ void load4(const uint16_t *row, int first, int width, float (&v)[4]) {
  if (first + 4 <= width) {
    uint32_t two[2];
    __builtin_memcpy(two, row + first, 8);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = __uint_as_float(i & 1 ? two[i / 2] & 0xffff0000u : two[i / 2] << 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = first + i < width ? sub1::bf16_to_f32(row[first + i]) : 0.0f;
  }
}

__device__ __forceinline__ double wave_sum(double v) {   // in lane 63
  auto add = [&](auto control, auto rows) {
    constexpr int kControl = decltype(control)::value, kMask = decltype(rows)::value;
    const unsigned long long u = __double_as_longlong(v);
    const uint32_t low = sub1::dpp_or_zero<kControl, kMask>(static_cast<int>(u));
    const uint32_t high = sub1::dpp_or_zero<kControl, kMask>(static_cast<int>(u >> 32));
    v += __longlong_as_double(static_cast<unsigned long long>(high) << 32 | low);
  };
  add(std::integral_constant<int, sub1::kDppRowShr1>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr2>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr4>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppRowShr8>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, sub1::kDppBcast15>{}, std::integral_constant<int, 0xa>{});
  add(std::integral_constant<int, sub1::kDppBcast31>{}, std::integral_constant<int, 0xc>{});
  return v;
}

// kExperts by kTokens a workgroup, whose four wavefronts share a row's length, 256 values at a time, or (kShare false) a
// wavefront, where there are enough of them.  Sums in 64 bits, in which the products are exact: which of two close
// logits is the larger then follows from the values, not from the order of the sum.
template <class R, int kExperts, int kTokens, bool kShare>
__global__ __launch_bounds__(256) void mx4_logits_kernel(const LayerArgs a) {
  __shared__ double parts[4][kExperts * kTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int expert0 = (kShare ? blockIdx.x : blockIdx.x * 4 + wave) * kExperts, token0 = blockIdx.y * kTokens;
  const R *row[kExperts];
  const uint16_t *x[kTokens];
#pragma unroll
  for (int e = 0; e < kExperts; e++)
    row[e] = static_cast<const R *>(a.router) + static_cast<int64_t>(min(expert0 + e, a.experts - 1)) * a.d_model;
#pragma unroll
  for (int n = 0; n < kTokens; n++) x[n] = a.x + static_cast<int64_t>(min(token0 + n, a.tokens - 1)) * a.d_model;
  double sum[kExperts][kTokens];
#pragma unroll
  for (int e = 0; e < kExperts; e++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) sum[e][n] = 0;
  auto add = [&](int first) {
    float r[kExperts][4], v[kTokens][4];
#pragma unroll
    for (int e = 0; e < kExperts; e++) load4(row[e], first, a.d_model, r[e]);
#pragma unroll
    for (int n = 0; n < kTokens; n++) load4(x[n], first, a.d_model, v[n]);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int e = 0; e < kExperts; e++)
#pragma unroll
        for (int n = 0; n < kTokens; n++)
          sum[e][n] = fma(static_cast<double>(r[e][i]), static_cast<double>(v[n][i]), sum[e][n]);
  };
  int k = kShare ? wave * 256 : 0;
#pragma unroll 2
  for (; k + 256 <= a.d_model; k += kShare ? 1024 : 256) {
    __builtin_assume(k + 4 * lane + 4 <= a.d_model);
    add(k + 4 * lane);
  }
  if (k < a.d_model) add(k + 4 * lane);
#pragma unroll
  for (int e = 0; e < kExperts; e++)
#pragma unroll
    for (int n = 0; n < kTokens; n++) {
      const double all = wave_sum(sum[e][n]);
      if (kShare) {
        if (lane == 63) parts[wave][e * kTokens + n] = all;
      } else if (lane == 63 && expert0 + e < a.experts && token0 + n < a.tokens) {
        a.logits[static_cast<int64_t>(token0 + n) * a.experts + expert0 + e] = static_cast<float>(all);
      }
    }
  if (!kShare) return;
  __syncthreads();
  if (threadIdx.x < kExperts * kTokens) {
    const int i = threadIdx.x, expert = expert0 + i / kTokens, token = token0 + i % kTokens;
    if (expert < a.experts && token < a.tokens)
      a.logits[static_cast<int64_t>(token) * a.experts + expert] =
          static_cast<float>(((parts[0][i] + parts[1][i]) + parts[2][i]) + parts[3][i]);
  }
}

// ------------------------------------------------------------ which experts ---

// Logits in the order in which experts are taken, as whole numbers: larger first, those that are no numbers
// last (0); of equal ones the expert of the lower index comes first.
__device__ __forceinline__ uint32_t rank_of(float logit) {
  const uint32_t bits = __float_as_uint(logit + 0.0f);   // -0 is 0
  return logit != logit ? 0u : bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {   // in all lanes
  auto most = [&](auto control, auto rows) {
    v = max(v, static_cast<uint32_t>(sub1::dpp_or_zero<decltype(control)::value, decltype(rows)::value>(static_cast<int>(v))));
  };
  most(std::integral_constant<int, sub1::kDppRowShr1>{}, std::integral_constant<int, 0xf>{});
  most(std::integral_constant<int, sub1::kDppRowShr2>{}, std::integral_constant<int, 0xf>{});
  most(std::integral_constant<int, sub1::kDppRowShr4>{}, std::integral_constant<int, 0xf>{});
  most(std::integral_constant<int, sub1::kDppRowShr8>{}, std::integral_constant<int, 0xf>{});
  most(std::integral_constant<int, sub1::kDppBcast15>{}, std::integral_constant<int, 0xa>{});
  most(std::integral_constant<int, sub1::kDppBcast31>{}, std::integral_constant<int, 0xc>{});
  return __builtin_amdgcn_readlane(v, 63);
}

struct Choice {
  uint32_t rank;
  int expert;
};
constexpr Choice kNone = {0xffffffffu, -1};   // before the first (no logit has this rank)

// A wavefront's token's next expert behind `last`.
__device__ __forceinline__ Choice next_choice(const float *logits, int experts, Choice last) {
  const int lane = threadIdx.x & 63;
  Choice best = {0, -1};
  auto look = [&](float logit, int e) {
    const uint32_t rank = rank_of(logit);
    const bool left = rank < last.rank || (rank == last.rank && e > last.expert);
    if (e < experts && left && (best.expert < 0 || rank > best.rank)) best = {rank, e};
  };
  for (int first = lane; first < experts; first += 256) {   // four loads on their way at once
    float logit[4];
#pragma unroll
    for (int i = 0; i < 4; i++) logit[i] = logits[min(first + 64 * i, experts - 1)];
#pragma unroll
    for (int i = 0; i < 4; i++) look(logit[i], first + 64 * i);
  }
  const uint32_t rank = wave_max(best.expert < 0 ? 0 : best.rank);
  return {rank, static_cast<int>(~wave_max(best.expert < 0 || best.rank != rank ? 0 : ~static_cast<uint32_t>(best.expert)))};
}

// A wavefront's token's experts and their shares: to index, and (expert, share) of place j to put(j, ..).
template <class Put>
__device__ __forceinline__ void choose(const LayerArgs &a, int token, Put put) {
  const int lane = threadIdx.x & 63;
  const float *logits = a.logits + static_cast<int64_t>(token) * a.experts;
  Choice c = kNone;
  float most = 0, sum = 0, taken = 0, mine = 0;
  int expert = 0;
  for (int j = 0; j < a.top_k; j++) {
    c = next_choice(logits, a.experts, c);
    if (j == 0) {
      most = logits[c.expert];
      for (int first = lane; first < a.experts; first += 256) {
        float logit[4];
#pragma unroll
        for (int i = 0; i < 4; i++) logit[i] = logits[min(first + 64 * i, a.experts - 1)];
#pragma unroll
        for (int i = 0; i < 4; i++) sum += first + 64 * i < a.experts ? expf(logit[i] - most) : 0.0f;
      }
      sum = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(lanes_sum<64>(sum)), 63));
    }
    const float p = expf(logits[c.expert] - most) / sum;
    taken += p;
    if (lane == j) mine = p, expert = c.expert;
  }
  if (a.normalize) mine /= taken;
  // no share is negative, and one that is no number has no sign either: a sign marks a token that keeps its input
  mine = __uint_as_float(__float_as_uint(mine) & 0x7fffffffu);
  if (lane < a.top_k) {
    a.index[static_cast<int64_t>(token) * a.top_k + lane] = expert;
    put(lane, expert, mine);
  }
}

constexpr int kPlanThreads = 1024;

// One workgroup: every token's experts and their shares, and the pairs of token and expert in the order of
// the experts, up to kTile of one expert a tile.
__global__ __launch_bounds__(kPlanThreads) void mx4_plan_kernel(const LayerArgs a) {
  __shared__ int32_t expert_of[SUB1_MX4_LAYER_TOKENS * SUB1_MX4_LAYER_TOP_K];   // -1: none takes the pair
  __shared__ int32_t count[SUB1_MX4_LAYER_EXPERTS];
  __shared__ int32_t pairs_before[kPlanThreads / 64], tiles_before[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int pairs = a.tokens * a.top_k;
  for (int e = tid; e < a.experts; e += kPlanThreads) count[e] = 0;
  for (int t = wave; t < a.tokens; t += kPlanThreads / 64)
    choose(a, t, [&](int j, int expert, float p) {
      expert_of[t * a.top_k + j] = expert;
      a.p[t * a.top_k + j] = p;
    });
  __syncthreads();

  // a token beyond its expert's capacity in its sequence (with one expert a token)
  bool full = false;
  if (a.capacity && tid < a.tokens) {
    int before = 0;
    for (int t = tid - tid % a.length; t < tid; t++) before += expert_of[t] == expert_of[tid];
    full = before >= a.capacity;
  }
  __syncthreads();
  if (full) {
    expert_of[tid] = -1;
    a.p[tid] = -a.p[tid];
  }
  __syncthreads();
  for (int i = tid; i < pairs; i += kPlanThreads)
    if (expert_of[i] >= 0) atomicAdd(&count[expert_of[i]], 1);
  __syncthreads();

  // sums over the experts before, of pairs and of tiles; a thread has kMine experts
  constexpr int kMine = SUB1_MX4_LAYER_EXPERTS / kPlanThreads;
  int my_pairs = 0, my_tiles = 0;
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    const int e = tid * kMine + i;
    if (e < a.experts) my_pairs += count[e], my_tiles += (count[e] + kTile - 1) / kTile;
  }
  int upto_pairs = sub1::wave_prefix_sum(my_pairs), upto_tiles = sub1::wave_prefix_sum(my_tiles);
  if (lane == 63) pairs_before[wave] = upto_pairs, tiles_before[wave] = upto_tiles;
  __syncthreads();
  int first_pair = upto_pairs - my_pairs, first_tile = upto_tiles - my_tiles, all_tiles = 0;
  for (int w = 0; w < kPlanThreads / 64; w++) {
    if (w < wave) first_pair += pairs_before[w], first_tile += tiles_before[w];
    all_tiles += tiles_before[w];
  }
  if (tid == 0) a.tiles[0] = all_tiles;
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    const int e = tid * kMine + i;
    if (e >= a.experts) break;
    const int n = count[e];
    count[e] = first_pair;   // from here on where the expert's pairs begin (read by its own thread so far)
    for (int k = 0; k < n; k += kTile, first_tile++) {
      int32_t *tile = a.tiles + 4 + 4 * first_tile;
      tile[0] = e, tile[1] = first_pair + k, tile[2] = min(n - k, kTile), tile[3] = 0;
    }
    first_pair += n;
  }
  __syncthreads();
  for (int i = tid; i < pairs; i += kPlanThreads) {
    const int e = expert_of[i];
    if (e < 0) continue;
    int before = 0;
    for (int k = 0; k < i; k++) before += expert_of[k] == e;
    a.pairs[count[e] + before] = i;
  }
}

// ----------------------------------------------------------------- the experts ---

struct Tile {
  int expert, first, pairs;
};
__device__ __forceinline__ bool tile_of(const LayerArgs &a, int i, Tile &t) {
  if (i >= a.tiles[0]) return false;
  t = {a.tiles[4 + 4 * i], a.tiles[4 + 4 * i + 1], a.tiles[4 + 4 * i + 2]};
  return true;
}

__device__ __forceinline__ int h_width(const LayerArgs &a) { return blocks_of(a.d_ff) * kBlock; }

// The last row of workgroups, where a capacity may leave tokens with their input, writes those tokens' y.
__device__ __forceinline__ void keep_inputs(const LayerArgs &a) {
  for (int t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const float p = a.p[t];
    if (!(__float_as_uint(p) >> 31)) continue;
    for (int d = threadIdx.x; d < a.d_model; d += 64 * kFewWaves) {
      const int64_t at = static_cast<int64_t>(t) * a.d_model + d;
      a.y[at] = static_cast<uint16_t>(two_bf16(-p * sub1::bf16_to_f32(a.x[at]), 0));
    }
  }
}

__global__ __launch_bounds__(64 * kFewWaves) void mx4_wi_kernel(const LayerArgs a) {
  __shared__ f32x4 lds[kFewLds<1, 1>];
  if (a.capacity && blockIdx.y == gridDim.y - 1) {
    keep_inputs(a);
    return;
  }
  Tile t;
  if (!tile_of(a, blockIdx.y, t)) return;
  const int lane = threadIdx.x & 63, row0 = blockIdx.x * 16, width = h_width(a), mine = lane & 15;
  const int64_t pair = mine < t.pairs ? a.pairs[t.first + mine] : -1;
  uint16_t *h = a.h + pair * width + row0 + 4 * (lane >> 4);
  FewSums<1, 1> sums;
  if (row0 < a.d_ff) {
    const uint16_t *x[1] = {a.x + (pair >= 0 ? pair / a.top_k : 0) * a.d_model};
    const int64_t row = static_cast<int64_t>(t.expert) * a.d_ff + row0, blocks = blocks_of(a.d_model);
    few_products<1, 1>(sums, a.wi_codes + row * blocks * kBlockBytes, a.wi_scales + row * blocks, a.d_ff - row0,
                       a.d_model, x);
    few_join<1, 1>(sums, lds, [&](int, int, f32x4 sum) {
      if (pair < 0) return;
      // h goes to the matrix cores as bf16, as between two layers of a model in that type; what is no
      // number stays none (a comparison with it is false); behind the last row there are zeros
#pragma unroll
      for (int i = 0; i < 4; i++) sum[i] = row0 + 4 * (lane >> 4) + i >= a.d_ff || sum[i] < 0 ? 0.0f : sum[i];
      const uint32_t two[2] = {two_bf16(sum[0], sum[1]), two_bf16(sum[2], sum[3])};
      __builtin_memcpy(h, two, 8);
    });
  } else if (threadIdx.x < 64 && pair >= 0) {
    const uint32_t two[2] = {0, 0};
    __builtin_memcpy(h, two, 8);
  }
}

// With one expert a token the product, times the token's share, is its y; else it waits for the others.
template <bool kOnly>
__global__ __launch_bounds__(64 * kFewWaves) void mx4_wo_kernel(const LayerArgs a) {
  __shared__ f32x4 lds[kFewLds<1, 1>];
  Tile t;
  if (!tile_of(a, blockIdx.y, t)) return;
  const int lane = threadIdx.x & 63, row0 = blockIdx.x * 16, width = h_width(a), mine = lane & 15;
  const int64_t pair = mine < t.pairs ? a.pairs[t.first + mine] : -1;
  const uint16_t *x[1] = {a.h + (pair >= 0 ? pair : a.pairs[t.first]) * width};
  const int64_t row = static_cast<int64_t>(t.expert) * a.d_model + row0, blocks = blocks_of(a.d_ff);
  FewSums<1, 1> sums;
  few_products<1, 1>(sums, a.wo_codes + row * blocks * kBlockBytes, a.wo_scales + row * blocks, a.d_model - row0, width,
                     x);
  few_join<1, 1>(sums, lds, [&](int, int, f32x4 sum) {
    if (pair < 0) return;
    const int row = row0 + 4 * (lane >> 4);
    const float p = kOnly ? a.p[pair] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (row + i >= a.d_model) break;
      if (kOnly)
        a.y[pair * a.d_model + row + i] = static_cast<uint16_t>(two_bf16(p * sum[i], 0));
      else
        a.out[pair * a.d_model + row + i] = sum[i];
    }
  });
}

__global__ __launch_bounds__(256) void mx4_combine_kernel(const LayerArgs a) {
  const int d = blockIdx.x * 256 + threadIdx.x;
  const int64_t t = blockIdx.y;
  if (d >= a.d_model) return;
  float sum = 0;
  for (int j = 0; j < a.top_k; j++) sum += a.p[t * a.top_k + j] * a.out[(t * a.top_k + j) * a.d_model + d];
  a.y[t * a.d_model + d] = static_cast<uint16_t>(two_bf16(sum, 0));
}

// ---- a token at a time, each with its own experts' rows ----
//
// Where few tokens share an expert, grouping them costs more than it saves: a workgroup finds its token's expert by
// itself and takes the token through kRows rows a wavefront, and the workgroups of wo add the token's experts up.
// Three launches, or four, with nothing between workgroups of one.

// A launch of its own for many experts, whose logits are looked through once a token, and where an expert's capacity
// makes the choice one among a sequence's tokens: a workgroup a sequence, a wavefront a token.
constexpr int kChooseWaves = 16;
__global__ __launch_bounds__(64 * kChooseWaves) void mx4_choose_kernel(const LayerArgs a) {
  __shared__ int32_t expert_of[SUB1_MX4_LAYER_TOKENS];
  __shared__ float p_of[SUB1_MX4_LAYER_TOKENS];
  const int first = blockIdx.x * a.length, waves = blockDim.x >> 6;
  for (int i = threadIdx.x >> 6; i < a.length; i += waves)
    choose(a, first + i, [&](int j, int expert, float p) {
      a.chosen[(first + i) * a.top_k + j] = expert;
      a.p[(first + i) * a.top_k + j] = p;
      if (a.capacity) expert_of[i] = expert, p_of[i] = p;
    });
  if (!a.capacity) return;
  __syncthreads();
  const int mine = threadIdx.x;
  if (mine >= a.length) return;
  int before = 0;
  for (int i = 0; i < mine; i++) before += expert_of[i] == expert_of[mine];
  if (before >= a.capacity) a.p[first + mine] = -p_of[mine];
}
static_assert(SUB1_MX4_LAYER_TOKENS <= 64 * kChooseWaves, "a thread a token");

template <int kRows, int kLanes, bool kChosen>
__global__ __launch_bounds__(64 * kOneWaves) void mx4_one_wi_kernel(const LayerArgs a) {
  extern __shared__ u32x4 one_lds[];
  const int pair = blockIdx.y, token = pair / a.top_k, place = pair - token * a.top_k, width = h_width(a);
  stage_one<kLanes>(one_lds, a.x + static_cast<int64_t>(token) * a.d_model, a.d_model);
  int expert;
  if (kChosen) {
    if (a.capacity && __float_as_uint(a.p[pair]) >> 31) return;   // (the whole workgroup: no expert takes it)
    expert = a.chosen[pair];
  } else {
    const float *logits = a.logits + static_cast<int64_t>(token) * a.experts;
    Choice c = kNone;
    for (int j = 0; j <= place; j++) c = next_choice(logits, a.experts, c);
    expert = c.expert;
    if (blockIdx.x == 0 && place == 0 && threadIdx.x < 64)   // for wo, and for the caller
      choose(a, token, [&](int j, int e, float p) {
        a.chosen[pair + j] = e;
        a.p[pair + j] = p;
      });
  }
  const int blocks = blocks_of(a.d_model), row0 = blockIdx.x * kRows * kOneRows<kLanes> + threadIdx.x / kLanes;
  auto first_of = [&](int r) {   // rows that are not there: the last again
    return (static_cast<int64_t>(expert) * a.d_ff + min(row0 + r * kOneRows<kLanes>, a.d_ff - 1)) * blocks;
  };
  OneFirst next = one_block(a.wi_codes, a.wi_scales, first_of(0), threadIdx.x % kLanes, blocks);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRows; r++) {
    const int row = row0 + r * kOneRows<kLanes>;
    // the next row's first blocks are on their way meanwhile (all rows' at once: more registers, 10 % longer)
    const OneFirst begin = next;
    if (r + 1 < kRows) next = one_block(a.wi_codes, a.wi_scales, first_of(r + 1), threadIdx.x % kLanes, blocks);
    const float sum = one_product<kLanes>(begin, a.wi_codes, a.wi_scales, first_of(r), blocks, one_lds);
    // (bf16 between the layers, and zeros behind the last row, as above)
    if (threadIdx.x % kLanes == kLanes - 1 && row < width)
      a.h[static_cast<int64_t>(pair) * width + row] = static_cast<uint16_t>(two_bf16(row >= a.d_ff || sum < 0 ? 0.0f : sum, 0));
  }
}

template <int kRows, int kLanes>
__global__ __launch_bounds__(64 * kOneWaves) void mx4_one_wo_kernel(const LayerArgs a) {
  extern __shared__ u32x4 one_lds[];
  const int token = blockIdx.y, width = h_width(a), blocks = blocks_of(a.d_ff);
  float all[kRows];
#pragma unroll
  for (int r = 0; r < kRows; r++) all[r] = 0;
  for (int j = 0; j < a.top_k; j++) {
    const int pair = token * a.top_k + j;
    const float p = a.p[pair];
    if (a.capacity && __float_as_uint(p) >> 31) {   // no expert takes the token: its input, times its share
#pragma unroll
      for (int r = 0; r < kRows; r++) {
        const int row = (blockIdx.x * kRows + r) * kOneRows<kLanes> + threadIdx.x / kLanes;
        all[r] = -p * sub1::bf16_to_f32(a.x[static_cast<int64_t>(token) * a.d_model + min(row, a.d_model - 1)]);
      }
      break;   // (a capacity goes with one expert a token)
    }
    const int expert = a.chosen[pair];
    auto first_of = [&](int r) {
      const int row = (blockIdx.x * kRows + r) * kOneRows<kLanes> + threadIdx.x / kLanes;
      return (static_cast<int64_t>(expert) * a.d_model + min(row, a.d_model - 1)) * blocks;
    };
    OneFirst next = one_block(a.wo_codes, a.wo_scales, first_of(0), threadIdx.x % kLanes, blocks);
    if (j) __syncthreads();
    stage_one<kLanes>(one_lds, a.h + static_cast<int64_t>(pair) * width, width);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; r++) {
      const OneFirst begin = next;
      if (r + 1 < kRows) next = one_block(a.wo_codes, a.wo_scales, first_of(r + 1), threadIdx.x % kLanes, blocks);
      all[r] += p * one_product<kLanes>(begin, a.wo_codes, a.wo_scales, first_of(r), blocks, one_lds);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; r++) {
    const int row = (blockIdx.x * kRows + r) * kOneRows<kLanes> + threadIdx.x / kLanes;
    if (threadIdx.x % kLanes == kLanes - 1 && row < a.d_model)
      a.y[static_cast<int64_t>(token) * a.d_model + row] = static_cast<uint16_t>(two_bf16(all[r], 0));
  }
}

// ------------------------------------------------------------------- launching ---

template <class R>
int launch_logits(const LayerArgs &a, hipStream_t s) {
  const unsigned fours = (a.tokens + 3) / 4;
  if (a.tokens == 1)
    mx4_logits_kernel<R, 1, 1, true><<<a.experts, 256, 0, s>>>(a);
  else if (static_cast<int64_t>(a.experts) * a.tokens <= 8192)
    mx4_logits_kernel<R, 1, 4, true><<<dim3(a.experts, fours), 256, 0, s>>>(a);
  else
    mx4_logits_kernel<R, 4, 4, false><<<dim3((a.experts + 15) / 16, fours), 256, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

template <int kRows, int kLanes, bool kChosen>
int launch_one_wi(const LayerArgs &a, hipStream_t s) {
  constexpr int kAll = kRows * kOneRows<kLanes>;
  if (one_lds_bytes(a.d_model) > kPlainLds) HIP_TRY(sub1::allow_lds<kOneMostBytes>(mx4_one_wi_kernel<kRows, kLanes, kChosen>));
  mx4_one_wi_kernel<kRows, kLanes, kChosen>
      <<<dim3((blocks_of(a.d_ff) * kBlock + kAll - 1) / kAll, a.tokens * a.top_k), 64 * kOneWaves,
         one_lds_bytes(a.d_model), s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

template <int kRows, int kLanes>
int launch_one_wo(const LayerArgs &a, hipStream_t s) {
  constexpr int kAll = kRows * kOneRows<kLanes>;
  if (one_lds_bytes(a.d_ff) > kPlainLds) HIP_TRY(sub1::allow_lds<kOneMostBytes>(mx4_one_wo_kernel<kRows, kLanes>));
  mx4_one_wo_kernel<kRows, kLanes>
      <<<dim3((a.d_model + kAll - 1) / kAll, a.tokens), 64 * kOneWaves, one_lds_bytes(a.d_ff), s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}

// Rows a wavefront (or half one), by how many workgroups one each would make: more of them use a token that is in LDS
// already, fewer leave compute units idle (us of a call with 1 / 2 / 4 / 8 rows of wi: one token through 2080 x 6144,
// 384 workgroups, 12.0 / 12.5 / 14.3 / 17.7; three, 1152, 19.0 / 18.6 / 20.1 / 23.2; eight pairs through 1024 x 4096,
// 2048, 20.7 / 18.4 / 17.8 / 19.0; 26, 6656, 41.7 / 34.8 / 31.7 / 31.7; with 1 / 2 / 4 of wo, 260 workgroups,
// 12.3 / 12.6 / 14.5, 512, 21.6 / 21.6 / 24, 1664, 48 / 47 / 46).
template <int kLanes, bool kChosen>
int launch_wi(const LayerArgs &a, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(a.tokens) * a.top_k * ((a.d_ff + kOneRows<kLanes> - 1) / kOneRows<kLanes>);
  return n < 1000   ? launch_one_wi<1, kLanes, kChosen>(a, s)
         : n < 2000 ? launch_one_wi<2, kLanes, kChosen>(a, s)
         : n < 8000 ? launch_one_wi<4, kLanes, kChosen>(a, s)
                    : launch_one_wi<8, kLanes, kChosen>(a, s);
}
template <int kLanes>
int launch_wo(const LayerArgs &a, hipStream_t s) {
  const int64_t n = static_cast<int64_t>(a.tokens) * ((a.d_model + kOneRows<kLanes> - 1) / kOneRows<kLanes>);
  return n < 400 ? launch_one_wo<1, kLanes>(a, s) : n < 1500 ? launch_one_wo<2, kLanes>(a, s) : launch_one_wo<4, kLanes>(a, s);
}
template <bool kChosen>
int launch_ones(const LayerArgs &a, hipStream_t s) {
  const int64_t wi_rows = static_cast<int64_t>(a.tokens) * a.top_k * a.d_ff, wo_rows = static_cast<int64_t>(a.tokens) * a.d_model;
  const int rc = halves_pay(a.d_model, wi_rows) ? launch_wi<32, kChosen>(a, s) : launch_wi<64, kChosen>(a, s);
  if (rc) return rc;
  return halves_pay(a.d_ff, wo_rows) ? launch_wo<32>(a, s) : launch_wo<64>(a, s);
}

int most_tiles(const sub1_mx4_layer *l, int tokens) {
  const int pairs = tokens * l->top_k, taking = pairs < l->experts ? pairs : l->experts;
  return (pairs + (kTile - 1) * taking) / kTile;   // every expert's last tile may hold one
}

int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Parts {
  int64_t tiles, pairs, chosen, p, h, out, bytes;
};
Parts parts_of(const sub1_mx4_layer *l, int tokens) {
  const int64_t pairs = static_cast<int64_t>(tokens) * l->top_k;
  Parts at;
  at.tiles = 0;
  at.pairs = at.tiles + up(16 + 16 * static_cast<int64_t>(most_tiles(l, tokens)));
  at.chosen = at.pairs + up(4 * pairs);
  at.p = at.chosen + up(4 * pairs);
  at.h = at.p + up(4 * pairs);
  at.out = at.h + up(pairs * blocks_of(l->d_ff) * kBlock * 2);
  at.bytes = at.out + up(pairs * l->d_model * 4);
  return at;
}

int check_layer(const sub1_mx4_layer *l, int tokens, const char *who) {
  if (!l) return fail(SUB1_ERR_NULL, "%s: NULL layer", who);
  if (l->experts < 1 || l->experts > SUB1_MX4_LAYER_EXPERTS)
    return fail(SUB1_ERR_SHAPE, "%s: %d experts (1..%d)", who, l->experts, SUB1_MX4_LAYER_EXPERTS);
  if (l->d_model < 1 || l->d_model > SUB1_MX4_MAX_WIDTH || l->d_ff < 1 || l->d_ff > SUB1_MX4_MAX_WIDTH)
    return fail(SUB1_ERR_SHAPE, "%s: d_model %d d_ff %d (1..%d)", who, l->d_model, l->d_ff, SUB1_MX4_MAX_WIDTH);
  if (l->top_k < 1 || l->top_k > SUB1_MX4_LAYER_TOP_K || l->top_k > l->experts)
    return fail(SUB1_ERR_SHAPE, "%s: top_k %d of %d experts (1..%d)", who, l->top_k, l->experts, SUB1_MX4_LAYER_TOP_K);
  if (l->router_type != SUB1_MX4_BF16 && l->router_type != SUB1_MX4_FP32)
    return fail(SUB1_ERR_SHAPE, "%s: router_type %d (SUB1_MX4_BF16 or _FP32)", who, l->router_type);
  if (l->capacity < 0 || (l->capacity && l->top_k != 1))
    return fail(SUB1_ERR_SHAPE, "%s: capacity %d with top_k %d (a capacity goes with one expert a token)", who,
                l->capacity, l->top_k);
  if (tokens < 0 || tokens > SUB1_MX4_LAYER_TOKENS)
    return fail(SUB1_ERR_SHAPE, "%s: tokens %d outside 0..%d", who, tokens, SUB1_MX4_LAYER_TOKENS);
  return SUB1_OK;
}

}  // namespace

// ================================================================ C ABI =====

extern "C" int64_t sub1_mx4_layer_scratch_bytes(const sub1_mx4_layer *layer, int tokens) {
  if (check_layer(layer, tokens, "sub1_mx4_layer_scratch_bytes")) return 0;
  return parts_of(layer, tokens).bytes;
}

extern "C" int sub1_mx4_layer_forward(const sub1_mx4_layer *layer, const void *x, int tokens, int length, void *y,
                                      float *logits, int64_t *index, void *scratch, int64_t scratch_bytes,
                                      void *stream) {
  const char *who = "sub1_mx4_layer_forward";
  int rc = check_layer(layer, tokens, who);
  if (rc || tokens == 0) return rc;
  if (length < 1 || tokens % length)
    return fail(SUB1_ERR_SHAPE, "%s: %d tokens are no whole sequences of %d", who, tokens, length);
  if (!layer->router || !layer->wi_codes || !layer->wi_scales || !layer->wo_codes || !layer->wo_scales || !x || !y ||
      !logits || !index || !scratch)
    return fail(SUB1_ERR_NULL, "%s: NULL argument", who);
  if (misaligned(layer->router, layer->router_type == SUB1_MX4_FP32 ? 4 : 2) || misaligned(layer->wi_codes, 16) ||
      misaligned(layer->wo_codes, 16) || misaligned(x, 2) || misaligned(y, 2) || misaligned(logits, 4) ||
      misaligned(index, 8) || misaligned(scratch, 256))
    return fail(SUB1_ERR_ALIGN, "%s: misaligned pointer", who);
  const Parts at = parts_of(layer, tokens);
  if (scratch_bytes < at.bytes)
    return fail(SUB1_ERR_SHAPE, "%s: scratch of %lld bytes, %lld needed", who, static_cast<long long>(scratch_bytes),
                static_cast<long long>(at.bytes));
  hipStream_t s = static_cast<hipStream_t>(stream);
  char *base = static_cast<char *>(scratch);
  // one that no sequence reaches is none: its choice would be a launch more (a token at a time), or workgroups that
  // look for tokens that keep their input
  const int capacity = layer->capacity < length ? layer->capacity : 0;
  LayerArgs a{layer->router, layer->wi_codes, layer->wi_scales, layer->wo_codes, layer->wo_scales,
              static_cast<const uint16_t *>(x), static_cast<uint16_t *>(y), logits, index, tokens, length,
              layer->experts, layer->d_model, layer->d_ff, layer->top_k, layer->normalize, capacity,
              reinterpret_cast<int32_t *>(base + at.tiles), reinterpret_cast<int32_t *>(base + at.pairs),
              reinterpret_cast<int32_t *>(base + at.chosen), reinterpret_cast<float *>(base + at.p),
              reinterpret_cast<uint16_t *>(base + at.h), reinterpret_cast<float *>(base + at.out)};
  rc = layer->router_type == SUB1_MX4_FP32 ? launch_logits<float>(a, s) : launch_logits<uint16_t>(a, s);
  if (rc) return rc;
  // A token at a time up to three pairs an expert (us, grouped by expert in brackets: one pair of 2080 x 6144 11.9 (18.4),
  // 26 over 128 experts of 1024 x 4096 32 (58), 128 over 64 91 (125), 32 over 8 31 (34), 64 over 8 50 (40); 64 over 32 of
  // 1000 x 2501 39 (52); 16 over 8 of 2080 x 6144 48 (47), 32 over 8 77 (58)).
  if (tokens * a.top_k <= 3 * a.experts) {
    sub1::note_kernel("mx4_one_wo_kernel");
    if (a.experts <= 256 && !a.capacity) return launch_ones<false>(a, s);
    mx4_choose_kernel<<<tokens / length, 64 * (length < kChooseWaves ? length : kChooseWaves), 0, s>>>(a);
    HIP_TRY(hipGetLastError());
    return launch_ones<true>(a, s);
  }
  mx4_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  const unsigned tiles = static_cast<unsigned>(most_tiles(layer, tokens));
  mx4_wi_kernel<<<dim3(blocks_of(a.d_ff) * 2, tiles + (a.capacity ? 1 : 0)), 64 * kFewWaves, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  sub1::note_kernel("mx4_wo_kernel");
  const dim3 wo((a.d_model + 15) / 16, tiles);
  if (a.top_k == 1) {
    mx4_wo_kernel<true><<<wo, 64 * kFewWaves, 0, s>>>(a);
    HIP_TRY(hipGetLastError());
    return SUB1_OK;
  }
  mx4_wo_kernel<false><<<wo, 64 * kFewWaves, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  mx4_combine_kernel<<<dim3((a.d_model + 255) / 256, tokens), 256, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}
