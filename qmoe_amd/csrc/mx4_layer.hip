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
  float *p;            // [tokens * top_k], negative where the token keeps its input
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

// A wavefront an expert, kTokens tokens at once.  Sums in 64 bits, in which the products are exact: which of
// two close logits is the larger then follows from the values, not from the order of the sum.
template <class R, int kTokens>
__global__ __launch_bounds__(256) void mx4_logits_kernel(const LayerArgs a) {
  const int lane = threadIdx.x & 63, expert = blockIdx.x * 4 + (threadIdx.x >> 6), token0 = blockIdx.y * kTokens;
  if (expert >= a.experts) return;
  const R *row = static_cast<const R *>(a.router) + static_cast<int64_t>(expert) * a.d_model;
  double sum[kTokens];
#pragma unroll
  for (int n = 0; n < kTokens; n++) sum[n] = 0;
  for (int k = 4 * lane; k < a.d_model; k += 256) {
    float r[4], v[4];
    load4(row, k, a.d_model, r);
#pragma unroll
    for (int n = 0; n < kTokens; n++) {
      if (token0 + n >= a.tokens) break;
      load4(a.x + static_cast<int64_t>(token0 + n) * a.d_model, k, a.d_model, v);
#pragma unroll
      for (int i = 0; i < 4; i++) sum[n] = fma(static_cast<double>(r[i]), static_cast<double>(v[i]), sum[n]);
    }
  }
#pragma unroll
  for (int n = 0; n < kTokens; n++) {
    for (int d = 32; d; d >>= 1) sum[n] += __shfl_xor(sum[n], d);
    if (lane == 0 && token0 + n < a.tokens)
      a.logits[static_cast<int64_t>(token0 + n) * a.experts + expert] = static_cast<float>(sum[n]);
  }
}

// ------------------------------------------------------------ which experts ---

// Logits in the order in which experts are taken: larger first, of equals the one of the lower index, those
// that are no numbers last.
__device__ __forceinline__ unsigned long long rank_of(float logit, int expert) {
  uint32_t bits = __float_as_uint(logit + 0.0f);   // -0 is 0
  bits = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  if (logit != logit) bits = 0;
  return static_cast<unsigned long long>(bits) << 32 | (0xffffffffu - static_cast<uint32_t>(expert));
}

__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
  for (int d = 32; d; d >>= 1) {
    const unsigned long long u = __shfl_xor(v, d);
    v = u > v ? u : v;
  }
  return v;
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

  for (int t = wave; t < a.tokens; t += kPlanThreads / 64) {
    const float *logits = a.logits + static_cast<int64_t>(t) * a.experts;
    float most = -__builtin_inff(), sum = 0;
    for (int e = lane; e < a.experts; e += 64) most = fmaxf(most, logits[e]);
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    for (int e = lane; e < a.experts; e += 64) sum += expf(logits[e] - most);
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
    unsigned long long last = ~0ull;
    float taken = 0, mine = 0;
    for (int j = 0; j < a.top_k; j++) {
      unsigned long long best = 0;
      for (int e = lane; e < a.experts; e += 64) {
        const unsigned long long r = rank_of(logits[e], e);
        if (r < last && r > best) best = r;
      }
      last = wave_max(best);
      const int e = static_cast<int>(0xffffffffu - static_cast<uint32_t>(last));
      const float p = expf(logits[e] - most) / sum;
      taken += p;
      if (lane == j) mine = p;
      if (lane == 0) {
        expert_of[t * a.top_k + j] = e;
        a.index[t * a.top_k + j] = e;
      }
    }
    if (lane < a.top_k) a.p[t * a.top_k + lane] = a.normalize ? mine / taken : mine;
  }
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

__global__ __launch_bounds__(64 * kFewWaves) void mx4_wi_kernel(const LayerArgs a) {
  __shared__ f32x4 lds[kFewLds<1, 1>];
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
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (row + i < a.d_model) a.out[pair * a.d_model + row + i] = sum[i];
  });
}

__global__ __launch_bounds__(256) void mx4_combine_kernel(const LayerArgs a) {
  const int d = blockIdx.x * 256 + threadIdx.x;
  const int64_t t = blockIdx.y;
  if (d >= a.d_model) return;
  float sum = 0;
  for (int j = 0; j < a.top_k; j++) {
    const int64_t pair = t * a.top_k + j;
    const float p = a.p[pair];
    sum += __float_as_uint(p) >> 31 ? -p * sub1::bf16_to_f32(a.x[t * a.d_model + d]) : p * a.out[pair * a.d_model + d];
  }
  a.y[t * a.d_model + d] = sub1::f32_to_bf16(sum);
}

// ------------------------------------------------------------------- launching ---

int most_tiles(const sub1_mx4_layer *l, int tokens) {
  const int pairs = tokens * l->top_k, taking = pairs < l->experts ? pairs : l->experts;
  return (pairs + (kTile - 1) * taking) / kTile;   // every expert's last tile may hold one
}

int64_t up(int64_t bytes) { return (bytes + 255) / 256 * 256; }

struct Parts {
  int64_t tiles, pairs, p, h, out, bytes;
};
Parts parts_of(const sub1_mx4_layer *l, int tokens) {
  const int64_t pairs = static_cast<int64_t>(tokens) * l->top_k;
  Parts at;
  at.tiles = 0;
  at.pairs = at.tiles + up(16 + 16 * static_cast<int64_t>(most_tiles(l, tokens)));
  at.p = at.pairs + up(4 * pairs);
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
  const int rc = check_layer(layer, tokens, who);
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
  LayerArgs a{layer->router, layer->wi_codes, layer->wi_scales, layer->wo_codes, layer->wo_scales,
              static_cast<const uint16_t *>(x), static_cast<uint16_t *>(y), logits, index, tokens, length,
              layer->experts, layer->d_model, layer->d_ff, layer->top_k, layer->normalize, layer->capacity,
              reinterpret_cast<int32_t *>(base + at.tiles), reinterpret_cast<int32_t *>(base + at.pairs),
              reinterpret_cast<float *>(base + at.p), reinterpret_cast<uint16_t *>(base + at.h),
              reinterpret_cast<float *>(base + at.out)};
  constexpr int kTokens = 4;
  const dim3 routers((a.experts + 3) / 4, (tokens + kTokens - 1) / kTokens);
  if (layer->router_type == SUB1_MX4_FP32)
    mx4_logits_kernel<float, kTokens><<<routers, 256, 0, s>>>(a);
  else
    mx4_logits_kernel<uint16_t, kTokens><<<routers, 256, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  mx4_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  const unsigned tiles = static_cast<unsigned>(most_tiles(layer, tokens));
  mx4_wi_kernel<<<dim3(blocks_of(a.d_ff) * 2, tiles), 64 * kFewWaves, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  mx4_wo_kernel<<<dim3((a.d_model + 15) / 16, tiles), 64 * kFewWaves, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  sub1::note_kernel("mx4_combine_kernel");
  mx4_combine_kernel<<<dim3((a.d_model + 255) / 256, tokens), 256, 0, s>>>(a);
  HIP_TRY(hipGetLastError());
  return SUB1_OK;
}
