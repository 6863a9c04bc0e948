// Routing in its other forms (zmoe_route): sigmoid or softmax scores, a bias for the selection, groups of experts of
// which the best stay, weights renormalised or as they are; and its gradient.
//   p = sigmoid(z) or softmax(z), rounded once to f32 (a row of -inf alone: p = 0);  s = p + b in f32
//   a group's score: its highest s, or the sum of its two highest; the top_groups best groups stay
//   idx = the k best s in them (s desc, expert asc, NaN first);  w = c p_idx / max(sum p_idx, 1e-12), or c p_idx
// Backward: dp_j = c (dw_j - sum_i dw_i p_i / S) / S (S the clamped sum; clamped or not renormalised: without the
// sum's part). Sigmoid: dz = dp p (1 - p), 1 - p from the logit again, for a rounded p has lost it (at z = 12 it is off by 0.5%, from
// 17.4 on 0). Softmax: dz_e = p_e (dp_e - sum_j dp_j p_j), where the sum is 0 if the weights are renormalised: then
// only selected experts have a grad and the logits are not read.
//
// Where p + b decides, one f32 rounding of p can decide: p comes from double, whose error (some 2^-52) moves an f32
// rounding for one value in 2^28. Without a bias the experts' order is their logits' order.
//
// Few bytes (8192 tokens of 256 experts 5 MB, 1 us at the copy's rate) and many instructions: a token's experts lie over a
// row of lanes, so that a wave has several tokens; of its 1650 vector and 600 scalar instructions (counted) for four of them 570
// are the sigmoids in double, 1030 the k = 8 rounds of maximum, first holder and mark, 200 the groups (by the listing). 8192
// tokens of 256 experts in 8 groups 9.6 us in a graph's replays (11.5 traced; two waves a SIMD), 32768 of 128 by softmax 12.9
// (14.6), 32749 of 160 in f32 23 traced; the softmaxes' backwards, a pass over the [T, E] grad, 5.4 and 12 traced (4.2 and 11.5 in
// replays, 3.0 and 3.9 TB/s). A sigmoid's, with the logits of those taken, 5.3 and 7.6 in replays (4.8 and 6.4 from p alone).
#include "zmoe_route.h"

namespace zmoe {
namespace {

constexpr int kMaxSlots = 64;
constexpr int kWaves = 4;  // of a workgroup

struct RouteArgs {
  const void* logits;
  const float* bias;  // or null
  int64_t T;
  int E, k, groups, group_size, top_groups, group_scores, renorm, vec, bias_vec;
  int lanes_of_group;  // where a group is whole lanes, a power of two of them; else 0, and
  int log_together;    // 2^that many lanes score a group
  int inv_group;       // 2^20 / experts of a group, rounded up
  float scale;
  int64_t* idx;
  float* w;
  float* p;  // or null
};

// What a wave wrote to LDS is there for its other lanes (a wave's LDS accesses stay in order).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// score_key in fewer instructions: -0 goes with +0 by an addition.
__device__ __forceinline__ uint32_t order_key(float s) {
  const uint32_t b = __float_as_uint(s + 0.f);
  const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return s != s ? 0xffffffffu : key;
}

// The float whose score_key is key (a NaN, +0 for both zeros).
__device__ __forceinline__ float key_score(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Rows of LPR lanes, VPL consecutive experts a lane, 64 / LPR tokens a wave at once; waves stride over the tokens.
template <int LPR, int VPL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void route_kernel(const RouteArgs a) {
  constexpr int TPW = 64 / LPR, W = LPR * VPL;
  __shared__ float ps[kWaves][TPW][W];
  __shared__ uint32_t gk[kWaves][TPW][W];
  __shared__ uint16_t slots[kWaves][TPW][kMaxSlots];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane / LPR, r = lane % LPR, e0 = r * VPL;
  const int E = a.E, k = a.k, G = a.groups, gsz = a.group_size;
  const bool two = a.group_scores == 2 && G > 1;
  const bool by_p = a.bias != nullptr;
  float b[VPL];  // past E -inf, as the logits: behind every expert
  if (by_p) load_lane<VPL>(a.bias, e0, E, a.bias_vec, true, -INFINITY, b);

  const int64_t step = (int64_t)gridDim.x * kWaves * TPW;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * TPW; t0 < a.T; t0 += step) {
    const int64_t t = t0 + row;
    const bool live = t < a.T;
    float z[VPL], p[VPL];
    load_lane<VPL>((const LT*)a.logits + t * E, e0, E, a.vec, live, -INFINITY, z);
    if constexpr (SOFT) {
      float m = z[0];
#pragma unroll
      for (int q = 1; q < VPL; ++q) m = fmaxf(m, z[q]);
      m = lanes_fmax<LPR>(m);
      m = m == -INFINITY ? 0.f : m;  // nothing to choose from: all p are 0
      double e[VPL], sum = 0.0;
#pragma unroll
      for (int q = 0; q < VPL; ++q) {
        e[q] = exp_f64((double)z[q] - (double)m);
        sum += e[q];
      }
      sum = lanes_sum<LPR>(sum);
      const double inv = sum == 0.0 ? 0.0 : rcp_f64(sum);
#pragma unroll
      for (int q = 0; q < VPL; ++q) p[q] = (float)(e[q] * inv);
    } else {
      sigmoids_rounded(z, p);
    }
    if (by_p) {
#pragma unroll
      for (int q = 0; q < VPL; ++q) z[q] = p[q] + b[q];
    }
    uint32_t key[VPL];
#pragma unroll
    for (int q = 0; q < VPL; ++q) {
      key[q] = order_key(z[q]);
      ps[wave][row][e0 + q] = p[q];
    }
    if (G > 1) {
      constexpr int PER = (64 + LPR - 1) / LPR;  // groups of a lane
      const int share = 1 << a.log_together;
      uint32_t mine[PER];
      if (a.lanes_of_group) {  // a group is whole lanes, a power of two of them: its first lane speaks for it
        uint32_t k1 = 0, k2 = 0;
#pragma unroll
        for (int q = 0; q < VPL; ++q) {
          const uint32_t v = two && !by_p ? order_key(p[q]) : key[q];
          k2 = max(k2, min(k1, v));
          k1 = max(k1, v);
        }
        for (int o = 1; o < a.lanes_of_group; o <<= 1) {
          const uint32_t o1 = __shfl_xor(k1, o, 64), o2 = __shfl_xor(k2, o, 64);
          k2 = max(max(k2, o2), min(k1, o1));
          k1 = max(k1, o1);
        }
        const uint32_t best = two ? order_key(key_score(k1) + key_score(k2)) : k1;
        mine[0] = live && e0 < E && (r & (a.lanes_of_group - 1)) == 0 ? best : 0u;
#pragma unroll
        for (int i = 1; i < PER; ++i) mine[i] = 0;
      } else {
#pragma unroll
        for (int q = 0; q < VPL; ++q) gk[wave][row][e0 + q] = two && !by_p ? order_key(p[q]) : key[q];
        wave_sync();
        // share lanes score a group together (a power of two, one where there are more groups than half the lanes): lane r
        // entries r % share, ... of group r / share, then of the next groups
        const int ro = opaque(r);  // (nothing of this path is kept over the loop)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int g = (ro >> a.log_together) + i * LPR;
          mine[i] = 0;
          uint32_t k1 = 0, k2 = 0;
          if (g < G && live) {
            const uint32_t* at = &gk[wave][row][g * gsz];
#pragma unroll 4
            for (int u = ro & (share - 1); u < gsz; u += share) {
              const uint32_t v = at[u];
              k2 = max(k2, min(k1, v));
              k1 = max(k1, v);
            }
          }
          for (int o = 1; o < share; o <<= 1) {
            const uint32_t o1 = __shfl_xor(k1, o, 64), o2 = __shfl_xor(k2, o, 64);
            k2 = max(max(k2, o2), min(k1, o1));
            k1 = max(k1, o1);
          }
          if (g < G && live && (ro & (share - 1)) == 0) mine[i] = two ? order_key(key_score(k1) + key_score(k2)) : k1;
        }
      }
      uint64_t keep = 0;  // by the number of the lane that speaks for a group, the same in a row's lanes
      for (int j = 0; j < a.top_groups; ++j) {
        uint32_t m = mine[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) m = max(m, mine[i]);
        m = lanes_max<LPR>(m);
        uint32_t g = 0xffffffffu;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) g = mine[i] == m ? (uint32_t)(r + i * LPR) : g;
        g = lanes_min<LPR>(g);
        keep |= 1ull << (g & 63);
#pragma unroll
        for (int i = 0; i < PER; ++i) mine[i] = (uint32_t)(r + i * LPR) == g ? 0u : mine[i];
      }
      if (a.lanes_of_group) {
        const bool stays = (keep >> (r & -a.lanes_of_group)) & 1;
#pragma unroll
        for (int q = 0; q < VPL; ++q) key[q] = stays ? key[q] : 0u;
      } else {
        const uint32_t lo = (uint32_t)keep, hi = (uint32_t)(keep >> 32);
        uint32_t e = (uint32_t)opaque(e0);
#pragma unroll
        for (int q = 0; q < VPL; ++q, ++e) {
          const uint32_t bit = (e * (uint32_t)a.inv_group >> 20) << a.log_together;  // e / gsz, exact below 1024
          key[q] = ((bit < 32 ? lo : hi) >> (bit & 31)) & 1 ? key[q] : 0u;
        }
      }
    }
    for (int j = 0; j < k; ++j) {
      uint32_t m = key[0];
#pragma unroll
      for (int q = 1; q < VPL; ++q) m = max(m, key[q]);
      m = lanes_max<LPR>(m);
      // this lane's lowest expert holding m, then the row's; that one is taken (the lane's first hit, by wave masks)
      uint64_t hit[VPL];
#pragma unroll
      for (int q = 0; q < VPL; ++q) hit[q] = __builtin_amdgcn_ballot_w64(key[q] == m);
      uint32_t e = 0xffffffffu;
#pragma unroll
      for (int q = VPL - 1; q >= 0; --q) e = __builtin_amdgcn_inverse_ballot_w64(hit[q]) ? (uint32_t)(e0 + q) : e;
      const uint32_t best = lanes_min<LPR>(e);
      const uint64_t owner = __builtin_amdgcn_ballot_w64(e == best);
      uint64_t seen = 0;
#pragma unroll
      for (int q = 0; q < VPL; ++q) {
        const uint64_t first = hit[q] & owner & ~seen;
        seen |= hit[q];
        key[q] = __builtin_amdgcn_inverse_ballot_w64(first) ? 0u : key[q];
      }
      if (r == 0) slots[wave][row][j] = (uint16_t)best;
    }
    wave_sync();
    float sum = 0.f;
    for (int j = r; j < k; j += LPR) sum += ps[wave][row][slots[wave][row][j]];
    sum = lanes_sum<LPR>(sum);
    const float denom = sum < 1e-12f ? 1e-12f : sum;  // NaN propagates
    if (live) {
      for (int j = r; j < k; j += LPR) {
        const int e = slots[wave][row][j];
        const float pj = ps[wave][row][e];
        a.idx[t * k + j] = e;
        a.w[t * k + j] = a.scale * (a.renorm ? pj / denom : pj);
        if (a.p) a.p[t * k + j] = pj;
      }
    }
    wave_sync();  // before the next token's values
  }
}

struct RouteBackwardArgs {
  const float* dw;
  const float* p;
  const int64_t* idx;
  const void* logits;  // null: sigmoids of which p is all there is
  const void* add;     // or null: [T, E] of the grad's type, rows ld_add apart
  int64_t ld_add, T, ld;
  int E, k, renorm, vec;
  float scale;
  void* dz;
};

template <int LPR, int VPL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void route_backward_kernel(const RouteBackwardArgs a) {
#pragma clang fp contract(off)  // (one expert's renormalised weight has a grad of rounding errors alone: 0, not fused ones)
  constexpr int TPW = 64 / LPR, W = LPR * VPL, STEP = kSpread<LPR, VPL, LT>;
  __shared__ float ds[kWaves][TPW][W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = lane / LPR, r = lane % LPR, e0 = spread_first<VPL, LT>(r);
  const int E = a.E, k = a.k;
  const int64_t step = (int64_t)gridDim.x * kWaves * TPW;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWaves + wave) * TPW; t0 < a.T; t0 += step) {
    const int64_t t = t0 + row;
    const bool live = t < a.T;
    float* mine = &ds[wave][row][0];
#pragma unroll
    for (int q = 0; q < VPL; ++q) mine[e0 + lane_element<VPL, STEP, LT>(q)] = 0.f;
    float add[VPL];
    if (a.add) load_lane<VPL, STEP>((const LT*)a.add + t * a.ld_add, e0, E, a.vec, live, 0.f, add);
    float S = 0.f, dot = 0.f;  // sum p, sum c dw p
    if (live)
      for (int j = r; j < k; j += LPR) {
        const float pj = a.p[t * k + j];
        S += pj;
        dot += a.scale * a.dw[t * k + j] * pj;
      }
    S = lanes_sum<LPR>(S);
    dot = lanes_sum<LPR>(dot);
    // not scaled: the weights are c p (/ 1e-12), and the softmax's sum of dp p is not 0
    const bool scaled = a.renorm && !(S <= 1e-12f);
    const float total = !a.renorm ? 1.f : scaled ? S : 1e-12f;
    const float mean = scaled ? dot / total : 0.f, inner = scaled ? 0.f : dot / total;
    wave_sync();
    if (live)
      for (int j = r; j < k; j += LPR) {
        const int64_t e = a.idx[t * k + j];
        const float pj = a.p[t * k + j], dp = (a.scale * a.dw[t * k + j] - mean) / total;
        if (e < 0 || e >= E) continue;
        if constexpr (SOFT) mine[e] = pj * (dp - inner);
        else mine[e] = dp * pj * (a.logits ? sigmoid_complement(to_f32(((const LT*)a.logits)[t * E + e])) : 1.f - pj);
      }
    wave_sync();
    float v[VPL];
#pragma unroll
    for (int q = 0; q < VPL; ++q) v[q] = mine[e0 + lane_element<VPL, STEP, LT>(q)];
    if constexpr (SOFT) {
      if (!scaled) {  // every logit has a grad: -p_e sum dp p where it is not selected
        float z[VPL];
        load_lane<VPL, STEP>((const LT*)a.logits + t * E, e0, E, a.vec, live, -INFINITY, z);
        float m = z[0], sum = 0.f;
#pragma unroll
        for (int q = 1; q < VPL; ++q) m = fmaxf(m, z[q]);
        m = lanes_fmax<LPR>(m);
        m = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int q = 0; q < VPL; ++q) {
          z[q] = exp_fast(z[q] - m);
          sum += z[q];
        }
        sum = lanes_sum<LPR>(sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint32_t sel = 0;
        if (live)
          for (int j = 0; j < k; ++j) {
            const int64_t d = a.idx[t * k + j] - e0;  // the lane's chunk d / STEP, and its place in it
            constexpr int N = LaneChunk<VPL, LT>::N;
            if (d >= 0 && d < W && d % STEP < N) sel |= 1u << (int)(d / STEP * N + d % STEP);
          }
#pragma unroll
        for (int q = 0; q < VPL; ++q) v[q] = (sel >> q) & 1 ? v[q] : -(z[q] * inv) * inner;
      }
    }
    if (a.add) {
#pragma unroll
      for (int q = 0; q < VPL; ++q) v[q] += add[q];
    }
    if (live) store_lane<VPL, STEP>((LT*)a.dz + t * a.ld, e0, E, a.vec, v);
    wave_sync();
  }
}

// Few tokens are a wave's latency, which fewer experts a lane shorten (us in a graph's replays, sigmoids and groups):
//   tokens of 256 experts      3    512   2048   4096   8192  32768
//   64 lanes of 4            5.2    5.5    6.3    8.6   13.5   48.4
//   32 lanes of 8            5.3    5.6    5.7    6.8    9.9   29.9
//   16 lanes of 16           6.8    7.3    7.5    7.6    9.6   27.2
//   512 experts, 64 of 8     5.9    6.3    7.5   10.8   17.9   65.1
//   32 of 16                 7.3    7.6    7.8    9.7   16.0   52.4
// (160 experts: 64 of 4 4.8, 5.3, 6.0, 8.2, 12.5; 16 of 12 6.4, 6.9, 6.9, 7.0, 8.6; 128: 16 of 8 4.1 to 4.7, 8 of 16 5.7 to 6.3.)
constexpr int64_t kFewTokens = 512, kSomeTokens = 4096, kFewOfMany = 2048;

// Workgroups that hold the tokens, at most eight a CU: their waves loop over the others.
unsigned grid_of(int64_t T, int lpr) {
  const int64_t blocks = cdiv(T, (int64_t)kWaves * (64 / lpr));
  return (unsigned)(blocks < 2048 ? blocks : 2048);
}

}  // namespace
}  // namespace zmoe

using namespace zmoe;

extern "C" int zmoe_route(const void* logits, int logits_dtype, int64_t T, int E, int k, int score,
                          const float* expert_biases, int groups, int top_groups, int group_scores, int renormalize,
                          float scale, int64_t* topk_idx, float* topk_weight, float* topk_prob, void* stream) {
  ZMOE_REQUIRE(dtype_ok(logits_dtype), ZMOE_ERR_DTYPE, "route: logits dtype %d", logits_dtype);
  ZMOE_REQUIRE(T >= 0 && E >= 1 && E <= 1024, ZMOE_ERR_SHAPE, "route: need 1 <= E <= 1024 (E=%d)", E);
  ZMOE_REQUIRE(score == ZMOE_SCORE_SIGMOID || score == ZMOE_SCORE_SOFTMAX, ZMOE_ERR_SHAPE, "route: score %d", score);
  ZMOE_REQUIRE(groups >= 1 && groups <= 64 && E % groups == 0, ZMOE_ERR_SHAPE,
               "route: need 1 to 64 groups of equal size (groups=%d, E=%d)", groups, E);
  ZMOE_REQUIRE(top_groups >= 1 && top_groups <= groups, ZMOE_ERR_SHAPE, "route: need 1 <= top_groups <= groups (%d, %d)",
               top_groups, groups);
  ZMOE_REQUIRE(group_scores >= 1 && group_scores <= 2 && (groups == 1 || group_scores <= E / groups), ZMOE_ERR_SHAPE,
               "route: a group's score is of its 1 or 2 best experts (group_scores=%d, %d in a group)", group_scores,
               E / groups);
  ZMOE_REQUIRE(k >= 1 && k <= kMaxSlots && k <= top_groups * (E / groups), ZMOE_ERR_SHAPE,
               "route: need 1 <= k <= %d and experts to choose from (k=%d, %d)", kMaxSlots, k, top_groups * (E / groups));
  if (T == 0) return ZMOE_OK;
  ZMOE_REQUIRE(logits && topk_idx && topk_weight, ZMOE_ERR_NULL, "route: null pointer");
  RouteArgs a{logits, expert_biases, T, E, k, groups, E / groups, top_groups, group_scores, renormalize,
              rows_on_16(logits, E, E, logits_dtype), rows_on_16(expert_biases, E, E, ZMOE_DTYPE_F32), 0, 1,
              (1 << 20) / (E / groups) + 1, scale, topk_idx, topk_weight, topk_prob};
  auto go = [&](auto lpr, auto vpl, auto soft, auto lt) {
    const int lanes = E / groups / decltype(vpl)::value;
    a.lanes_of_group = lanes * decltype(vpl)::value == E / groups && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    for (a.log_together = 0; (2 << a.log_together) * groups <= decltype(lpr)::value;) ++a.log_together;
    hipLaunchKernelGGL((route_kernel<decltype(lpr)::value, decltype(vpl)::value, decltype(soft)::value, decltype(lt)>),
                       dim3(grid_of(T, decltype(lpr)::value)), dim3(64 * kWaves), 0, as_stream(stream), a);
  };
  if (E > 128 && T <= (E <= 256 ? kSomeTokens : E <= 512 ? kFewOfMany : 0)) {
    const auto typed = [&](auto lpr, auto vpl, auto soft) {
      if (logits_dtype == ZMOE_DTYPE_BF16) go(lpr, vpl, soft, uint16_t{});
      else go(lpr, vpl, soft, float{});
    };
    const auto scored = [&](auto lpr, auto vpl) {
      if (score == ZMOE_SCORE_SOFTMAX) typed(lpr, vpl, std::true_type{});
      else typed(lpr, vpl, std::false_type{});
    };
    if (E > 256) scored(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    else if (T <= kFewTokens) scored(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
    else scored(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
  } else {
    by_lanes(E, score == ZMOE_SCORE_SOFTMAX, logits_dtype, go);
  }
  return check_launch("route");
}

extern "C" int zmoe_route_backward(const float* d_weight, const float* topk_prob, const int64_t* topk_idx, int64_t T,
                                   int E, int k, int score, const void* logits, int renormalize, float scale,
                                   const void* add, int64_t ld_add, void* d_logits, int64_t ld_d_logits,
                                   int d_logits_dtype, void* stream) {
  ZMOE_REQUIRE(dtype_ok(d_logits_dtype), ZMOE_ERR_DTYPE, "route_backward: dtype %d", d_logits_dtype);
  ZMOE_REQUIRE(T >= 0 && E >= 1 && E <= 1024 && k >= 1 && k <= E && k <= kMaxSlots, ZMOE_ERR_SHAPE,
               "route_backward: bad sizes (E=%d, k=%d)", E, k);
  ZMOE_REQUIRE(score == ZMOE_SCORE_SIGMOID || score == ZMOE_SCORE_SOFTMAX, ZMOE_ERR_SHAPE, "route_backward: score %d",
               score);
  ZMOE_REQUIRE(ld_d_logits >= E && (!add || ld_add >= E), ZMOE_ERR_SHAPE, "route_backward: row stride below E=%d", E);
  if (T == 0) return ZMOE_OK;
  ZMOE_REQUIRE(d_weight && topk_prob && topk_idx && d_logits && (logits || score == ZMOE_SCORE_SIGMOID), ZMOE_ERR_NULL,
               "route_backward: null pointer");
  const bool vec = rows_on_16(d_logits, ld_d_logits, E, d_logits_dtype) &&
                   (!add || rows_on_16(add, ld_add, E, d_logits_dtype)) &&
                   (!logits || rows_on_16(logits, E, E, d_logits_dtype));
  const RouteBackwardArgs a{d_weight, topk_prob, topk_idx, logits, add, ld_add, T, ld_d_logits, E, k, renormalize, vec,
                            scale, d_logits};
  by_lanes(E, score == ZMOE_SCORE_SOFTMAX, d_logits_dtype, [&](auto lpr, auto vpl, auto soft, auto lt) {
    hipLaunchKernelGGL(
        (route_backward_kernel<decltype(lpr)::value, decltype(vpl)::value, decltype(soft)::value, decltype(lt)>),
        dim3(grid_of(T, decltype(lpr)::value)), dim3(64 * kWaves), 0, as_stream(stream), a);
  });
  return check_launch("route_backward");
}
