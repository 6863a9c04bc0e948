// The router's losses (zmoe_router_losses) over the tokens of S sequences, cu[s] .. cu[s + 1], and their gradient.
//   ph = p / sum_e p,  p = sigmoid(z) or softmax(z);  n_s tokens, c_se how often they chose expert e, S' sequences with any
//   a_se = E c_se / (k n_s^2 S'),  balance = sum_s sum_e a_se sum_{t in s} ph_te
//   z    = 1/N sum_t lse(z_t)^2 over the N tokens of all sequences
//   dz_te = gb ph_te [1 - sigmoid(z_te)] (a_se - sum_j ph_tj a_sj) + gz 2 lse_t / N softmax(z_t)_e     ([]: sigmoid only)
// The counts take no part in the gradient. A token whose logits are all -inf adds nothing and has no gradient; tokens
// outside the sequences neither.
//
// The forward reads the logits once: a workgroup has a tile of kTile tokens, a wave a token, and the sums of the tile's
// part of each sequence go to a slot of their own (tile i and sequence s meet in slot i + s: walking along the tokens
// either number grows by one), which a second launch adds up in a fixed order. The gradient reads the logits again.
#include <type_traits>

#include "zmoe_route.h"

namespace zmoe {
namespace {

constexpr int kTile = 64;
constexpr int kWaves = 4;

struct Sequences {
  const void* cu;  // null: one sequence of all tokens
  int wide;        // int64, else int32
  int S;
  int64_t T;
  __device__ __forceinline__ int64_t at(int s) const {
    if (!cu) return s ? T : 0;
    const int64_t v = wide ? ((const int64_t*)cu)[s] : ((const int32_t*)cu)[s];
    return v < 0 ? 0 : (v > T ? T : v);
  }
  // The first sequence that ends after token t (S if none does).
  __device__ __forceinline__ int after(int64_t t) const {
    int lo = 0, hi = S;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (at(mid + 1) > t) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  }
};

// Scratch: a slot's sums of ph [E], choices [E] and lse^2, then each sequence's part of the two losses.
struct Scratch {
  float* mass;      // [slots, E]
  int32_t* count;   // [slots, E]
  float* zsum;      // [slots]
  double* part;     // [S, 2]
  int32_t* done;    // workgroups of the second launch that have ended
};

__host__ __device__ inline int64_t slots_of(int64_t T, int S) { return (T + kTile - 1) / kTile + S; }

inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }

size_t lay_out(int64_t T, int E, int S, char* base, Scratch* out) {
  const size_t n = (size_t)slots_of(T, S);
  size_t o = 0;
  auto take = [&](size_t bytes) {
    char* p = base + o;
    o += up256(bytes);
    return p;
  };
  Scratch s{};
  s.mass = (float*)take(n * E * 4);
  s.count = (int32_t*)take(n * E * 4);
  s.zsum = (float*)take(n * 4);
  s.part = (double*)take((size_t)S * 16);
  s.done = (int32_t*)take(4);
  if (out) *out = s;
  return o;
}

__device__ __forceinline__ float wave_fmax(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// A token's row, expert lane + 64 q: ph, the softmax's shares (soft) and sigmoids (sig, sigmoid form), its lse; all 0
// where every logit is -inf.
template <int PL, bool SOFT, typename LT>
__device__ __forceinline__ float token_row(const LT* __restrict__ row, int E, int lane, float (&ph)[PL],
                                           float (&soft)[PL], float (&sig)[PL]) {
  float z[PL], m = -INFINITY;
#pragma unroll
  for (int q = 0; q < PL; ++q) {
    const int e = lane + 64 * q;
    z[q] = e < E ? to_f32(row[e]) : -INFINITY;
    m = fmaxf(m, z[q]);
  }
  m = wave_fmax(m);
  const bool none = m == -INFINITY;
  m = none ? 0.f : m;
  float sum = 0.f, total = 0.f;
#pragma unroll
  for (int q = 0; q < PL; ++q) {
    soft[q] = expf(z[q] - m);
    sum += soft[q];
    if constexpr (!SOFT) {
      sig[q] = 1.f / (1.f + expf(-z[q]));
      total += sig[q];
    }
  }
  sum = wave_sum(sum);
  const float inv = none && sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int q = 0; q < PL; ++q) soft[q] *= inv;
  if constexpr (SOFT) {
#pragma unroll
    for (int q = 0; q < PL; ++q) ph[q] = soft[q];
  } else {
    total = wave_sum(total);
    const float inv_total = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int q = 0; q < PL; ++q) ph[q] = sig[q] * inv_total;
  }
  return none && sum == 0.f ? 0.f : m + logf(sum);
}

template <int PL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void losses_tile_kernel(const LT* __restrict__ logits,
                                                                  const int64_t* __restrict__ idx, int E, int k,
                                                                  Sequences seq, Scratch w) {
  __shared__ float mass[kWaves][64 * PL];
  __shared__ int32_t count[64 * PL];
  __shared__ float zs[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tile = blockIdx.x, t0 = tile * kTile, t1 = t0 + kTile < seq.T ? t0 + kTile : seq.T;
  if (tile == 0 && threadIdx.x == 0) *w.done = 0;
  for (int s = seq.after(t0); s < seq.S; ++s) {
    int64_t lo = seq.at(s), hi = seq.at(s + 1);
    if (lo >= t1) break;
    lo = lo < t0 ? t0 : lo;
    hi = hi > t1 ? t1 : hi;
    if (lo >= hi) continue;
    float acc[PL], z2 = 0.f;
#pragma unroll
    for (int q = 0; q < PL; ++q) acc[q] = 0.f;
    for (int e = threadIdx.x; e < E; e += 64 * kWaves) count[e] = 0;
    __syncthreads();
    for (int64_t t = lo + wave; t < hi; t += kWaves) {
      float ph[PL], soft[PL], sig[PL];
      const float lse = token_row<PL, SOFT>(logits + t * E, E, lane, ph, soft, sig);
      z2 += lse * lse;
#pragma unroll
      for (int q = 0; q < PL; ++q) acc[q] += ph[q];
    }
    for (int64_t i = lo * k + threadIdx.x; i < hi * k; i += 64 * kWaves) {
      const int64_t e = idx[i];
      if (e >= 0 && e < E) atomicAdd(&count[e], 1);  // whole numbers: any order
    }
#pragma unroll
    for (int q = 0; q < PL; ++q) mass[wave][lane + 64 * q] = acc[q];
    if (lane == 0) zs[wave] = z2;
    __syncthreads();
    const int64_t slot = tile + s;
    for (int e = threadIdx.x; e < E; e += 64 * kWaves) {
      w.mass[slot * E + e] = mass[0][e] + mass[1][e] + mass[2][e] + mass[3][e];
      w.count[slot * E + e] = count[e];
    }
    if (threadIdx.x == 0) w.zsum[slot] = zs[0] + zs[1] + zs[2] + zs[3];
    __syncthreads();
  }
}

constexpr int kSumThreads = 1024;

// One workgroup a sequence: its slots added up, a_se and the sequence's parts of the losses; the workgroup that ends
// last adds those (their order is the sequences').
__global__ __launch_bounds__(kSumThreads) void losses_sum_kernel(int E, int k, Sequences seq, Scratch w,
                                                                 float* __restrict__ a, float* __restrict__ out,
                                                                 float* __restrict__ inv_tokens) {
  __shared__ double red[kSumThreads / 64][2];
  __shared__ int64_t tot[kSumThreads / 64][2];
  __shared__ int last;
  const int s = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // S' and N
  int64_t live = 0, tokens = 0;
  for (int i = threadIdx.x; i < seq.S; i += kSumThreads) {
    const int64_t n = seq.at(i + 1) - seq.at(i);
    live += n > 0;
    tokens += n > 0 ? n : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    live += __shfl_xor(live, o, 64);
    tokens += __shfl_xor(tokens, o, 64);
  }
  if (lane == 0) {
    tot[wave][0] = live;
    tot[wave][1] = tokens;
  }
  __syncthreads();
  live = tokens = 0;
#pragma unroll
  for (int i = 0; i < kSumThreads / 64; ++i) {
    live += tot[i][0];
    tokens += tot[i][1];
  }
  const int64_t lo = seq.at(s), hi = seq.at(s + 1), n = hi > lo ? hi - lo : 0;
  const int64_t first = lo / kTile + s, end = n > 0 ? (hi - 1) / kTile + s + 1 : first;  // its slots
  const double f = n > 0 ? (double)E / ((double)k * (double)n * (double)n * (double)live) : 0.0;
  double balance = 0.0, z2 = 0.0;
  for (int e = threadIdx.x; e < E; e += kSumThreads) {
    double mass = 0.0;
    int64_t count = 0;
    for (int64_t i = first; i < end; ++i) {
      mass += (double)w.mass[i * E + e];
      count += w.count[i * E + e];
    }
    const double ae = f * (double)count;
    a[(int64_t)s * E + e] = (float)ae;
    balance += ae * mass;
  }
  for (int64_t i = first + threadIdx.x; i < end; i += kSumThreads) z2 += (double)w.zsum[i];
  auto block_sum = [&](double u, double v, double* to) {
    u = [&] { double x = u; for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64); return x; }();
    v = [&] { double x = v; for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64); return x; }();
    if (lane == 0) {
      red[wave][0] = u;
      red[wave][1] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      to[0] = to[1] = 0.0;
      for (int i = 0; i < kSumThreads / 64; ++i) {
        to[0] += red[i][0];
        to[1] += red[i][1];
      }
    }
    __syncthreads();
  };
  double sums[2] = {0.0, 0.0};
  block_sum(balance, z2, sums);
  if (threadIdx.x == 0) {
    w.part[2 * s] = sums[0];
    w.part[2 * s + 1] = sums[1];
    __threadfence();
    last = atomicAdd(w.done, 1) == seq.S - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  balance = z2 = 0.0;
  for (int i = threadIdx.x; i < seq.S; i += kSumThreads) {
    balance += __hip_atomic_load(&w.part[2 * i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    z2 += __hip_atomic_load(&w.part[2 * i + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  block_sum(balance, z2, sums);
  if (threadIdx.x == 0) {
    const double inv = tokens > 0 ? 1.0 / (double)tokens : 0.0;
    out[0] = (float)sums[0];
    out[1] = (float)(sums[1] * inv);
    *inv_tokens = (float)inv;
  }
}

template <int PL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void losses_backward_kernel(const LT* __restrict__ logits, int E,
                                                                      Sequences seq, const float* __restrict__ a,
                                                                      const float* __restrict__ inv_tokens,
                                                                      const float* __restrict__ g_balance,
                                                                      const float* __restrict__ g_z,
                                                                      LT* __restrict__ dz) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tile = blockIdx.x, t0 = tile * kTile, t1 = t0 + kTile < seq.T ? t0 + kTile : seq.T;
  const float gb = g_balance ? *g_balance : 0.f, gz = g_z ? 2.f * *g_z * *inv_tokens : 0.f;
  int s = seq.after(t0 + wave);
  for (int64_t t = t0 + wave; t < t1; t += kWaves) {
    while (s < seq.S && seq.at(s + 1) <= t) ++s;
    const bool in = s < seq.S && seq.at(s) <= t;
    float v[PL];
#pragma unroll
    for (int q = 0; q < PL; ++q) v[q] = 0.f;
    if (in) {
      float ph[PL], soft[PL], sig[PL], as[PL], dot = 0.f;
      const float lse = token_row<PL, SOFT>(logits + t * E, E, lane, ph, soft, sig);
#pragma unroll
      for (int q = 0; q < PL; ++q) {
        const int e = lane + 64 * q;
        as[q] = e < E ? a[(int64_t)s * E + e] : 0.f;
        dot += ph[q] * as[q];
      }
      dot = wave_sum(dot);
#pragma unroll
      for (int q = 0; q < PL; ++q) {
        float d = gb * (ph[q] * (as[q] - dot));
        if constexpr (!SOFT) d *= 1.f - sig[q];
        v[q] = d + gz * lse * soft[q];
      }
    }
#pragma unroll
    for (int q = 0; q < PL; ++q) {
      const int e = lane + 64 * q;
      if (e < E) dz[t * E + e] = from_f32<LT>(v[q]);
    }
  }
}

template <typename F>
void by_width(int E, bool soft, int dtype, F&& f) {
  auto typed = [&](auto pl) {
    auto scored = [&](auto lt) {
      if (soft) f(pl, std::true_type{}, lt);
      else f(pl, std::false_type{}, lt);
    };
    if (dtype == ZMOE_DTYPE_BF16) scored(uint16_t{});
    else scored(float{});
  };
  if (E <= 64) typed(std::integral_constant<int, 1>{});
  else if (E <= 128) typed(std::integral_constant<int, 2>{});
  else if (E <= 256) typed(std::integral_constant<int, 4>{});
  else if (E <= 512) typed(std::integral_constant<int, 8>{});
  else typed(std::integral_constant<int, 16>{});
}

int check_sizes(const char* what, int dtype, int64_t T, int E, int score, const void* cu, int64_t S) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "%s: logits dtype %d", what, dtype);
  ZMOE_REQUIRE(T >= 0 && E >= 1 && E <= 1024, ZMOE_ERR_SHAPE, "%s: need 1 <= E <= 1024 (E=%d)", what, E);
  ZMOE_REQUIRE(score == ZMOE_SCORE_SIGMOID || score == ZMOE_SCORE_SOFTMAX, ZMOE_ERR_SHAPE, "%s: score %d", what, score);
  ZMOE_REQUIRE(S >= 1 && S <= ZMOE_ROUTER_LOSSES_MAX_SEQUENCES, ZMOE_ERR_SHAPE, "%s: need 1 to %d sequences (%lld)", what,
               ZMOE_ROUTER_LOSSES_MAX_SEQUENCES, (long long)S);
  ZMOE_REQUIRE(cu || S == 1, ZMOE_ERR_NULL, "%s: null pointer", what);
  ZMOE_REQUIRE(launch_fits(cdiv(T, kTile), 64 * kWaves), ZMOE_ERR_SHAPE, "%s: too many tokens for one launch", what);
  return ZMOE_OK;
}

}  // namespace
}  // namespace zmoe

using namespace zmoe;

extern "C" size_t zmoe_router_losses_workspace_bytes(int64_t T, int E, int64_t S) {
  if (T < 0 || T >= (1LL << 40) || E < 1 || E > 1024 || S < 1 || S > ZMOE_ROUTER_LOSSES_MAX_SEQUENCES) return 0;
  return lay_out(T, E, (int)S, nullptr, nullptr);
}

extern "C" int zmoe_router_losses(const void* logits, int logits_dtype, int64_t T, int E, const int64_t* topk_idx, int k,
                                  int score, const void* cu_seqlens, int cu_int64, int64_t S, float* losses,
                                  float* seq_grad, float* inv_tokens, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (const int rc = check_sizes("router_losses", logits_dtype, T, E, score, cu_seqlens, S)) return rc;
  ZMOE_REQUIRE(k >= 1 && k <= E, ZMOE_ERR_SHAPE, "router_losses: need 1 <= k <= E (k=%d, E=%d)", k, E);
  ZMOE_REQUIRE(losses && seq_grad && inv_tokens && workspace && (T == 0 || (logits && topk_idx)),
               ZMOE_ERR_NULL, "router_losses: null pointer");
  ZMOE_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, ZMOE_ERR_ALIGN,
               "router_losses: the workspace must be 16-byte aligned");
  Scratch w{};
  const size_t need = lay_out(T, E, (int)S, (char*)workspace, &w);
  ZMOE_REQUIRE(workspace_bytes >= need, ZMOE_ERR_WORKSPACE, "router_losses: workspace %zu < %zu bytes", workspace_bytes,
               need);
  const Sequences seq{cu_seqlens, cu_int64 != 0, (int)S, T};
  const unsigned tiles = (unsigned)(T > 0 ? cdiv(T, kTile) : 1);
  by_width(E, score == ZMOE_SCORE_SOFTMAX, logits_dtype, [&](auto pl, auto soft, auto lt) {
    using LT = decltype(lt);
    hipLaunchKernelGGL((losses_tile_kernel<decltype(pl)::value, decltype(soft)::value, LT>), dim3(tiles),
                       dim3(64 * kWaves), 0, as_stream(stream), (const LT*)logits, topk_idx, E, k, seq, w);
  });
  if (const int rc = check_launch("router_losses")) return rc;
  hipLaunchKernelGGL(losses_sum_kernel, dim3((unsigned)S), dim3(kSumThreads), 0, as_stream(stream), E, k, seq, w,
                     seq_grad, losses, inv_tokens);
  return check_launch("router_losses");
}

extern "C" int zmoe_router_losses_backward(const void* logits, int logits_dtype, int64_t T, int E, int score,
                                           const void* cu_seqlens, int cu_int64, int64_t S, const float* seq_grad,
                                           const float* inv_tokens, const float* d_balance, const float* d_z,
                                           void* d_logits, void* stream) {
  if (const int rc = check_sizes("router_losses_backward", logits_dtype, T, E, score, cu_seqlens, S)) return rc;
  if (T == 0) return ZMOE_OK;
  ZMOE_REQUIRE(logits && seq_grad && inv_tokens && d_logits, ZMOE_ERR_NULL,
               "router_losses_backward: null pointer");
  const Sequences seq{cu_seqlens, cu_int64 != 0, (int)S, T};
  by_width(E, score == ZMOE_SCORE_SOFTMAX, logits_dtype, [&](auto pl, auto soft, auto lt) {
    using LT = decltype(lt);
    hipLaunchKernelGGL((losses_backward_kernel<decltype(pl)::value, decltype(soft)::value, LT>),
                       dim3((unsigned)cdiv(T, kTile)), dim3(64 * kWaves), 0, as_stream(stream), (const LT*)logits, E, seq,
                       seq_grad, inv_tokens, d_balance, d_z, (LT*)d_logits);
  });
  return check_launch("router_losses_backward");
}
