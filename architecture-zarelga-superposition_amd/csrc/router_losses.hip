// The router's losses (zmoe_router_losses) over the tokens of S sequences, cu[s] .. cu[s + 1], and their gradient.
//   ph = p / sum_e p,  p = sigmoid(z) or softmax(z);  n_s tokens, c_se how often they chose expert e, S' sequences with any
//   a_se = E c_se / (k n_s^2 S'),  balance = sum_s sum_e a_se sum_{t in s} ph_te
//   z    = 1/N sum_t lse(z_t)^2 over the N tokens of all sequences
//   dz_te = gb ph_te [1 - sigmoid(z_te)] (a_se - sum_j ph_tj a_sj) + gz 2 lse_t / N softmax(z_t)_e     ([]: sigmoid only)
// The counts take no part in the gradient. A token whose logits are all -inf adds nothing and has no gradient; tokens
// outside the sequences neither.
//
// The forward reads the logits once: a workgroup has a tile of tokens, a row of LPR lanes a token (VPL experts a
// lane), and the sums of the tile's part of each sequence go to a slot of their own (tile i and sequence s meet in slot
// i + s: walking along the tokens either number grows by one), which a second launch adds up in a fixed order, a
// workgroup for each sequence and 32 experts. The gradient reads the logits again. Both are short: what bounds them is
// the latency of a few dependent reads in each of the launches, and the exponentials (32749 tokens of 256 experts in 37
// sequences, f32: 15.3 us, 2.4 TB/s, then 10.8 for the sums and 18.8 for the gradient, 3.6 TB/s; 32768 of 128, bf16, one
// sequence: 6.8, 7.3 and 7.7; 517 of 32: 6.2, 6.7 and 4.3).
//
// A workgroup takes the sequences of its tile one after the other, empty ones among them (two dependent reads, 0.4 us, each), and
// the second launch has a workgroup for each sequence, empty or not, and 32 experts. So the forward grows with short, empty or very long
// sequences (in a graph's replays, 128 experts, bf16): 32768 tokens in 37 sequences 15.6 us; with the last border repeated up to
// S = 4096 286 where it is a tile's border or T, 1755 inside a tile; in 4096 sequences of 8 tokens 313, in 32768 of one 2460; 2^20
// tokens in one sequence 137 (of 32 experts 112). The backward skips empty sequences 64 at a time from its wave's first
// token on (5.6 to 12 us for those of 32768 tokens), and walks one by one from there: 605 us where a wave has rows past T and
// T's border is repeated up to S = 4096.
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
  // The first sequence that ends after token t (S if none does), for a t that is the same in the wave: all borders
  // counted at once, many of them halved first.
  __device__ __forceinline__ int after(int64_t t) const {
    if (!cu) return t < T ? 0 : 1;
    int lo = 0, hi = S;
    while (hi - lo > 512) {
      const int mid = (lo + hi) >> 1;
      if (at(mid + 1) > t) hi = mid;
      else lo = mid + 1;
    }
    int n = 0;
    for (int i = lo + (int)(threadIdx.x & 63); i - (int)(threadIdx.x & 63) < hi; i += 64)
      n += __popcll(__ballot(i < hi && at(i + 1) <= t));
    return lo + n;
  }
};

// Scratch: a slot's sums of ph [E], choices [E] and lse^2, then the parts of the two losses, S' and N, a counter.
struct Scratch {
  float* mass;      // [slots, E]
  int32_t* count;   // [slots, E]
  float* zsum;      // [slots]
  double* part;     // [S, column blocks, 2]
  int64_t* total;   // S', N
  int32_t* done;    // workgroups of the second launch that have ended
};

__host__ __device__ inline int64_t slots_of(int64_t T, int S) { return (T + kTile - 1) / kTile + S; }
constexpr int kColumns = 32;  // experts of a workgroup of the second launch
inline int column_blocks(int E) { return (E + kColumns - 1) / kColumns; }

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
  s.part = (double*)take((size_t)S * column_blocks(E) * 16);
  s.total = (int64_t*)take(16);
  s.done = (int32_t*)take(4);
  if (out) *out = s;
  return o;
}

// A token's values in a row of lanes from its logits z (-inf past E): ph and the softmax's shares, all 0 where every logit
// is -inf, and (sigmoid form) 1 - sigmoid, for z > 0 from e^-z, as the difference would lose it; its lse.
template <int LPR, int VPL, bool SOFT>
__device__ __forceinline__ float token_row(const float (&z)[VPL], float (&ph)[VPL], float (&soft)[VPL],
                                           float (&rest)[VPL]) {
  float m = z[0];
#pragma unroll
  for (int q = 1; q < VPL; ++q) m = fmaxf(m, z[q]);
  m = lanes_fmax<LPR>(m);
  const bool none = m == -INFINITY;
  m = fabsf(m) == INFINITY ? 0.f : m;  // (+inf: an lse of inf, unless a NaN is there too)
  float sum = 0.f, total = 0.f;
#pragma unroll
  for (int q = 0; q < VPL; ++q) {
    soft[q] = exp_fast(z[q] - m);
    sum += soft[q];
    if constexpr (!SOFT) {
      const float u = exp_fast(-z[q]);
      ph[q] = __builtin_amdgcn_rcpf(1.f + u);
      rest[q] = z[q] > 0.f ? u * ph[q] : 1.f - ph[q];
      total += ph[q];
    }
  }
  sum = lanes_sum<LPR>(sum);
  const float inv = none && sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int q = 0; q < VPL; ++q) soft[q] *= inv;
  if constexpr (SOFT) {
#pragma unroll
    for (int q = 0; q < VPL; ++q) ph[q] = soft[q];
  } else {
    total = lanes_sum<LPR>(total);
    const float inv_total = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int q = 0; q < VPL; ++q) ph[q] *= inv_total;
  }
  return none && sum == 0.f ? 0.f : m + logf(sum);
}

template <int LPR, int VPL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void losses_tile_kernel(const LT* __restrict__ logits,
                                                                  const int64_t* __restrict__ idx, int E, int k, bool vec,
                                                                  Sequences seq, Scratch w) {
  constexpr int TPW = 64 / LPR, ROWS = kWaves * TPW, W = LPR * VPL;
  __shared__ float mass[kWaves][W];
  __shared__ int32_t count[W];
  __shared__ float zs[kWaves];
  constexpr int STEP = kSpread<LPR, VPL, LT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane / LPR;
  const int e0 = spread_first<VPL, LT>(lane % LPR);
  const int64_t tile = blockIdx.x, t0 = tile * kTile, t1 = t0 + kTile < seq.T ? t0 + kTile : seq.T;
  if (tile == gridDim.x - 1) {  // a workgroup of its own: S' and N
    int64_t live = 0, tokens = 0;
    for (int i = threadIdx.x; i < seq.S; i += 64 * kWaves) {
      const int64_t n = seq.at(i + 1) - seq.at(i);
      live += n > 0;
      tokens += n > 0 ? n : 0;
    }
    __shared__ int64_t part[kWaves][2];
    live = lanes_sum<64>(live);
    tokens = lanes_sum<64>(tokens);
    if (lane == 0) {
      part[wave][0] = live;
      part[wave][1] = tokens;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      *w.done = 0;
      w.total[0] = part[0][0] + part[1][0] + part[2][0] + part[3][0];
      w.total[1] = part[0][1] + part[1][1] + part[2][1] + part[3][1];
    }
    return;
  }
  for (int s = seq.after(t0); s < seq.S; ++s) {
    int64_t lo = seq.at(s), hi = seq.at(s + 1);
    if (lo >= t1) break;
    lo = lo < t0 ? t0 : lo;
    hi = hi > t1 ? t1 : hi;
    if (lo >= hi) continue;
    const int64_t slot = tile + s;
    float acc[VPL], z2 = 0.f, nxt[VPL];
    int64_t t = lo + wave * TPW + row;
    load_lane<VPL, STEP>(logits + t * E, e0, E, vec, t < hi, -INFINITY, nxt);
#pragma unroll
    for (int q = 0; q < VPL; ++q) acc[q] = 0.f;
    for (int e = threadIdx.x; e < E; e += 64 * kWaves) count[e] = 0;
    __syncthreads();
    for (int64_t i = lo * k + threadIdx.x; i < hi * k; i += 64 * kWaves) {
      const int64_t e = idx[i];
      if (e >= 0 && e < E) atomicAdd(&count[e], 1);  // whole numbers: any order
    }
    for (int64_t b = lo; b < hi; b += ROWS, t += ROWS) {  // the next rows are on their way while these are added
      float z[VPL], ph[VPL], soft[VPL], rest[VPL];
#pragma unroll
      for (int q = 0; q < VPL; ++q) z[q] = nxt[q];
      load_lane<VPL, STEP>(logits + (t + ROWS) * E, e0, E, vec, t + ROWS < hi, -INFINITY, nxt);
      const float lse = token_row<LPR, VPL, SOFT>(z, ph, soft, rest);  // (past the end: a row of -inf)
      z2 += lse * lse;
#pragma unroll
      for (int q = 0; q < VPL; ++q) acc[q] += ph[q];
    }
    // over the wave's rows
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) {
      z2 += __shfl_xor(z2, o, 64);
#pragma unroll
      for (int q = 0; q < VPL; ++q) acc[q] += __shfl_xor(acc[q], o, 64);
    }
    if (row == 0) {
#pragma unroll
      for (int q = 0; q < VPL; ++q) mass[wave][e0 + lane_element<VPL, STEP, LT>(q)] = acc[q];
    }
    if (lane == 0) zs[wave] = z2;
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 64 * kWaves) {
      w.mass[slot * E + e] = mass[0][e] + mass[1][e] + mass[2][e] + mass[3][e];
      w.count[slot * E + e] = count[e];
    }
    if (threadIdx.x == 0) w.zsum[slot] = zs[0] + zs[1] + zs[2] + zs[3];
    __syncthreads();
  }
}

constexpr int kSumThreads = 512;

// A workgroup for each sequence and 32 experts: its slots added up, a_se and its parts of the losses; the workgroup that
// ends last adds those, in the sequences' order.
__global__ __launch_bounds__(kSumThreads) void losses_sum_kernel(int E, int k, Sequences seq, Scratch w,
                                                                 float* __restrict__ a, float* __restrict__ out,
                                                                 float* __restrict__ inv_tokens) {
  constexpr int GROUPS = kSumThreads / kColumns;  // threads of one expert
  constexpr int WAVES = kSumThreads / 64;
  __shared__ double red[WAVES][kColumns];
  __shared__ int64_t redc[WAVES][kColumns];
  __shared__ double wave_sums[kSumThreads / 64][2];
  __shared__ int last;
  const int s = blockIdx.x, cb = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t lo = seq.at(s), hi = seq.at(s + 1), n = hi > lo ? hi - lo : 0;
  const int64_t first = lo / kTile + s, end = n > 0 ? (hi - 1) / kTile + s + 1 : first;  // its slots
  const int col = threadIdx.x % kColumns, group = threadIdx.x / kColumns, e = cb * kColumns + col;
  double mass = 0.0;
  int64_t count = 0;
  if (e < E) {
#pragma unroll 8
    for (int64_t i = first + group; i < end; i += GROUPS) {
      mass += (double)w.mass[i * E + e];
      count += w.count[i * E + e];
    }
  }
  double z2 = 0.0;
  if (cb == 0)
    for (int64_t i = first + threadIdx.x; i < end; i += kSumThreads) z2 += (double)w.zsum[i];
  mass += __shfl_xor(mass, kColumns, 64);  // a wave has two threads of an expert
  count += __shfl_xor(count, kColumns, 64);
  if (lane < kColumns) {
    red[wave][col] = mass;
    redc[wave][col] = count;
  }
  __syncthreads();
  double balance = 0.0;
  if (group == 0) {
#pragma unroll
    for (int w2 = 1; w2 < WAVES; ++w2) {
      mass += red[w2][col];
      count += redc[w2][col];
    }
    if (e < E) {
      const double ae =
          n > 0 ? (double)E * (double)count / ((double)k * (double)n * (double)n * (double)w.total[0]) : 0.0;
      a[(int64_t)s * E + e] = (float)ae;
      balance = ae * mass;
    }
  }
  auto block_sum = [&](double& u, double& v) {  // in thread 0
    u = lanes_sum<64>(u);
    v = lanes_sum<64>(v);
    if (lane == 0) {
      wave_sums[wave][0] = u;
      wave_sums[wave][1] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kSumThreads / 64; ++i) {
        u += wave_sums[i][0];
        v += wave_sums[i][1];
      }
    }
    __syncthreads();
  };
  block_sum(balance, z2);
  const int parts = gridDim.x * gridDim.y;
  if (threadIdx.x == 0) {
    double* p = w.part + 2 * ((int64_t)s * gridDim.y + cb);
    __hip_atomic_store(p, balance, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(p + 1, z2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __threadfence();
    last = atomicAdd(w.done, 1) == parts - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  balance = z2 = 0.0;
  for (int i = threadIdx.x; i < parts; i += kSumThreads) {
    balance += __hip_atomic_load(&w.part[2 * (int64_t)i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    z2 += __hip_atomic_load(&w.part[2 * (int64_t)i + 1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  block_sum(balance, z2);
  if (threadIdx.x == 0) {
    const double inv = w.total[1] > 0 ? 1.0 / (double)w.total[1] : 0.0;
    out[0] = (float)balance;
    out[1] = (float)(z2 * inv);
    *inv_tokens = (float)inv;
  }
}

// A lane's numbers of a row of E in f32, at the places of its logits (of type LT), 0 past it; rows of whole 16 bytes in
// fours.
template <int VPL, int STEP, typename LT>
__device__ __forceinline__ void load_of(const float* __restrict__ row, int e0, int E, bool live, float (&v)[VPL]) {
  const bool vec = E % 4 == 0;
#pragma unroll
  for (int q = 0; q < VPL; q += 4) {
    const int e = e0 + lane_element<VPL, STEP, LT>(q);
    if (vec && live && e < E) {
      const float4 x = *reinterpret_cast<const float4*>(row + e);
      v[q] = x.x, v[q + 1] = x.y, v[q + 2] = x.z, v[q + 3] = x.w;
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) v[q + u] = !vec && live && e + u < E ? row[e + u] : 0.f;
    }
  }
}

// A workgroup has ROWS tokens at a time, a quarter of a tile or so: as many workgroups as keep every CU's loads going.
template <int LPR, int VPL, bool SOFT, typename LT>
__global__ __launch_bounds__(64 * kWaves) void losses_backward_kernel(const LT* __restrict__ logits, int E, bool vec,
                                                                      Sequences seq, const float* __restrict__ a,
                                                                      const float* __restrict__ inv_tokens,
                                                                      const float* __restrict__ g_balance,
                                                                      const float* __restrict__ g_z,
                                                                      LT* __restrict__ dz) {
  constexpr int TPW = 64 / LPR, STEP = kSpread<LPR, VPL, LT>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane / LPR, e0 = spread_first<VPL, LT>(lane % LPR);
  const int64_t tw = ((int64_t)blockIdx.x * kWaves + wave) * TPW, t = tw + row;
  if (tw >= seq.T) return;
  const bool there = t < seq.T;
  float z[VPL];
  load_lane<VPL, STEP>(logits + t * E, e0, E, vec, there, -INFINITY, z);
  const float gb = g_balance ? *g_balance : 0.f, gz = g_z ? 2.f * *g_z * *inv_tokens : 0.f;
  int s = seq.after(tw);
  while (s < seq.S && seq.at(s + 1) <= t) ++s;
  const bool in = there && s < seq.S && seq.at(s) <= t;
  float as[VPL];
  load_of<VPL, STEP, LT>(a + (int64_t)s * E, e0, E, in, as);
  float ph[VPL], soft[VPL], rest[VPL], dot = 0.f;
  const float lse = token_row<LPR, VPL, SOFT>(z, ph, soft, rest);
#pragma unroll
  for (int q = 0; q < VPL; ++q) dot += ph[q] * as[q];
  dot = lanes_sum<LPR>(dot);
#pragma unroll
  for (int q = 0; q < VPL; ++q) {
    float d = gb * (ph[q] * (as[q] - dot));
    if constexpr (!SOFT) d *= rest[q];
    if (g_z) d += gz * lse * soft[q];  // (not 0 times an lse of inf)
    z[q] = in ? d : 0.f;
  }
  if (there) store_lane<VPL, STEP>(dz + t * E, e0, E, vec, z);
}

int check_sizes(const char* what, int dtype, int64_t T, int E, int score, const void* cu, int64_t S) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "%s: logits dtype %d", what, dtype);
  ZMOE_REQUIRE(T >= 0 && E >= 1 && E <= 1024, ZMOE_ERR_SHAPE, "%s: need 1 <= E <= 1024 (E=%d)", what, E);
  ZMOE_REQUIRE(score == ZMOE_SCORE_SIGMOID || score == ZMOE_SCORE_SOFTMAX, ZMOE_ERR_SHAPE, "%s: score %d", what, score);
  ZMOE_REQUIRE(S >= 1 && S <= ZMOE_ROUTER_LOSSES_MAX_SEQUENCES, ZMOE_ERR_SHAPE, "%s: need 1 to %d sequences (%lld)", what,
               ZMOE_ROUTER_LOSSES_MAX_SEQUENCES, (long long)S);
  ZMOE_REQUIRE(cu || S == 1, ZMOE_ERR_NULL, "%s: null pointer", what);
  // the backward has four tokens a workgroup where E > 256
  ZMOE_REQUIRE(launch_fits(cdiv(T, kWaves) + 1, 64 * kWaves), ZMOE_ERR_SHAPE, "%s: too many tokens for one launch", what);
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
  const bool vec = rows_on_16(logits, E, E, logits_dtype);
  by_lanes(E, score == ZMOE_SCORE_SOFTMAX, logits_dtype, [&](auto lpr, auto vpl, auto soft, auto lt) {
    using LT = decltype(lt);
    hipLaunchKernelGGL((losses_tile_kernel<decltype(lpr)::value, decltype(vpl)::value, decltype(soft)::value, LT>),
                       dim3((unsigned)(cdiv(T, kTile) + 1)), dim3(64 * kWaves), 0, as_stream(stream), (const LT*)logits,
                       topk_idx, E, k, vec, seq, w);
  });
  if (const int rc = check_launch("router_losses")) return rc;
  hipLaunchKernelGGL(losses_sum_kernel, dim3((unsigned)S, (unsigned)column_blocks(E)), dim3(kSumThreads), 0,
                     as_stream(stream), E, k, seq, w, seq_grad, losses, inv_tokens);
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
  ZMOE_REQUIRE(E % 4 != 0 || aligned16(seq_grad), ZMOE_ERR_ALIGN, "router_losses_backward: seq_grad must be 16-byte aligned");
  const Sequences seq{cu_seqlens, cu_int64 != 0, (int)S, T};
  const bool vec = rows_on_16(logits, E, E, logits_dtype) && rows_on_16(d_logits, E, E, logits_dtype);
  by_lanes(E, score == ZMOE_SCORE_SOFTMAX, logits_dtype, [&](auto lpr, auto vpl, auto soft, auto lt) {
    using LT = decltype(lt);
    constexpr int rows = kWaves * (64 / decltype(lpr)::value);
    hipLaunchKernelGGL((losses_backward_kernel<decltype(lpr)::value, decltype(vpl)::value, decltype(soft)::value, LT>),
                       dim3((unsigned)cdiv(T, rows)), dim3(64 * kWaves), 0, as_stream(stream), (const LT*)logits, E, vec,
                       seq, seq_grad, inv_tokens, d_balance, d_z, (LT*)d_logits);
  });
  return check_launch("router_losses_backward");
}
