// What the routing kernels share: sort keys of scores, the sigmoid rounded once, tokens in rows of lanes, reductions over
// them.
#pragma once

#include <type_traits>

#include "zmoe_internal.h"

namespace zmoe {

// Sort key of a routing candidate's score; a larger key takes an earlier slot. A monotone
// image of the biased score: every NaN canonicalised above +inf, -0 folded into +0. Equal
// scores go to the lower expert. Key 0 marks a taken (or padding) candidate: a real
// score's key is at least 0x007fffff (that of -inf).
__device__ __forceinline__ uint32_t score_key(float s) {
  uint32_t b = __float_as_uint(s);
  b = s != s ? 0x7fffffffu : b;  // selects, not branches
  b = s == 0.f ? 0u : b;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Logits at or below this value give probability 0: there torch's sigmoid, which forms
// 1 / (1 + exp(-z)) in fp32, overflows exp(-z) to inf (fp32 exp overflows from
// 88.72283935546875 up; the true probabilities, below 2.9e-39, would be subnormal).
constexpr float kSigmoidZeroBelow = -88.72283935546875f;

// Below this |z| the probability comes from p = 0.5 + z/4 - z^3/48 + ...: 0.5 + z/4 is
// exact in double, and the cubic term cannot move it across an fp32 rounding midpoint
// unless it lies exactly on one (its distance from a midpoint is a multiple of z's last
// bit / 4, more than |z|^3/48 here).
constexpr float kSigmoidSeriesBelow = 0x1p-12f;

// sigmoid correctly rounded to float: for |z| < kSigmoidSeriesBelow, 0.5 + z/4 rounded to
// nearest with an exact tie going to the side the cubic term puts the true value on (down
// for z > 0, up for z < 0; many small bf16 logits land on such ties, where a double
// evaluation's rounding would hang on the last bit of its exp); otherwise
// 1 / (1 + exp(-z)) in double, rounded once; 0 at or below kSigmoidZeroBelow.
__device__ __forceinline__ float sigmoid_f64(float z) {
  if (z <= kSigmoidZeroBelow) return 0.f;
  if (fabsf(z) < kSigmoidSeriesBelow) {
    const double s = 0.5 + 0.25 * (double)z;
    const float f = (float)s;
    const double fd = (double)f;
    if (fd != s) {  // f > 0: its other neighbour around s is one bit pattern up or down
      const float o = __uint_as_float(__float_as_uint(f) + (fd < s ? 1u : 0xffffffffu));
      if (fabs(s - fd) == fabs((double)o - s)) return z > 0.f ? fminf(f, o) : fmaxf(f, o);
    }
    return f;
  }
  return (float)(1.0 / (1.0 + exp(-(double)z)));
}

// Wave-wide max of a 32-bit key, the same value in every lane: DPP within rows of 16
// (xor 1, xor 2, half mirror, mirror: no LDS round trip), then the four row maxima
// through readlane.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x141, 0xF, 0xF, false));  // row_half_mirror
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x140, 0xF, 0xF, false));  // row_mirror
  const uint32_t r0 = (uint32_t)__builtin_amdgcn_readlane((int)v, 0);
  const uint32_t r1 = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t r2 = (uint32_t)__builtin_amdgcn_readlane((int)v, 32);
  const uint32_t r3 = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  return max(max(r0, r1), max(r2, r3));
}

// Reductions over rows of LPR = 16 or 8 lanes by DPP (xor 1, xor 2, mirror within 8 lanes,
// mirror within 16); every lane of a row ends with the row's result.
template <int LPR>
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, true));
  if (LPR == 16) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, true));
  return v;
}
template <int LPR>
__device__ __forceinline__ uint32_t row_min_u32(uint32_t v) {
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0xB1, 0xF, 0xF, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x4E, 0xF, 0xF, false));
  v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x141, 0xF, 0xF, false));
  if (LPR == 16) v = min(v, (uint32_t)__builtin_amdgcn_update_dpp(-1, (int)v, 0x140, 0xF, 0xF, false));
  return v;
}
template <int LPR>
__device__ __forceinline__ float row_sum_f32(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, true));
  if (LPR == 16) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, true));
  return v;
}

// e^x in double, x below 709 (e^-745 and less are 0; NaN stays): x = n ln 2 + r with |r| <= ln 2 / 2 by the reduction of Cody and
// Waite (ln 2 as a sum of two numbers, of which the first has so few bits that n times it is exact), and Taylor's polynomial
// of degree 12, whose first missing term is below 2^-52.
__device__ __forceinline__ double exp_f64(double x) {
  x = x < -760.0 ? -760.0 : x;
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0x1.62e42fee00000p-1, x);
  r = fma(n, -0x1.a39ef35793c76p-33, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return ldexp(p, (int)n);
}
// 1 / x in double for a normal x with a normal reciprocal, to a rounding or two: two steps of Newton's from v_rcp_f64.
__device__ __forceinline__ double rcp_f64(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = fma(fma(-x, y, 1.0), y, y);
  return fma(fma(-x, y, 1.0), y, y);
}
// 1 - sigmoid(z) rounded once, with all its digits where the sigmoid is near 1 (past 100 below every f32).
__device__ __forceinline__ float sigmoid_complement(float z) {
  return (float)rcp_f64(1.0 + exp_f64((double)(z > 100.f ? 100.f : z)));
}
// sigmoid_f64 of a lane's logits by these two, all at once (their chains overlap); exact ties near 0 apart.
template <int N>
__device__ __forceinline__ void sigmoids_rounded(const float (&z)[N], float (&p)[N]) {
  bool small = false;
#pragma unroll
  for (int q = 0; q < N; ++q) {
    const float v = (float)rcp_f64(1.0 + exp_f64(-(double)z[q]));
    p[q] = z[q] <= kSigmoidZeroBelow ? 0.f : v;
    small |= fabsf(z[q]) < kSigmoidSeriesBelow;
  }
  if (small) {
#pragma unroll
    for (int q = 0; q < N; ++q)
      if (fabsf(z[q]) < kSigmoidSeriesBelow) p[q] = sigmoid_f64(z[q]);
  }
}

// e^x in f32 by the hardware's exp2: off by |x| + 1 roundings (the product with log2 e, and the instruction); -inf gives 0,
// +inf inf, NaN stays. Where no selection hangs on it.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// A row of 16 lanes and its neighbour's value: two rows' results together, in 32 lanes.
struct Two {
  uint32_t a, b;
};
__device__ __forceinline__ Two rows_swapped(uint32_t v) {
  const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return {(uint32_t)both[0], (uint32_t)both[1]};
}

// Over the LPR (8, 16, 32 or 64) lanes of a row; every lane gets the result.
template <int LPR>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  if constexpr (LPR == 64) return wave_max_u32(v);
  else if constexpr (LPR == 32) {
    const Two t = rows_swapped(row_max_u32<16>(v));
    return max(t.a, t.b);
  } else return row_max_u32<LPR>(v);
}
template <int LPR>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
  if constexpr (LPR == 64) return ~wave_max_u32(~v);
  else if constexpr (LPR == 32) {
    const Two t = rows_swapped(row_min_u32<16>(v));
    return min(t.a, t.b);
  } else return row_min_u32<LPR>(v);
}
// (xor 1, xor 2, mirrors within 8 and 16 lanes as above; between rows of 16 by shuffles)
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const int64_t b = __double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, true);
  return __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  if (LPR >= 16) v += dpp_f32<0x140>(v);
  if (LPR >= 32) {
    const Two t = rows_swapped(__float_as_uint(v));
    v = __uint_as_float(t.a) + __uint_as_float(t.b);
  }
  if (LPR == 64) v += __shfl_xor(v, 32, 64);
  return v;
}
template <int LPR>
__device__ __forceinline__ double lanes_sum(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  if (LPR >= 16) v += dpp_f64<0x140>(v);
  if (LPR >= 32) v += __shfl_xor(v, 16, 64);
  if (LPR == 64) v += __shfl_xor(v, 32, 64);
  return v;
}
template <int LPR>
__device__ __forceinline__ int64_t lanes_sum(int64_t v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int LPR>
__device__ __forceinline__ float lanes_fmax(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  v = fmaxf(v, dpp_f32<0x4E>(v));
  v = fmaxf(v, dpp_f32<0x141>(v));
  if (LPR >= 16) v = fmaxf(v, dpp_f32<0x140>(v));
  if (LPR >= 32) {
    const Two t = rows_swapped(__float_as_uint(v));
    v = fmaxf(__uint_as_float(t.a), __uint_as_float(t.b));
  }
  if (LPR == 64) v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}

// Chunks of a lane's VPL elements: 16 bytes, or four bf16 where a lane's elements are no whole 16.
template <int VPL, typename LT>
struct LaneChunk {
  static constexpr int N = VPL * sizeof(LT) % 16 == 0 ? 16 / sizeof(LT) : 4;
  static_assert(VPL % N == 0 && N % 4 == 0, "lanes of whole chunks");
};

// x as a value that the compiler knows nothing of (so nothing computed from it leaves the loop).
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Where a lane's element q lies: VPL consecutive ones (STEP 0), or chunks STEP elements apart, so that a row's lanes
// read and write consecutive chunks (from the lane's first, `spread_first`): f32 grads of 32749 x 256 logits 18.2 us against
// 21.8 with 64 bytes from lane to lane.
template <int VPL, int STEP, typename LT>
__device__ __forceinline__ constexpr int lane_element(int q) {
  constexpr int N = LaneChunk<VPL, LT>::N;
  return STEP ? q / N * STEP + q % N : q;
}
template <int LPR, int VPL, typename LT>
constexpr int kSpread = LPR * LaneChunk<VPL, LT>::N;
template <int VPL, typename LT>
__device__ __forceinline__ int spread_first(int lane_of_row) {
  return lane_of_row * LaneChunk<VPL, LT>::N;
}

// A lane's elements of a row of E from e0 on, `fill` past it. vec: rows are whole 16-byte chunks and lie on 16 (so a
// lane's chunks are wholly in the row or out of it).
template <int VPL, int STEP = 0, typename LT>
__device__ __forceinline__ void load_lane(const LT* __restrict__ row, int e0, int E, bool vec, bool live, float fill,
                                          float (&v)[VPL]) {
  constexpr int N = LaneChunk<VPL, LT>::N;
  if (vec) {
#pragma unroll
    for (int c = 0; c < VPL / N; ++c) {
      const int e = e0 + lane_element<VPL, STEP, LT>(c * N);
      if (live && e < E) {
        if constexpr (N * sizeof(LT) == 16) {
          unpack_chunk(*reinterpret_cast<const uint4*>(row + e), &v[c * N], LT{});
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(row + e);
          v[c * N] = __uint_as_float(x.x << 16), v[c * N + 1] = __uint_as_float(x.x & 0xffff0000u);
          v[c * N + 2] = __uint_as_float(x.y << 16), v[c * N + 3] = __uint_as_float(x.y & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int u = 0; u < N; ++u) v[c * N + u] = fill;
      }
    }
  } else {
    const int have = live ? opaque(E - e0) : 0;  // (not kept as VPL masks over a caller's loop: registers)
#pragma unroll
    for (int q = 0; q < VPL; ++q) {
      const int at = lane_element<VPL, STEP, LT>(q);
      v[q] = at < have ? to_f32(row[e0 + at]) : fill;
    }
  }
}
template <int VPL, int STEP = 0, typename LT>
__device__ __forceinline__ void store_lane(LT* __restrict__ row, int e0, int E, bool vec, const float (&v)[VPL]) {
  constexpr int N = LaneChunk<VPL, LT>::N;
  if (vec) {
#pragma unroll
    for (int c = 0; c < VPL / N; ++c) {
      const int e = e0 + lane_element<VPL, STEP, LT>(c * N);
      if (e >= E) continue;
      if constexpr (N * sizeof(LT) == 16) {
        *reinterpret_cast<uint4*>(row + e) = pack_chunk(&v[c * N], LT{});
      } else {
        *reinterpret_cast<uint2*>(row + e) =
            make_uint2(pack_bf16x2(v[c * N], v[c * N + 1]), pack_bf16x2(v[c * N + 2], v[c * N + 3]));
      }
    }
  } else {
    const int have = opaque(E - e0);
#pragma unroll
    for (int q = 0; q < VPL; ++q) {
      const int at = lane_element<VPL, STEP, LT>(q);
      if (at < have) row[e0 + at] = from_f32<LT>(v[q]);
    }
  }
}

// f(lanes of a row, experts a lane, softmax?, logits' type), the layout by the number of experts: the fewest lanes that
// hold them at 16 a lane (up to 128 at 8: 32768 tokens are routed in 12.9-13.4 us by 16 lanes of 8, 11.7-13.4 by 8 of 16, 3
// tokens in 4 and 5.7; 32768 of 512 experts in 46-52 by 32 lanes of 16, 62-65 by 64 of 8).
template <typename F>
void by_lanes(int E, bool soft, int dtype, F&& f) {
  auto typed = [&](auto lpr, auto vpl) {
    auto scored = [&](auto lt) {
      if (soft) f(lpr, vpl, std::true_type{}, lt);
      else f(lpr, vpl, std::false_type{}, lt);
    };
    if (dtype == ZMOE_DTYPE_BF16) scored(uint16_t{});
    else scored(float{});
  };
  using I8 = std::integral_constant<int, 8>;
  using I12 = std::integral_constant<int, 12>;
  using I16 = std::integral_constant<int, 16>;
  using I32 = std::integral_constant<int, 32>;
  using I64 = std::integral_constant<int, 64>;
  if (E <= 64) typed(I8{}, I8{});
  else if (E <= 96) typed(I8{}, I12{});
  else if (E <= 128) typed(I16{}, I8{});
  else if (E <= 192) typed(I16{}, I12{});
  else if (E <= 256) typed(I16{}, I16{});
  else if (E <= 512) typed(I32{}, I16{});
  else typed(I64{}, I16{});
}

// Whether a matrix of rows of E, ld apart, may be accessed in 16-byte chunks.
inline bool rows_on_16(const void* base, int64_t ld, int E, int dtype) {
  const int size = dtype_size(dtype);
  return aligned16(base) && (ld * size) % 16 == 0 && (E * size) % 16 == 0;
}

}  // namespace zmoe
