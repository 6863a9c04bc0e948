// An AdamW step over many tensors at once (zmoe_adamw), with moments in 32 or in 8 bits, and the grads' global norm with
// the factor that clips it (zmoe_sum_squares, zmoe_clip_factor).
//   g' = clip g,  m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2
//   p' = p - lr wd p - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
// in f32, p' rounded once to its type. t is each tensor's own count on the device, so a captured step counts on.
//
// 8 bits: a block of 256 consecutive elements keeps its largest magnitude A in f32 and for each element the code q of
//   m = sign q^2 A / 127^2 (signed),   v = q^4 A / 255^4 (unsigned)
// rounded to f32: codes are spaced evenly in sqrt(|m|) and v^(1/4), so that a moment 10^-4 of the block's largest still has
// one (16 bits of range under a root, as large as the step of an element with the largest moments; evenly spaced codes would
// take all below 1 / 254 to 0). A code is the nearest in the root's domain, half-way ones up: that is the comparison of
// (2q - 1)^2 A with 4 127^2 |m| (and of fourth powers), which double holds exactly (v: to 2^-53), so the same codes come
// from any evaluation that is right to a few bits. v' > 0 never becomes 0: its root stands under the step. The scale is
// the magnitude itself, not a power of two, for a moment that decays by 0.1% a step has to be able to. The moments are
// formed in double and rounded to f32 before the step and the codes are taken from them; a moment that is not
// finite makes its block's scale so, and all of the block's moments NaN.
//
// Everything is one pass over memory: 28 bytes an element (f32, 32 bits), 16 (f32, 8 bits), 22 and 10 (bf16). Tensors'
// pointers travel in the launches' arguments, so nothing is copied to the device and a graph keeps them. The norm is a
// pass of its own (302 M f32 elements 240 us, 5.0 TB/s), for the clip has to be known before the first element moves.
#include <cmath>
#include <type_traits>

#include "zmoe_route.h"  // row_max_u32

namespace zmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;   // elements with one scale
constexpr int kBlocks = 8;    // of them in a workgroup's chunk: two a wave
constexpr int kChunk = kBlock * kBlocks;
constexpr int kMomentBlocks = 16;  // the same where moments are decoded: four (302 M elements 541 us, with two 582)
constexpr int kMomentChunk = kBlock * kMomentBlocks;
constexpr int kTensors = 48;  // in a launch's arguments (under 4 KB)
constexpr int kNormChunk = 16384;
constexpr int kNormTensors = 128;

struct Table {
  zmoe_adamw_tensor t[kTensors];
  int32_t start[kTensors + 1];  // first chunk of each tensor in this launch
  uint64_t vec;                 // bit i: tensor i's arrays lie on whole vectors
  int count;
};

struct Hyper {
  double b1, b2, c1, c2;  // c = 1 - b
  float b1f, b2f, c1f, c2f, eps;
};

// The tensor that a launch's chunk belongs to.
__device__ __forceinline__ int owner_of(const int32_t* start, int count, int chunk) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ------------------------------------------------------------------ the step count and what follows from it
struct StepTable {
  float* step[kNormTensors];
  int count;
};

// coef[i] = {lr / (1 - b1^t), 1 / sqrt(1 - b2^t), lr wd, clip} with t counted on.
__global__ void adamw_prepare_kernel(const StepTable s, const float* lr_ptr, double lr, double b1, double b2, double wd,
                                     const float* clip, float4* coef) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= s.count) return;
  const float t = *s.step[i] + 1.f;
  *s.step[i] = t;
  const double rate = lr_ptr ? (double)*lr_ptr : lr;
  coef[i] = make_float4((float)(rate / (1.0 - pow(b1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(b2, (double)t))),
                        (float)(rate * wd), clip ? *clip : 1.f);
}

// ------------------------------------------------------------------ codes
constexpr int kTop2 = 127, kTop4 = 255;
constexpr double kDiv2 = 127.0 * 127.0, kDiv4 = 255.0 * 255.0 * 255.0 * 255.0;

// A / div rounded once: the product with the reciprocal, mended by what it leaves.
__device__ __forceinline__ double unit_of(float A, double div, double inv) {
  const double q = (double)A * inv;
  return fma(fma(-q, div, (double)A), inv, q);
}
__device__ __forceinline__ double unit2(float A) { return unit_of(A, kDiv2, 1.0 / kDiv2); }
__device__ __forceinline__ double unit4(float A) { return unit_of(A, kDiv4, 1.0 / kDiv4); }
// x a + y b, each step rounded: with a fused multiply-add the sum differs in its last bit, and with grads of few bits one
// value in a thousand lies half-way between two f32 numbers, where that decides.
__device__ __forceinline__ float blend(double x, double a, double y, double b) {
#pragma clang fp contract(off)
  const double xa = x * a, yb = y * b;
  return (float)(xa + yb);
}

// The f32 values of codes: sign q^2 unit, q^4 unit.
__device__ __forceinline__ float value2(int q, double unit) {
  const double x = (double)q;
  return (float)(x * fabs(x) * unit);
}
__device__ __forceinline__ float value4(uint32_t q, double unit) {
  const double x = (double)q, x2 = x * x;
  return (float)(x2 * x2 * unit);
}

// A code's place in the root's domain: the code is the whole number next to it, unless half-way between two lies within
// kNear2 or kNear4. What the hardware's reciprocals and roots (one unit in the last place, 2^-23) and the products make
// of it: 127 times 2.4 2^-23 = 3.7e-5 at most, and 255 times 2.8 2^-23 = 8.4e-5 from the step's own root of v
// (root: 1, the other's reciprocal root: 1, their product: 1/2; halved by the second root: 1.25, its own 1, the product 1/2).
constexpr float kNear2 = 0x1p-14f, kNear4 = 0x1p-13f;
__device__ __forceinline__ float place2(float mag, float inv) {
  return __builtin_amdgcn_sqrtf(mag * inv) * (float)kTop2;
}
__device__ __forceinline__ float place4(float root, float inv_root) {
  return __builtin_amdgcn_sqrtf(root * inv_root) * (float)kTop4;
}

// The code itself, from one that is off by one at most: set right by the borders on its two sides.
__device__ __forceinline__ int settle2(int q, float mag, double A) {
  const double at = (double)mag * (4.0 * kDiv2);
  const int l = 2 * q - 1, h = 2 * q + 1;
  return q + (int)(q < kTop2 && at > 0.0 && (double)(h * h) * A <= at) - (int)(q > 0 && (double)(l * l) * A > at);
}
__device__ __forceinline__ int settle4(int q, float mag, double A) {
  const double at = (double)mag * (16.0 * kDiv4);
  const double l = (double)((2 * q - 1) * (2 * q - 1)), h = (double)((2 * q + 1) * (2 * q + 1));
  return q + (int)(q < kTop4 && at > 0.0 && h * h * A <= at) - (int)(q > 0 && l * l * A > at);
}

// The codes of a lane's N elements of each moment (v > 0 at least 1), the bytes of dwords; r = root(v). A block whose
// largest magnitude has no f32 reciprocal, or so small a second moment that a root taken for 0 could have a code, takes its
// estimates from double; one that is not finite has any codes (its scale says it all).
template <int N>
__device__ __forceinline__ void encode(const float (&m)[N], const float (&v)[N], const float (&r)[N], float Am, float Av,
                                       uint32_t (&qm)[N / 4], uint32_t (&qv)[N / 4]) {
  const bool odd = (Am > 0.f && Am < 0x1p-100f) || Am > 0x1p100f || (Av > 0.f && Av < 0x1p-88f) || Av > 0x1p100f;
  const float im = Am > 0.f ? __builtin_amdgcn_rcpf(Am) : 0.f, iv = Av > 0.f ? __builtin_amdgcn_rsqf(Av) : 0.f;
  float far_m = 0.f, far_v = 0.f;  // from the nearest whole number, at most
  float cm[N], cv[N];              // magnitudes
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = place2(fabsf(m[e]), im), z = place4(r[e], iv);
    cm[e] = rintf(y);
    cv[e] = rintf(z);
    far_m = fmaxf(far_m, fabsf(y - cm[e]));
    far_v = fmaxf(far_v, fabsf(z - cv[e]));
  }
  if (odd) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      cm[e] = Am > 0.f ? rintf(sqrtf((float)(fabs((double)m[e]) / (double)Am)) * (float)kTop2) : 0.f;
      cv[e] = Av > 0.f ? rintf(sqrtf(sqrtf((float)((double)v[e] / (double)Av))) * (float)kTop4) : 0.f;
    }
    far_m = far_v = 0.5f;
  }
  if (far_m > 0.5f - kNear2) {  // one lane in a thousand
#pragma unroll
    for (int e = 0; e < N; ++e) cm[e] = (float)settle2((int)cm[e], fabsf(m[e]), (double)Am);
  }
  if (far_v > 0.5f - kNear4) {
#pragma unroll
    for (int e = 0; e < N; ++e) cv[e] = (float)settle4((int)cv[e], v[e], (double)Av);
  }
#pragma unroll
  for (int d = 0; d < N / 4; ++d) {
    int c[4];
    qv[d] = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * d + e;
      c[e] = (int)copysignf(cm[i], m[i]);
      const float some = __builtin_amdgcn_fmed3f(__builtin_ldexpf(v[i], 200), 0.f, 1.f);  // 1 where v > 0, else 0
      qv[d] = __builtin_amdgcn_cvt_pk_u8_f32(fmaxf(cv[i], some), e, qv[d]);
    }
    const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
    qm[d] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);  // their low bytes
  }
}

// Max over each half of a wave, in its 32 lanes: within rows of 16 by DPP, then a row and its neighbour exchanged.
__device__ __forceinline__ uint32_t half_max_u32(uint32_t v) {
  v = row_max_u32<16>(v);
  const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max((uint32_t)both[0], (uint32_t)both[1]);
}

// A square root to one rounding of f32. v_sqrt_f32 takes subnormals for 0 (SCALED false): their roots, below 2^-63, stand in
// the denominator as at most 2^-63 / sqrt(1 - b2), 2^-25 of an eps of 2^-38 / sqrt(1 - b2) or more.
template <bool SCALED>
__device__ __forceinline__ float root(float v) {
  if constexpr (!SCALED) return __builtin_amdgcn_sqrtf(v);
  const bool small = v < 0x1p-96f;
  const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v);
  return small ? r * 0x1p-16f : r;
}

// The parameter after the step (r: the root of v): the quotient by v_rcp_f32, whose argument has to be a normal number. Without
// an eps, or with one that is none (SCALED), it may not be: then a division, and no change where there is no moment.
template <bool SCALED>
__device__ __forceinline__ float stepped(float w, float m, float r, const float4& c, float eps) {
  const float kept = fmaf(-c.z, w, w), d = fmaf(r, c.y, eps);
  if constexpr (SCALED)
    if (d < 0x1p-126f) return m == 0.f ? kept : kept - c.x * m / d;
  return fmaf(-(c.x * m), __builtin_amdgcn_rcpf(d), kept);
}

// ------------------------------------------------------------------ elements
// Four elements i .. i + 3 of n; vec: all of them there and on a whole vector (the same in a wave).
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t i, int64_t n, bool vec, float (&v)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 x = *reinterpret_cast<const float4*>(p + i);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(p + i);
      v[0] = __uint_as_float(x.x << 16), v[1] = __uint_as_float(x.x & 0xffff0000u);
      v[2] = __uint_as_float(x.y << 16), v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = i + u < n ? to_f32(p[i + u]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, const float (&v)[4]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[0], v[1], v[2], v[3]);
    else *reinterpret_cast<uint2*>(p + i) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
  } else {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u < n) p[i + u] = from_f32<T>(v[u]);
  }
}
// Eight of a block's last elements or of arrays that do not lie on whole vectors.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int i, int64_t n, float (&v)[8]) {
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = i + u < n ? to_f32(p[i + u]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int i, int64_t n, bool vec, const float (&v)[8]) {
  if (vec) {
    constexpr int VC = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < 8 / VC; ++c) *reinterpret_cast<uint4*>(p + i + c * VC) = pack_chunk(&v[c * VC], T{});
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < n) p[i + u] = from_f32<T>(v[u]);
  }
}
// Eight codes as the bytes of two dwords.
__device__ __forceinline__ void load_codes8(const uint8_t* p, int i, int64_t n, uint32_t (&c)[2]) {
  c[0] = c[1] = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (i + u < n) c[u >> 2] |= (uint32_t)p[i + u] << (8 * (u & 3));
}
__device__ __forceinline__ void store_codes8(uint8_t* p, int i, int64_t n, bool vec, const uint32_t (&c)[2]) {
  if (vec) {
    *reinterpret_cast<uint2*>(p + i) = make_uint2(c[0], c[1]);
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u < n) p[i + u] = (uint8_t)(c[u >> 2] >> (8 * (u & 3)));
  }
}
// Four codes as the bytes of a dword.
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int64_t i, int64_t n, bool vec) {
  if (vec) return *reinterpret_cast<const uint32_t*>(p + i);
  uint32_t c = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (i + u < n) c |= (uint32_t)p[i + u] << (8 * u);
  return c;
}

// Moments in 32 bits: memory alone (302 M f32 elements 1544-1564 us, 5.4 TB/s, as many of bf16 1247, 5.3 TB/s); four consecutive elements a lane, a wave's
// two blocks read before the first is written.
template <typename T, bool SCALED>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Table tab, const Hyper h,
                                                         const float4* __restrict__ coef) {
  const int which = owner_of(tab.start, tab.count, blockIdx.x);
  const zmoe_adamw_tensor& t = tab.t[which];
  const bool wide = (tab.vec >> which) & 1;
  const float4 c = coef[which];
  const int64_t n = t.n;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)(blockIdx.x - tab.start[which]) * kBlocks + wave * (kBlocks / 4);
#pragma unroll 2
  for (int u = 0; u < kBlocks / 4; ++u) {
    const int64_t at = (first + u) * kBlock, left = n - at;
    if (left <= 0) break;
    const bool vec = wide && left >= kBlock;
    const int i = lane * 4;
    T* p = (T*)t.param + at;
    float *pm = (float*)t.exp_avg + at, *pv = (float*)t.exp_avg_sq + at;
    float w[4], gr[4], m[4], v[4];
    load4(p, i, left, vec, w);
    load4((const T*)t.grad + at, i, left, vec, gr);
    load4(pm, i, left, vec, m);
    load4(pv, i, left, vec, v);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gs = gr[e] * c.w;
      m[e] = fmaf(h.b1f, m[e], h.c1f * gs);
      v[e] = fmaf(h.b2f, v[e], h.c2f * (gs * gs));
      w[e] = stepped<SCALED>(w[e], m[e], root<SCALED>(v[e]), c, h.eps);
    }
    store4(pm, i, left, vec, m);
    store4(pv, i, left, vec, v);
    store4(p, i, left, vec, w);
  }
}

// What a lane reads of two whole blocks, as it lies in memory: all on its way at once (with a branch for whole vectors at
// each of the reads they come one after the other: 24.5 M bf16 elements 72 us against 61).
template <typename T>
struct Raw8 {
  uint4 p[8 * sizeof(T) / 16], g[8 * sizeof(T) / 16];
  uint2 m, v;
  float am, av;
  __device__ __forceinline__ void load(const zmoe_adamw_tensor& t, int64_t block, int lane) {
    const int64_t at = block * kBlock + lane * 8;
#pragma unroll
    for (int c = 0; c < (int)(8 * sizeof(T) / 16); ++c) {
      g[c] = reinterpret_cast<const uint4*>((const T*)t.grad + at)[c];
      p[c] = reinterpret_cast<const uint4*>((const T*)t.param + at)[c];
    }
    m = *reinterpret_cast<const uint2*>((const uint8_t*)t.exp_avg + at);
    v = *reinterpret_cast<const uint2*>((const uint8_t*)t.exp_avg_sq + at);
    am = t.scale_avg[block + (lane >> 5)];
    av = t.scale_sq[block + (lane >> 5)];
  }
  __device__ __forceinline__ void unpack(float (&w)[8], float (&gr)[8], uint32_t (&qm)[2], uint32_t (&qv)[2], float& a,
                                         float& b) const {
    constexpr int VC = 16 / sizeof(T);
#pragma unroll
    for (int c = 0; c < 8 / VC; ++c) {
      unpack_chunk(p[c], &w[c * VC], T{});
      unpack_chunk(g[c], &gr[c * VC], T{});
    }
    qm[0] = m.x, qm[1] = m.y, qv[0] = v.x, qv[1] = v.y;
    a = am;
    b = av;
  }
};

// Moments in 8 bits: a wave has two blocks at once, eight consecutive elements a lane, so that what is done once for a
// block (the largest magnitudes over its lanes, the scales' quotients) is shared by twice as many. The arithmetic is the
// bound as much as memory: 503 vector instructions a wave (counted), 42 of them roots and reciprocals at a quarter of the rate
// (doubles run at f32's), 50 us of 61 for 24.5 M bf16 elements (4.0 TB/s); 302 M f32 elements 900 us, 5.4 TB/s. One pair a
// wave: with two, the second's reads under way while the first is worked on, 28 more registers cost more than that
// hides (repeated on the same tensors, 24.5 M bf16 elements 51 and 56 us, 100 M f32 295 and 299).
template <typename T, bool SCALED>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(const Table tab, const Hyper h,
                                                          const float4* __restrict__ coef) {
  static_assert(kBlocks == 2 * kThreads / 64);
  const int which = owner_of(tab.start, tab.count, blockIdx.x);
  const zmoe_adamw_tensor& t = tab.t[which];
  const float4 c = coef[which];
  const double clip = (double)c.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)(blockIdx.x - tab.start[which]) * kBlocks + wave * 2;
  const int64_t at = first * kBlock, left = t.n - at;
  if (left <= 0) return;
  const bool vec = ((tab.vec >> which) & 1) && left >= 2 * kBlock;
  const int i = lane * 8, half = lane >> 5;
  const bool there = left > half * kBlock;  // this half's block has elements
  T* p = (T*)t.param + at;
  uint8_t *pm = (uint8_t*)t.exp_avg + at, *pv = (uint8_t*)t.exp_avg_sq + at;
  float *sm = t.scale_avg + first, *sv = t.scale_sq + first;
  float w[8], m[8], v[8], r[8], am, av;
  uint32_t qm[2], qv[2];
  if (vec) {
    Raw8<T> raw;
    raw.load(t, first, lane);
    raw.unpack(w, v, qm, qv, am, av);
  } else {
    load_codes8(pm, i, left, qm);
    load_codes8(pv, i, left, qv);
    load8((const T*)t.grad + at, i, left, v);
    load8(p, i, left, w);
    am = there ? sm[half] : 0.f;
    av = there ? sv[half] : 0.f;
  }
  const double um = unit2(am), uv = unit4(av);
  uint32_t top_m = 0, top_v = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double gd = (double)v[e] * clip;
    const uint32_t byte = 8 * (e & 3);
    m[e] = blend(h.b1, (double)value2((int)(int8_t)(qm[e >> 2] >> byte), um), h.c1, gd);
    v[e] = blend(h.b2, (double)value4((qv[e >> 2] >> byte) & 0xffu, uv), h.c2, gd * gd);
    // magnitudes order as their bits, NaN above all (past the end everything is 0; v has no sign but a NaN's)
    top_m = max(top_m, __float_as_uint(m[e]) & 0x7fffffffu);
    top_v = max(top_v, __float_as_uint(v[e]));
    r[e] = root<SCALED>(v[e]);
    w[e] = stepped<SCALED>(w[e], m[e], r[e], c, h.eps);
  }
  store8(p, i, left, vec, w);
  const float Am = __uint_as_float(half_max_u32(top_m)), Av = __uint_as_float(half_max_u32(top_v));
  encode<8>(m, v, r, Am, Av, qm, qv);
  store_codes8(pm, i, left, vec, qm);
  store_codes8(pv, i, left, vec, qv);
  if ((lane & 31) == 0 && there) {
    sm[half] = Am;
    sv[half] = Av;
  }
}

// ------------------------------------------------------------------ moments in f32 again
struct MomentTable {
  zmoe_moment t[kTensors];
  int32_t start[kTensors + 1];
  uint64_t vec;
  int count;
};

__global__ __launch_bounds__(kThreads) void moments_kernel(const MomentTable tab) {
  const int which = owner_of(tab.start, tab.count, blockIdx.x);
  const zmoe_moment& t = tab.t[which];
  const bool wide = (tab.vec >> which) & 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)(blockIdx.x - tab.start[which]) * kMomentBlocks + wave * (kMomentBlocks / 4);
#pragma unroll
  for (int u = 0; u < kMomentBlocks / 4; ++u) {
    const int64_t b = first + u, i = b * kBlock + lane * 4;
    if (b * kBlock >= t.n) break;
    const bool vec = wide && (b + 1) * kBlock <= t.n;
    const uint32_t q = load_codes((const uint8_t*)t.codes, i, t.n, vec);
    const double unit = t.second ? unit4(t.scale[b]) : unit2(t.scale[b]);
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = t.second ? value4((q >> (8 * e)) & 0xffu, unit) : value2((int)(int8_t)(q >> (8 * e)), unit);
    store4(t.out, i, t.n, vec, v);
  }
}

// ------------------------------------------------------------------ the grads' norm
struct NormTable {
  const void* g[kNormTensors];
  int64_t n[kNormTensors];
  int32_t start[kNormTensors + 1];
  int count;
};

// parts[chunk] = sum g^2 over a chunk, in double: a clip that moved by one f32 rounding would turn codes.
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_squares_kernel(const NormTable tab, double* __restrict__ parts) {
  __shared__ double red[kThreads / 64];
  constexpr int VC = 16 / sizeof(T);
  const int which = owner_of(tab.start, tab.count, blockIdx.x);
  const T* g = (const T*)tab.g[which];
  const int64_t a = (int64_t)(blockIdx.x - tab.start[which]) * kNormChunk;
  const int64_t b = a + kNormChunk < tab.n[which] ? a + kNormChunk : tab.n[which];
  double sum = 0.0;
  int64_t i = a;
  if ((reinterpret_cast<uintptr_t>(g) & 15u) == 0) {  // (a is a whole number of chunks)
    i = a + (b - a) / VC * VC;
#pragma unroll 4
    for (int64_t j = a + threadIdx.x * VC; j < i; j += kThreads * VC) {
      float v[VC];
      unpack_chunk(*reinterpret_cast<const uint4*>(g + j), v, T{});
#pragma unroll
      for (int u = 0; u < VC; ++u) sum += (double)v[u] * (double)v[u];
    }
  }
  for (i += threadIdx.x; i < b; i += kThreads) sum += (double)to_f32(g[i]) * (double)to_f32(g[i]);
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__global__ __launch_bounds__(1024) void clip_factor_kernel(const double* __restrict__ parts, int64_t count,
                                                           float max_norm, float* __restrict__ out) {
  __shared__ double red[16];
  double sum = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < count; i += 1024) sum += parts[i];
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) sum += red[w];
    const float norm = (float)sqrt(sum), f = max_norm / (norm + 1e-6f);
    out[0] = norm;
    out[1] = f > 1.f ? 1.f : f;  // a norm that is NaN stays so
  }
}

bool on(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace
}  // namespace zmoe

using namespace zmoe;

extern "C" size_t zmoe_sum_squares_workspace_bytes(int64_t n) {
  return n > 0 && n < (1LL << 40) ? (size_t)cdiv(n, kNormChunk) * 8 : 0;
}

extern "C" int zmoe_sum_squares(const void* const* tensors, const int64_t* n, int count, int dtype, double* parts,
                                void* stream) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "sum_squares: dtype %d", dtype);
  ZMOE_REQUIRE(count >= 0, ZMOE_ERR_SHAPE, "sum_squares: %d tensors", count);
  ZMOE_REQUIRE(count == 0 || (tensors && n && parts), ZMOE_ERR_NULL, "sum_squares: null pointer");
  for (int i = 0; i < count; ++i) {
    ZMOE_REQUIRE(n[i] >= 0 && n[i] < (1LL << 40), ZMOE_ERR_SHAPE, "sum_squares: tensor %d of %lld elements", i,
                 (long long)n[i]);
    ZMOE_REQUIRE(n[i] == 0 || tensors[i], ZMOE_ERR_NULL, "sum_squares: null pointer");
  }
  NormTable tab;
  tab.count = 0;
  tab.start[0] = 0;
  int64_t done = 0;
  auto launch = [&]() {
    if (tab.count == 0) return (int)ZMOE_OK;
    const unsigned blocks = (unsigned)tab.start[tab.count];
    if (dtype == ZMOE_DTYPE_BF16)
      hipLaunchKernelGGL(sum_squares_kernel<uint16_t>, dim3(blocks), dim3(kThreads), 0, as_stream(stream), tab,
                         parts + done);
    else
      hipLaunchKernelGGL(sum_squares_kernel<float>, dim3(blocks), dim3(kThreads), 0, as_stream(stream), tab,
                         parts + done);
    done += blocks;
    tab.count = 0;
    return check_launch("sum_squares");
  };
  // a launch's chunks: fewer threads than a launch holds (one tensor of more is dealt out over several launches)
  constexpr int64_t kMost = kMaxLaunchThreads / kThreads / 2;
  const int size = dtype_size(dtype);
  for (int i = 0; i < count; ++i) {
    for (int64_t first = 0, all = cdiv(n[i], kNormChunk); first < all;) {
      const int64_t room = kMost - tab.start[tab.count];
      if (room <= 0 || tab.count == kNormTensors) {
        if (const int rc = launch()) return rc;
        continue;
      }
      const int64_t take = all - first < room ? all - first : room, at = first * kNormChunk;
      tab.g[tab.count] = (const char*)tensors[i] + at * size;
      tab.n[tab.count] = n[i] - at < take * kNormChunk ? n[i] - at : take * kNormChunk;
      tab.start[tab.count + 1] = tab.start[tab.count] + (int32_t)take;
      ++tab.count;
      first += take;
    }
  }
  return launch();
}

extern "C" int zmoe_clip_factor(const double* parts, int64_t count, float max_norm, float* norm_and_factor,
                                void* stream) {
  ZMOE_REQUIRE(count >= 0, ZMOE_ERR_SHAPE, "clip_factor: %lld parts", (long long)count);
  ZMOE_REQUIRE(norm_and_factor && (count == 0 || parts), ZMOE_ERR_NULL, "clip_factor: null pointer");
  hipLaunchKernelGGL(clip_factor_kernel, dim3(1), dim3(1024), 0, as_stream(stream), parts, count, max_norm,
                     norm_and_factor);
  return check_launch("clip_factor");
}

extern "C" int zmoe_adamw(const zmoe_adamw_tensor* tensors, int count, int dtype, int state_bits, const float* lr_ptr,
                          double lr, double beta1, double beta2, double eps, double weight_decay, const float* clip,
                          float* workspace, size_t workspace_bytes, void* stream) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "adamw: dtype %d", dtype);
  ZMOE_REQUIRE(state_bits == 32 || state_bits == 8, ZMOE_ERR_DTYPE, "adamw: moments in 32 or 8 bits (%d)", state_bits);
  ZMOE_REQUIRE(count >= 0, ZMOE_ERR_SHAPE, "adamw: %d tensors", count);
  ZMOE_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, ZMOE_ERR_SHAPE, "adamw: betas %g, %g", beta1,
               beta2);
  ZMOE_REQUIRE(eps >= 0.0, ZMOE_ERR_SHAPE, "adamw: eps %g", eps);
  if (count == 0) return ZMOE_OK;
  ZMOE_REQUIRE(tensors && workspace, ZMOE_ERR_NULL, "adamw: null pointer");
  ZMOE_REQUIRE(aligned16(workspace), ZMOE_ERR_ALIGN, "adamw: the workspace must be 16-byte aligned");
  ZMOE_REQUIRE(workspace_bytes >= (size_t)count * 16, ZMOE_ERR_WORKSPACE, "adamw: workspace %zu < %zu bytes",
               workspace_bytes, (size_t)count * 16);
  const int size = dtype_size(dtype);
  for (int i = 0; i < count; ++i) {
    const zmoe_adamw_tensor& t = tensors[i];
    ZMOE_REQUIRE(t.n >= 0 && t.n < (1LL << 40), ZMOE_ERR_SHAPE, "adamw: tensor %d of %lld elements", i, (long long)t.n);
    ZMOE_REQUIRE(t.step, ZMOE_ERR_NULL, "adamw: null pointer");
    if (t.n == 0) continue;
    ZMOE_REQUIRE(t.param && t.grad && t.exp_avg && t.exp_avg_sq && (state_bits == 32 || (t.scale_avg && t.scale_sq)),
                 ZMOE_ERR_NULL, "adamw: null pointer");
    ZMOE_REQUIRE(on(t.param, size) && on(t.grad, size) &&
                     (state_bits == 8 ? on(t.scale_avg, 4) && on(t.scale_sq, 4) : on(t.exp_avg, 4) && on(t.exp_avg_sq, 4)),
                 ZMOE_ERR_ALIGN, "adamw: tensor %d is not on whole elements", i);
  }
  float4* coef = reinterpret_cast<float4*>(workspace);
  for (int i = 0; i < count; i += kNormTensors) {
    StepTable s;
    s.count = count - i < kNormTensors ? count - i : kNormTensors;
    for (int j = 0; j < s.count; ++j) s.step[j] = tensors[i + j].step;
    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(kNormTensors / 64), dim3(64), 0, as_stream(stream), s, lr_ptr, lr, beta1,
                       beta2, weight_decay, clip, coef + i);
    if (const int rc = check_launch("adamw")) return rc;
  }
  const Hyper h{beta1,        beta2,        1.0 - beta1,          1.0 - beta2,         (float)beta1,
                (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), (float)eps};
  Table tab;
  tab.count = 0;
  tab.start[0] = 0;
  tab.vec = 0;
  int first_of_launch = 0;
  auto launch = [&](int next) {
    const bool any = tab.count > 0 && tab.start[tab.count] > 0;
    if (any) {
      const dim3 grid((unsigned)tab.start[tab.count]), block(kThreads);
      auto go = [&](auto type, auto scaled) {
        using T = decltype(type);
        constexpr bool S = decltype(scaled)::value;
        if (state_bits == 8)
          hipLaunchKernelGGL((adamw8_kernel<T, S>), grid, block, 0, as_stream(stream), tab, h, coef + first_of_launch);
        else
          hipLaunchKernelGGL((adamw_kernel<T, S>), grid, block, 0, as_stream(stream), tab, h, coef + first_of_launch);
      };
      auto typed = [&](auto type) {
        if (eps * std::sqrt(1.0 - beta2) >= 0x1p-38) go(type, std::false_type{});  // (root)
        else go(type, std::true_type{});
      };
      if (dtype == ZMOE_DTYPE_BF16) typed(uint16_t{});
      else typed(float{});
    }
    tab.count = 0;
    tab.vec = 0;
    first_of_launch = next;
    return any ? check_launch("adamw") : (int)ZMOE_OK;
  };
  constexpr int64_t kMost = kMaxLaunchThreads / kThreads / 2;
  const unsigned wide = state_bits == 8 ? 16 : 4 * size, codes = state_bits == 8 ? 8 : 16;
  for (int i = 0; i < count; ++i) {
    const zmoe_adamw_tensor& t = tensors[i];
    const int64_t all = cdiv(t.n, kChunk);
    for (int64_t first = 0; first < all || (all == 0 && first == 0);) {
      const int64_t room = kMost - tab.start[tab.count];
      if (room <= 0 || tab.count == kTensors) {
        if (const int rc = launch(i)) return rc;
        continue;
      }
      const int64_t take = all - first < room ? all - first : room, at = first * kChunk;
      zmoe_adamw_tensor& u = tab.t[tab.count];
      u = t;
      u.param = (char*)t.param + at * size;
      u.grad = (const char*)t.grad + at * size;
      u.exp_avg = (char*)t.exp_avg + at * (state_bits / 8);
      u.exp_avg_sq = (char*)t.exp_avg_sq + at * (state_bits / 8);
      if (state_bits == 8) {
        u.scale_avg = t.scale_avg + first * kBlocks;
        u.scale_sq = t.scale_sq + first * kBlocks;
      }
      u.n = t.n - at < take * kChunk ? t.n - at : take * kChunk;
      if (on(t.param, wide) && on(t.grad, wide) && on(t.exp_avg, codes) && on(t.exp_avg_sq, codes))
        tab.vec |= 1ull << tab.count;
      tab.start[tab.count + 1] = tab.start[tab.count] + (int32_t)take;
      ++tab.count;
      first += take;
      if (all == 0) break;  // no elements: its place in the table keeps coef's order
      if (first < all)      // the rest of this tensor opens the next launch, and has its coef there
        if (const int rc = launch(i)) return rc;
    }
  }
  return launch(count);
}

extern "C" int zmoe_adamw_moments(const zmoe_moment* moments, int count, void* stream) {
  ZMOE_REQUIRE(count >= 0, ZMOE_ERR_SHAPE, "adamw_moments: %d tensors", count);
  ZMOE_REQUIRE(count == 0 || moments, ZMOE_ERR_NULL, "adamw_moments: null pointer");
  for (int i = 0; i < count; ++i) {
    const zmoe_moment& t = moments[i];
    ZMOE_REQUIRE(t.n >= 0 && t.n < (1LL << 40), ZMOE_ERR_SHAPE, "adamw_moments: tensor %d of %lld elements", i,
                 (long long)t.n);
    ZMOE_REQUIRE(t.n == 0 || (t.codes && t.scale && t.out), ZMOE_ERR_NULL, "adamw_moments: null pointer");
    ZMOE_REQUIRE(on(t.scale, 4) && on(t.out, 4), ZMOE_ERR_ALIGN, "adamw_moments: tensor %d is not on whole elements", i);
  }
  MomentTable tab;
  tab.count = 0;
  tab.start[0] = 0;
  tab.vec = 0;
  auto launch = [&]() {
    if (tab.count == 0) return (int)ZMOE_OK;
    hipLaunchKernelGGL(moments_kernel, dim3((unsigned)tab.start[tab.count]), dim3(kThreads), 0, as_stream(stream), tab);
    tab.count = 0;
    tab.vec = 0;
    return check_launch("adamw_moments");
  };
  constexpr int64_t kMost = kMaxLaunchThreads / kThreads / 2;
  for (int i = 0; i < count; ++i) {
    const zmoe_moment& t = moments[i];
    for (int64_t first = 0, all = cdiv(t.n, kMomentChunk); first < all;) {
      const int64_t room = kMost - tab.start[tab.count];
      if (room <= 0 || tab.count == kTensors) {
        if (const int rc = launch()) return rc;
        continue;
      }
      const int64_t take = all - first < room ? all - first : room, at = first * kMomentChunk;
      zmoe_moment& u = tab.t[tab.count];
      u = t;
      u.codes = (const char*)t.codes + at;
      u.scale = t.scale + first * kMomentBlocks;
      u.out = t.out + at;
      u.n = t.n - at < take * kMomentChunk ? t.n - at : take * kMomentChunk;
      if (on(t.codes, 4) && on(t.out, 16)) tab.vec |= 1ull << tab.count;
      tab.start[tab.count + 1] = tab.start[tab.count] + (int32_t)take;
      ++tab.count;
      first += take;
    }
  }
  return launch();
}
