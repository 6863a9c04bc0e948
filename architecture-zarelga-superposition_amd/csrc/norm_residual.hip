// The step between two sublayers of a block: the norm after the first, its gate, the scaled residual
// and the norm in front of the second, in one pass over the rows, and its backward in another.
//   u  = y rho1 (1 + w1),   rho1 = rsqrt(mean(y^2) + eps)        (u = y without w1)
//   r' = alpha r + g u                                            (g: none, per channel, per row, or full)
//   x  = r' rho2 (1 + w2),  rho2 = rsqrt(mean(r'^2) + eps)        (no x without w2)
// in f32, r' and x rounded once each (x from the unrounded r'). Backward, from dr' and dx:
//   t  = dr' + rho2 (1 + w2) dx - r' rho2^3 / d sum_j dx_j (1 + w2_j) r'_j      (the whole grad of r')
//   dr = alpha t, dalpha = sum t r, dg = t u (summed over what g was broadcast over), du = g t
//   dy = rho1 (1 + w1) du - y rho1^3 / d sum_j du_j (1 + w1_j) y_j
//   dw1 = sum_rows du y rho1, dw2 = sum_rows dx r' rho2
// r' is formed again in the backward from r and y, which it has to read anyway, so nothing but the two
// rstds is kept and no rounding of a stored r' gets into the grads.
// Both passes are bound by HBM. A row belongs to the fewest waves that hold it at eight elements a
// thread (one wave up to d = 512, four at 2048, sixteen at 8192; above, more elements a thread): few
// registers, so several workgroups share a CU and one's loads fill the other's row sums and barriers.
// The backward walks rows with a fixed grid and loads its next row before it reduces the current one;
// the sums over rows stay in registers until the end, then go through per-block partials added in a
// fixed order (the same result on every run).
#include <type_traits>

#include "zmoe_internal.h"

namespace zmoe {
namespace {

constexpr int kVN = 8;        // elements of a thread's chunk
constexpr int kMaxWaves = 16; // waves of one row
constexpr int kMaxNQ = 4;
constexpr int kMaxPartials = 512;

enum Gate { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_ROW = 2, GATE_FULL = 3 };

// A parameter or gate tensor of either type (its type is uniform in a launch: one scalar branch).
struct Vec {
  const void* p;
  int bf16, vec;
};
struct Out {
  void* p;
  int bf16, vec;
};

template <typename T>
__device__ __forceinline__ void load_chunk(const T* __restrict__ row, int64_t c, int64_t d, bool vec, float (&v)[kVN]) {
  constexpr int VC = 16 / sizeof(T);
  if (vec && c + kVN <= d) {
#pragma unroll
    for (int q = 0; q < kVN / VC; ++q) unpack_chunk(*reinterpret_cast<const uint4*>(row + c + q * VC), &v[q * VC], T{});
  } else {
#pragma unroll
    for (int u = 0; u < kVN; ++u) v[u] = c + u < d ? to_f32(row[c + u]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ row, int64_t c, int64_t d, bool vec, const float (&v)[kVN]) {
  constexpr int VC = 16 / sizeof(T);
  if (vec && c + kVN <= d) {
#pragma unroll
    for (int q = 0; q < kVN / VC; ++q) *reinterpret_cast<uint4*>(row + c + q * VC) = pack_chunk(&v[q * VC], T{});
  } else {
#pragma unroll
    for (int u = 0; u < kVN; ++u)
      if (c + u < d) row[c + u] = from_f32<T>(v[u]);
  }
}
__device__ __forceinline__ void load_vec(const Vec& w, int64_t at, int64_t c, int64_t d, float (&v)[kVN]) {
  if (w.bf16) load_chunk(static_cast<const uint16_t*>(w.p) + at, c, d, w.vec != 0, v);
  else load_chunk(static_cast<const float*>(w.p) + at, c, d, w.vec != 0, v);
}
__device__ __forceinline__ float load_one(const Vec& w, int64_t i) {
  return w.bf16 ? to_f32(static_cast<const uint16_t*>(w.p)[i]) : static_cast<const float*>(w.p)[i];
}
__device__ __forceinline__ void store_one(const Out& o, int64_t i, float v) {
  if (o.bf16) static_cast<uint16_t*>(o.p)[i] = bf16_bits(v);
  else static_cast<float*>(o.p)[i] = v;
}

// Sums of v[0 .. N - 1] over the threads of a row, W waves, in every one of them. With W > 1 every
// thread of the block calls it; consecutive calls alternate `slot` (one barrier a call: a slot's
// values are read before the call after the next one writes it).
template <int W, int N, int WPB>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[WPB][2], int slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[slot][wave][i] = v[i];
    }
    __syncthreads();
    const int w0 = wave / W * W;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int q = 0; q < W; ++q) t += red[slot][w0 + q][i];
      v[i] = t;
    }
  }
}

struct NormArgs {
  const void *r, *y;
  int64_t ldr, ldy, n, d;
  int vec;  // r, y, outputs and grads take 16-byte accesses
  Vec w1, w2, gate;
  int gate_kind;
  int64_t ldg;
  const float* alpha_ptr;
  float alpha, eps;
  void *r_out, *x;
  float *rho1, *rho2;
  // backward
  const void *gr, *gx;
  void *dr, *dy;
  Out dgate;      // row or full gates
  float* partial; // [3][P][d] sums for w1, w2 and a channel gate, then [P] for alpha
};

template <int W>
struct Map {
  static constexpr int TPR = 64 * W;
  static constexpr int THREADS = TPR < 256 ? 256 : TPR;
  static constexpr int WPB = THREADS / 64, RPB = THREADS / TPR;
};

template <typename R, typename Y, int W, int NQ>
__global__ __launch_bounds__(Map<W>::THREADS) void norm_residual_kernel(NormArgs a) {
  using M = Map<W>;
  __shared__ float red[2][M::WPB][2];
  const int64_t i = (int64_t)blockIdx.x * M::RPB + threadIdx.x / M::TPR;
  const bool live = i < a.n;  // (every thread stays for the barriers)
  const int lt = threadIdx.x % M::TPR;
  const int64_t row = live ? i : 0;
  const float alpha = a.alpha_ptr ? *a.alpha_ptr : a.alpha;
  const float inv_d = 1.0f / (float)a.d;
  float y[NQ][kVN], h[NQ][kVN], g[NQ][kVN];
  float s[1] = {0.f};
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t c = (int64_t)(lt + q * M::TPR) * kVN, dd = live ? a.d : 0;
    load_chunk(static_cast<const Y*>(a.y) + row * a.ldy, c, dd, a.vec != 0, y[q]);
    load_chunk(static_cast<const R*>(a.r) + row * a.ldr, c, dd, a.vec != 0, h[q]);
    if (a.gate_kind == GATE_FULL) load_vec(a.gate, row * a.ldg, c, dd, g[q]);
    else if (a.gate_kind == GATE_CHANNEL) load_vec(a.gate, 0, c, a.d, g[q]);
#pragma unroll
    for (int u = 0; u < kVN; ++u) s[0] = fmaf(y[q][u], y[q][u], s[0]);
  }
  float rho1 = 1.f;
  if (a.w1.p) {
    row_sums<W, 1, M::WPB>(s, red, 0);
    rho1 = rsqrtf(s[0] * inv_d + a.eps);
    if (a.rho1 && live && lt == 0) a.rho1[i] = rho1;
  }
  const float g_row = a.gate_kind == GATE_ROW && live ? load_one(a.gate, i) : 1.f;
  s[0] = 0.f;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
    float w[kVN];
    if (a.w1.p) load_vec(a.w1, 0, c, a.d, w);
#pragma unroll
    for (int u = 0; u < kVN; ++u) {
      float v = y[q][u];
      if (a.w1.p) v = v * rho1 * (1.f + w[u]);
      if (a.gate_kind == GATE_ROW) v *= g_row;
      else if (a.gate_kind != GATE_NONE) v *= g[q][u];
      h[q][u] = fmaf(alpha, h[q][u], v);
      s[0] = fmaf(h[q][u], h[q][u], s[0]);
    }
    if (live) store_chunk(static_cast<R*>(a.r_out) + i * a.d, c, a.d, a.vec != 0, h[q]);
  }
  if (!a.x) return;  // uniform
  row_sums<W, 1, M::WPB>(s, red, 1);
  const float rho2 = rsqrtf(s[0] * inv_d + a.eps);
  if (!live) return;
  if (a.rho2 && lt == 0) a.rho2[i] = rho2;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
    float w[kVN];
    load_vec(a.w2, 0, c, a.d, w);
#pragma unroll
    for (int u = 0; u < kVN; ++u) h[q][u] = h[q][u] * rho2 * (1.f + w[u]);
    store_chunk(static_cast<Y*>(a.x) + i * a.d, c, a.d, a.vec != 0, h[q]);
  }
}

// One row's operands in the backward.
template <typename R, typename Y, int NQ>
struct Row {
  float r[NQ][kVN], y[NQ][kVN], gr[NQ][kVN], gx[NQ][kVN];
  float rho1, rho2;
  template <int TPR>
  __device__ __forceinline__ void load(const NormArgs& a, int64_t i, int lt) {
    const bool live = i < a.n;
    const int64_t row = live ? i : 0, dd = live ? a.d : 0;
    rho1 = live && a.w1.p ? a.rho1[row] : 1.f;
    rho2 = live && a.w2.p ? a.rho2[row] : 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int64_t c = (int64_t)(lt + q * TPR) * kVN;
      load_chunk(static_cast<const Y*>(a.y) + row * a.ldy, c, dd, a.vec != 0, y[q]);
      load_chunk(static_cast<const R*>(a.r) + row * a.ldr, c, dd, a.vec != 0, r[q]);
      load_chunk(static_cast<const R*>(a.gr) + row * a.d, c, a.gr ? dd : 0, a.vec != 0, gr[q]);
      load_chunk(static_cast<const Y*>(a.gx) + row * a.d, c, a.gx ? dd : 0, a.vec != 0, gx[q]);
    }
  }
};

template <typename R, typename Y, int W, int NQ>
__global__ __launch_bounds__(Map<W>::THREADS) void norm_residual_backward_kernel(NormArgs a) {
  using M = Map<W>;
  __shared__ float red[2][M::WPB][2];
  extern __shared__ float fold[];  // [RPB][d] (several rows a block)
  const int lt = threadIdx.x % M::TPR, sub = threadIdx.x / M::TPR;
  const float alpha = a.alpha_ptr ? *a.alpha_ptr : a.alpha;
  const float inv_d = 1.0f / (float)a.d;
  float w1[NQ][kVN], w2[NQ][kVN], gc[NQ][kVN], acc1[NQ][kVN], acc2[NQ][kVN], accg[NQ][kVN];
  float acc_alpha = 0.f;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
#pragma unroll
    for (int u = 0; u < kVN; ++u) w1[q][u] = w2[q][u] = acc1[q][u] = acc2[q][u] = accg[q][u] = 0.f;
    if (a.w1.p) load_vec(a.w1, 0, c, a.d, w1[q]);
    if (a.w2.p) load_vec(a.w2, 0, c, a.d, w2[q]);
    if (a.gate_kind == GATE_CHANNEL) load_vec(a.gate, 0, c, a.d, gc[q]);
  }
  const int64_t first = (int64_t)blockIdx.x * M::RPB, step = (int64_t)gridDim.x * M::RPB;
  Row<R, Y, NQ> cur, nxt;
  constexpr bool PREFETCH = NQ == 1;  // (more chunks a thread: no registers for the next row)
  cur.template load<M::TPR>(a, first + sub, lt);
  for (int64_t base = first; base < a.n; base += step) {  // uniform in the block
    const int64_t i = base + sub;
    const bool live = i < a.n;
    if constexpr (PREFETCH) nxt.template load<M::TPR>(a, i + step, lt);
    const float g_row = a.gate_kind == GATE_ROW && live ? load_one(a.gate, i) : 1.f;
    float g[NQ][kVN], uu[NQ][kVN], h[NQ][kVN];
    float s[1] = {0.f};
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
      if (a.gate_kind == GATE_FULL) load_vec(a.gate, (live ? i : 0) * a.ldg, c, live ? a.d : 0, g[q]);
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        if (a.gate_kind == GATE_CHANNEL) g[q][u] = gc[q][u];
        else if (a.gate_kind != GATE_FULL) g[q][u] = g_row;
        uu[q][u] = a.w1.p ? cur.y[q][u] * cur.rho1 * (1.f + w1[q][u]) : cur.y[q][u];
        h[q][u] = fmaf(alpha, cur.r[q][u], g[q][u] * uu[q][u]);
        s[0] = fmaf(cur.gx[q][u] * (1.f + w2[q][u]), h[q][u], s[0]);
        acc2[q][u] = fmaf(cur.gx[q][u] * cur.rho2, h[q][u], acc2[q][u]);
      }
    }
    float coef2 = 0.f;
    if (a.gx) {
      row_sums<W, 1, M::WPB>(s, red, 0);
      coef2 = cur.rho2 * cur.rho2 * cur.rho2 * s[0] * inv_d;
    }
    float s2[2] = {0.f, 0.f};  // du (1 + w1) y, t u
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
      float out[kVN];
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        const float t = cur.gr[q][u] + cur.rho2 * (1.f + w2[q][u]) * cur.gx[q][u] - h[q][u] * coef2;
        out[u] = alpha * t;
        acc_alpha = fmaf(t, cur.r[q][u], acc_alpha);
        const float du = g[q][u] * t, tu = t * uu[q][u];
        s2[0] = fmaf(du * (1.f + w1[q][u]), cur.y[q][u], s2[0]);
        s2[1] += tu;
        accg[q][u] += tu;
        acc1[q][u] = fmaf(du * cur.rho1, cur.y[q][u], acc1[q][u]);
        h[q][u] = du;  // (r' is not needed any more)
        uu[q][u] = tu;
      }
      if (live) store_chunk(static_cast<R*>(a.dr) + i * a.d, c, a.d, a.vec != 0, out);
      if (live && a.gate_kind == GATE_FULL && a.dgate.p) {
        if (a.dgate.bf16) store_chunk(static_cast<uint16_t*>(a.dgate.p) + i * a.d, c, a.d, a.dgate.vec != 0, uu[q]);
        else store_chunk(static_cast<float*>(a.dgate.p) + i * a.d, c, a.d, a.dgate.vec != 0, uu[q]);
      }
    }
    if (a.w1.p || a.gate_kind == GATE_ROW) row_sums<W, 2, M::WPB>(s2, red, 1);
    if (live && a.gate_kind == GATE_ROW && a.dgate.p && lt == 0) store_one(a.dgate, i, s2[1]);
    const float coef1 = cur.rho1 * cur.rho1 * cur.rho1 * s2[0] * inv_d;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int64_t c = (int64_t)(lt + q * M::TPR) * kVN;
      if (a.w1.p) {
#pragma unroll
        for (int u = 0; u < kVN; ++u) h[q][u] = cur.rho1 * (1.f + w1[q][u]) * h[q][u] - cur.y[q][u] * coef1;
      }
      if (live) store_chunk(static_cast<Y*>(a.dy) + i * a.d, c, a.d, a.vec != 0, h[q]);
    }
    if constexpr (PREFETCH) cur = nxt;
    else cur.template load<M::TPR>(a, i + step, lt);
    if constexpr (W > 1) {
      // a row with only one of the two sums reuses its slot in the next one
      if (!(a.gx && (a.w1.p || a.gate_kind == GATE_ROW))) __syncthreads();
    }
  }
  // this block's partials; several rows a block: their sums added in order through LDS
  const int64_t P = gridDim.x;
  auto write = [&](float (&acc)[NQ][kVN], int which) {
    float* dst = a.partial + ((int64_t)which * P + blockIdx.x) * a.d;
    if constexpr (M::RPB == 1) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int u = 0; u < kVN; ++u) {
          const int64_t c = (int64_t)(lt + q * M::TPR) * kVN + u;
          if (c < a.d) dst[c] = acc[q][u];
        }
    } else {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        const int64_t c = (int64_t)lt * kVN + u;
        if (c < a.d) fold[(int64_t)sub * a.d + c] = acc[0][u];
      }
      __syncthreads();
      for (int64_t c = threadIdx.x; c < a.d; c += M::THREADS) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < M::RPB; ++q) t += fold[(int64_t)q * a.d + c];
        dst[c] = t;
      }
    }
  };
  if (a.w1.p) write(acc1, 0);
  if (a.w2.p) write(acc2, 1);
  if (a.gate_kind == GATE_CHANNEL) write(accg, 2);
  if (a.alpha_ptr) {
    __syncthreads();
    const float t = wave_sum(acc_alpha);
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6][0] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
      float all = 0.f;
#pragma unroll
      for (int q = 0; q < M::WPB; ++q) all += red[0][q][0];
      a.partial[3 * P * a.d + blockIdx.x] = all;
    }
  }
}

// dw[c] = the sum of P partials in a fixed order, rounded once: 64 columns a block, wave v takes
// partials v, v + 16, ..., and the 16 sums are added in wave order. blockIdx.y: which of the three
// vectors; 3: alpha's P values, one block.
constexpr int kRedWaves = 16;
struct Reduce {
  const float* partial;
  int P;
  int64_t d;
  Out out[3];
  float* dalpha;
};
__global__ __launch_bounds__(64 * kRedWaves) void norm_residual_reduce_kernel(Reduce a) {
  __shared__ float red[kRedWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y;
  if (which == 3) {
    if (blockIdx.x != 0 || !a.dalpha) return;
    float t = 0.f;
    for (int p = threadIdx.x; p < a.P; p += 64 * kRedWaves) t += a.partial[3 * (int64_t)a.P * a.d + p];
    t = wave_sum(t);
    if (lane == 0) red[0][wave] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
      float all = 0.f;
#pragma unroll
      for (int q = 0; q < kRedWaves; ++q) all += red[0][q];
      *a.dalpha = all;
    }
    return;
  }
  const Out o = which == 0 ? a.out[0] : which == 1 ? a.out[1] : a.out[2];
  if (!o.p) return;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float t = 0.f;
  if (c < a.d) {
#pragma unroll 8
    for (int p = wave; p < a.P; p += kRedWaves) t += a.partial[((int64_t)which * a.P + p) * a.d + c];
  }
  red[wave][lane] = t;
  __syncthreads();
  if (wave != 0 || c >= a.d) return;
#pragma unroll
  for (int v = 1; v < kRedWaves; ++v) t += red[v][lane];
  store_one(o, c, t);
}

// Waves of a row and chunks of a thread for rows of d elements (0: too wide).
int row_waves(int64_t d) {
  int w = 1;
  while (w < kMaxWaves && (int64_t)w * 64 * kVN < d) w *= 2;
  return w;
}
int row_chunks(int64_t d) {
  int nq = 1;
  while (nq < kMaxNQ && (int64_t)kMaxWaves * 64 * kVN * nq < d) nq *= 2;
  return nq;
}
constexpr int64_t kMaxD = (int64_t)kMaxWaves * 64 * kVN * kMaxNQ;
int rows_per_block(int64_t d) {
  const int w = row_waves(d);
  return w < 4 ? 4 / w : 1;
}
int partials(int64_t n, int64_t d) {
  const int64_t want = cdiv(n > 0 ? n : 1, rows_per_block(d));
  return (int)(want < kMaxPartials ? want : kMaxPartials);
}

// f(waves, chunks) with compile-time constants.
template <typename F>
void with_map(int64_t d, F f) {
  using std::integral_constant;
  const integral_constant<int, 1> one{};
  switch (row_waves(d)) {
    case 1: return f(one, one);
    case 2: return f(integral_constant<int, 2>{}, one);
    case 4: return f(integral_constant<int, 4>{}, one);
    case 8: return f(integral_constant<int, 8>{}, one);
    default:
      if (row_chunks(d) == 1) return f(integral_constant<int, 16>{}, one);
      if (row_chunks(d) == 2) return f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
      return f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  }
}
template <typename F>
void with_types(int r_dtype, int y_dtype, F f) {
  const bool rb = r_dtype == ZMOE_DTYPE_BF16, yb = y_dtype == ZMOE_DTYPE_BF16;
  if (rb && yb) f(uint16_t{}, uint16_t{});
  else if (rb) f(uint16_t{}, float{});
  else if (yb) f(float{}, uint16_t{});
  else f(float{}, float{});
}

bool vec_ok(const void* p, int64_t ld, int dtype) { return aligned16(p) && ld % (16 / dtype_size(dtype)) == 0; }

int common_checks(const char* name, int64_t n, int64_t d, int r_dtype, int y_dtype, int p_dtype, int gate_kind,
                  int gate_dtype, int64_t ldr, int64_t ldy, int64_t ldg, const void* w1, const void* gate,
                  const void* w2) {
  ZMOE_REQUIRE(dtype_ok(r_dtype) && dtype_ok(y_dtype) && dtype_ok(p_dtype) && dtype_ok(gate_dtype), ZMOE_ERR_DTYPE,
               "%s: dtype", name);
  ZMOE_REQUIRE(n >= 0 && n < 0x7fffffffLL && d >= 1 && d <= kMaxD, ZMOE_ERR_SHAPE,
               "%s: n=%lld rows of d=%lld (at most %lld)", name, (long long)n, (long long)d, (long long)kMaxD);
  ZMOE_REQUIRE(gate_kind >= GATE_NONE && gate_kind <= GATE_FULL && (!gate == (gate_kind == GATE_NONE)), ZMOE_ERR_SHAPE,
               "%s: gate kind %d", name, gate_kind);
  ZMOE_REQUIRE(ldr >= d && ldy >= d && (gate_kind != GATE_FULL || ldg >= d), ZMOE_ERR_SHAPE, "%s: row strides", name);
  ZMOE_REQUIRE(w1 || w2, ZMOE_ERR_NULL, "%s: neither norm's weight given", name);
  return ZMOE_OK;
}

NormArgs fill(const void* r, int64_t ldr, int r_dtype, const void* y, int64_t ldy, int y_dtype, int64_t n, int64_t d,
              const void* w1, const void* w2, int p_dtype, const void* gate, int gate_kind, int64_t ldg,
              int gate_dtype, const float* alpha_ptr, float alpha) {
  NormArgs a{};
  a.r = r;
  a.y = y;
  a.ldr = ldr;
  a.ldy = ldy;
  a.n = n;
  a.d = d;
  const int pb = p_dtype == ZMOE_DTYPE_BF16, gb = gate_dtype == ZMOE_DTYPE_BF16;
  a.w1 = Vec{w1, pb, aligned16(w1)};
  a.w2 = Vec{w2, pb, aligned16(w2)};
  a.gate = Vec{gate, gb, gate_kind == GATE_FULL ? vec_ok(gate, ldg, gate_dtype) : aligned16(gate)};
  a.gate_kind = gate_kind;
  a.ldg = ldg;
  a.alpha_ptr = alpha_ptr;
  a.alpha = alpha;
  return a;
}

}  // namespace
}  // namespace zmoe

using namespace zmoe;

extern "C" int zmoe_norm_residual(const void* R, int64_t r_stride, int r_dtype, const void* Y, int64_t y_stride,
                                  int y_dtype, int64_t n, int64_t d, const void* w_post, const void* w_next,
                                  int w_dtype, const void* gate, int gate_kind, int64_t gate_stride, int gate_dtype,
                                  const float* scale_ptr, float scale, float eps, void* R_out, void* X, float* rstd_post,
                                  float* rstd_next, void* stream) {
  int rc = common_checks("norm_residual", n, d, r_dtype, y_dtype, w_dtype, gate_kind, gate_dtype, r_stride, y_stride,
                         gate_stride, w_post, gate, w_next);
  if (rc) return rc;
  if (n == 0) return ZMOE_OK;
  ZMOE_REQUIRE(R && Y && R_out && (!X == !w_next), ZMOE_ERR_NULL, "norm_residual: null pointer");
  NormArgs a = fill(R, r_stride, r_dtype, Y, y_stride, y_dtype, n, d, w_post, w_next, w_dtype, gate, gate_kind,
                    gate_stride, gate_dtype, scale_ptr, scale);
  a.eps = eps;
  a.vec = vec_ok(R, r_stride, r_dtype) && vec_ok(Y, y_stride, y_dtype) && vec_ok(R_out, d, r_dtype) &&
          vec_ok(X, d, y_dtype);
  a.r_out = R_out;
  a.x = X;
  a.rho1 = rstd_post;
  a.rho2 = rstd_next;
  hipStream_t s = as_stream(stream);
  with_types(r_dtype, y_dtype, [&](auto rt, auto yt) {
    with_map(d, [&](auto w, auto nq) {
      using M = Map<decltype(w)::value>;
      hipLaunchKernelGGL((norm_residual_kernel<decltype(rt), decltype(yt), decltype(w)::value, decltype(nq)::value>),
                         dim3((unsigned)cdiv(n, M::RPB)), dim3(M::THREADS), 0, s, a);
    });
  });
  return check_launch("norm_residual");
}

extern "C" size_t zmoe_norm_residual_backward_workspace_bytes(int64_t n, int64_t d) {
  if (n < 0 || d < 1 || d > kMaxD) return 0;
  return (size_t)partials(n, d) * (3 * (size_t)d + 1) * sizeof(float);
}

extern "C" int zmoe_norm_residual_backward(const void* dR_out, const void* dX, const void* R, int64_t r_stride,
                                           int r_dtype, const void* Y, int64_t y_stride, int y_dtype, int64_t n,
                                           int64_t d, const void* w_post, const void* w_next, int w_dtype,
                                           const void* gate, int gate_kind, int64_t gate_stride, int gate_dtype,
                                           const float* scale_ptr, float scale, const float* rstd_post,
                                           const float* rstd_next, void* dR, void* dY, void* dw_post, void* dw_next,
                                           void* dgate, float* dscale, void* workspace, size_t workspace_bytes,
                                           void* stream) {
  int rc = common_checks("norm_residual_backward", n, d, r_dtype, y_dtype, w_dtype, gate_kind, gate_dtype, r_stride,
                         y_stride, gate_stride, w_post, gate, w_next);
  if (rc) return rc;
  ZMOE_REQUIRE(n == 0 || (R && Y && dR && dY), ZMOE_ERR_NULL, "norm_residual_backward: null operand");
  ZMOE_REQUIRE(n == 0 || ((!w_post || rstd_post) && (!w_next || rstd_next)), ZMOE_ERR_NULL,
               "norm_residual_backward: a norm's rstd is missing");
  ZMOE_REQUIRE(!dX || w_next, ZMOE_ERR_NULL, "norm_residual_backward: dX without the next norm's weight");
  ZMOE_REQUIRE(!dscale || scale_ptr, ZMOE_ERR_NULL, "norm_residual_backward: the grad of a scale that is no tensor");
  const size_t need = zmoe_norm_residual_backward_workspace_bytes(n, d);
  ZMOE_REQUIRE(workspace && workspace_bytes >= need, ZMOE_ERR_WORKSPACE,
               "norm_residual_backward: workspace %zu < %zu bytes", workspace_bytes, need);
  ZMOE_REQUIRE(aligned16(workspace), ZMOE_ERR_ALIGN, "norm_residual_backward: workspace on 16 bytes");
  NormArgs a = fill(R, r_stride, r_dtype, Y, y_stride, y_dtype, n, d, w_post, w_next, w_dtype, gate, gate_kind,
                    gate_stride, gate_dtype, scale_ptr, scale);
  a.vec = vec_ok(R, r_stride, r_dtype) && vec_ok(Y, y_stride, y_dtype) && vec_ok(dR, d, r_dtype) &&
          vec_ok(dY, d, y_dtype) && vec_ok(dR_out, d, r_dtype) && vec_ok(dX, d, y_dtype);
  a.rho1 = const_cast<float*>(rstd_post);
  a.rho2 = const_cast<float*>(rstd_next);
  a.gr = dR_out;
  a.gx = dX;
  a.dr = dR;
  a.dy = dY;
  a.dgate = Out{gate_kind == GATE_ROW || gate_kind == GATE_FULL ? dgate : nullptr, gate_dtype == ZMOE_DTYPE_BF16,
                vec_ok(dgate, d, gate_dtype)};
  a.partial = static_cast<float*>(workspace);
  const int P = partials(n, d);
  hipStream_t s = as_stream(stream);
  with_types(r_dtype, y_dtype, [&](auto rt, auto yt) {
    with_map(d, [&](auto w, auto nq) {
      using M = Map<decltype(w)::value>;
      const size_t lds = M::RPB > 1 ? (size_t)M::RPB * (size_t)d * sizeof(float) : 0;  // at most 8 KB
      hipLaunchKernelGGL(
          (norm_residual_backward_kernel<decltype(rt), decltype(yt), decltype(w)::value, decltype(nq)::value>),
          dim3((unsigned)P), dim3(M::THREADS), lds, s, a);
    });
  });
  rc = check_launch("norm_residual_backward");
  if (rc) return rc;
  Reduce red{};
  red.partial = a.partial;
  red.P = P;
  red.d = d;
  const int pb = w_dtype == ZMOE_DTYPE_BF16;
  red.out[0] = Out{w_post ? dw_post : nullptr, pb, 0};
  red.out[1] = Out{w_next ? dw_next : nullptr, pb, 0};
  red.out[2] = Out{gate_kind == GATE_CHANNEL ? dgate : nullptr, gate_dtype == ZMOE_DTYPE_BF16, 0};
  red.dalpha = dscale;
  if (red.out[0].p || red.out[1].p || red.out[2].p || dscale) {
    hipLaunchKernelGGL(norm_residual_reduce_kernel, dim3((unsigned)cdiv(d, 64), 4), dim3(64 * kRedWaves), 0, s, red);
    rc = check_launch("norm_residual_backward sums");
  }
  return rc;
}
