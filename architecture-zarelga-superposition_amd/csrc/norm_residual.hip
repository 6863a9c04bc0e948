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
// thread (one wave up to d = 512, four at 2048, sixteen at 8192 in the forward; above, more elements a thread): few
// registers, so several workgroups share a CU and one's loads fill the other's row sums and barriers.
// The backward walks rows with a fixed grid; the sums over rows go through per-block partials added in
// a fixed order (the same result on every run).
#include <type_traits>

#include "zmoe_tiles.h"

namespace zmoe {
namespace {

constexpr int kVN = 8;        // elements of a thread's chunk
constexpr int kMaxWaves = 16; // waves of one row
constexpr int kMaxNQ = 4;

enum Gate { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_ROW = 2, GATE_FULL = 3 };

// A parameter, gate or gate grad of either type (uniform in a launch: one scalar branch).
struct Vec {
  const void* p;
  int bf16;
};
struct Out {
  void* p;
  int bf16;
};

// Chunk c .. c + 7 of a row of d elements (zeros past it). VEC: d is a multiple of 8 and every row starts on
// 16 bytes, so a chunk is whole or absent; else element by element.
template <bool VEC, typename T>
__device__ __forceinline__ void load_chunk(const T* __restrict__ row, int64_t c, int64_t d, float (&v)[kVN]) {
  constexpr int VC = 16 / sizeof(T);
  if constexpr (VEC) {
    if (c < d) {
#pragma unroll
      for (int q = 0; q < kVN / VC; ++q)
        unpack_chunk(*reinterpret_cast<const uint4*>(row + c + q * VC), &v[q * VC], T{});
    } else {
#pragma unroll
      for (int u = 0; u < kVN; ++u) v[u] = 0.f;
    }
  } else {
#pragma unroll
    for (int u = 0; u < kVN; ++u) v[u] = c + u < d ? to_f32(row[c + u]) : 0.f;
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store_chunk(T* __restrict__ row, int64_t c, int64_t d, const float (&v)[kVN]) {
  constexpr int VC = 16 / sizeof(T);
  if constexpr (VEC) {
    if (c < d) {
#pragma unroll
      for (int q = 0; q < kVN / VC; ++q) *reinterpret_cast<uint4*>(row + c + q * VC) = pack_chunk(&v[q * VC], T{});
    }
  } else {
#pragma unroll
    for (int u = 0; u < kVN; ++u)
      if (c + u < d) row[c + u] = from_f32<T>(v[u]);
  }
}
template <bool VEC>
__device__ __forceinline__ void load_vec(const Vec& w, int64_t at, int64_t c, int64_t d, float (&v)[kVN]) {
  if (w.bf16) load_chunk<VEC>(static_cast<const uint16_t*>(w.p) + at, c, d, v);
  else load_chunk<VEC>(static_cast<const float*>(w.p) + at, c, d, v);
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
__device__ __forceinline__ float lanes_sum(float v) {
  auto dpp = [](float x, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v += dpp(v, std::integral_constant<int, 0xB1>{});   // lane ^ 1
  v += dpp(v, std::integral_constant<int, 0x4E>{});   // lane ^ 2
  v += dpp(v, std::integral_constant<int, 0x141>{});  // 7 - lane within 8
  v += dpp(v, std::integral_constant<int, 0x140>{});  // 15 - lane within 16
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}
template <int W, int N, int WPB>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*red)[WPB][2], int slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lanes_sum(v[i]);
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

// TH: the fewest threads of a block.
template <int W, int TH = 256>
struct Map {
  static constexpr int TPR = 64 * W;
  static constexpr int THREADS = TPR < TH ? TH : TPR;
  static constexpr int WPB = THREADS / 64, RPB = THREADS / TPR;
};
template <int W>
using FwdMap = Map<W, 256>;

template <typename R, typename Y, int W, int NQ, bool VEC>
__global__ __launch_bounds__(FwdMap<W>::THREADS) void norm_residual_kernel(NormArgs a) {
  using M = FwdMap<W>;
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
    load_chunk<VEC>(static_cast<const Y*>(a.y) + row * a.ldy, c, dd, y[q]);
    load_chunk<VEC>(static_cast<const R*>(a.r) + row * a.ldr, c, dd, h[q]);
    if (a.gate_kind == GATE_FULL) load_vec<VEC>(a.gate, row * a.ldg, c, dd, g[q]);
    else if (a.gate_kind == GATE_CHANNEL) load_vec<VEC>(a.gate, 0, c, a.d, g[q]);
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
    if (a.w1.p) load_vec<VEC>(a.w1, 0, c, a.d, w);
#pragma unroll
    for (int u = 0; u < kVN; ++u) {
      float v = y[q][u];
      if (a.w1.p) v = v * rho1 * (1.f + w[u]);
      if (a.gate_kind == GATE_ROW) v *= g_row;
      else if (a.gate_kind != GATE_NONE) v *= g[q][u];
      h[q][u] = fmaf(alpha, h[q][u], v);
      s[0] = fmaf(h[q][u], h[q][u], s[0]);
    }
    if (live) store_chunk<VEC>(static_cast<R*>(a.r_out) + i * a.d, c, a.d, h[q]);
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
    load_vec<VEC>(a.w2, 0, c, a.d, w);
#pragma unroll
    for (int u = 0; u < kVN; ++u) h[q][u] = h[q][u] * rho2 * (1.f + w[u]);
    store_chunk<VEC>(static_cast<Y*>(a.x) + i * a.d, c, a.d, h[q]);
  }
}

// This block's part of the residual scale's grad.
template <int WPB>
__device__ __forceinline__ void block_alpha(const NormArgs& a, float v, float (*red)[WPB][2]) {
  if (!a.alpha_ptr) return;
  __syncthreads();
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6][0] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = 0.f;
#pragma unroll
    for (int q = 0; q < WPB; ++q) all += red[0][q][0];
    a.partial[3 * (int64_t)gridDim.x * a.d + blockIdx.x] = all;
  }
}

// A chunk as it was loaded: 16 (bf16) or 32 bytes.
template <typename T, bool VEC>
struct Chunk {
  uint4 w[kVN * sizeof(T) / 16];
  __device__ __forceinline__ void load(const T* __restrict__ row, int64_t c, int64_t d) {
    constexpr int VC = 16 / sizeof(T);
    if constexpr (VEC) {
#pragma unroll
      for (int q = 0; q < kVN / VC; ++q)
        w[q] = c < d ? *reinterpret_cast<const uint4*>(row + c + q * VC) : make_uint4(0, 0, 0, 0);
    } else {
      float v[kVN];
      load_chunk<false>(row, c, d, v);
#pragma unroll
      for (int q = 0; q < kVN / VC; ++q) w[q] = pack_chunk(&v[q * VC], T{});
    }
  }
  // What is formed from the chunk before this is formed again after it, not kept in registers.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (uint4& q : w) asm volatile("" : "+v"(q.x), "+v"(q.y), "+v"(q.z), "+v"(q.w));
  }
  __device__ __forceinline__ void get(float (&v)[kVN]) const {
    constexpr int VC = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < kVN / VC; ++q) unpack_chunk(w[q], &v[q * VC], T{});
  }
};

// A chunk of a full gate of either type, as it was loaded.
template <bool VEC>
struct GateChunk {
  Chunk<uint16_t, VEC> h;
  Chunk<float, VEC> f;
  int bf16;
  __device__ __forceinline__ void load(const Vec& g, int64_t at, int64_t c, int64_t d) {
    bf16 = g.bf16;
    if (bf16) h.load(static_cast<const uint16_t*>(g.p) + at, c, d);
    else f.load(static_cast<const float*>(g.p) + at, c, d);
  }
  __device__ __forceinline__ void forget() {
    if (bf16) h.forget();
    else f.forget();
  }
  __device__ __forceinline__ void get(float (&v)[kVN]) const {
    if (bf16) h.get(v);
    else f.get(v);
  }
};

// One row's operands in the backward: this thread's chunks of each.
template <typename R, typename Y, int NQ, bool VEC>
struct Row {
  Chunk<R, VEC> r[NQ], gr[NQ];
  Chunk<Y, VEC> y[NQ], gx[NQ];
  float rho1, rho2, g_row;
  template <typename Col>
  __device__ __forceinline__ void load(const NormArgs& a, int64_t i, Col col) {
    const bool live = i < a.n;
    const int64_t row = live ? i : 0, dd = live ? a.d : 0;
    rho1 = live && a.w1.p ? a.rho1[row] : 1.f;  // (no norm of y: u = y)
    rho2 = live && a.w2.p ? a.rho2[row] : 0.f;  // (no next norm: nothing through x)
    g_row = live && a.gate_kind == GATE_ROW ? load_one(a.gate, row) : 1.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int64_t c = col(q);
      y[q].load(static_cast<const Y*>(a.y) + row * a.ldy, c, dd);
      r[q].load(static_cast<const R*>(a.r) + row * a.ldr, c, dd);
      gr[q].load(static_cast<const R*>(a.gr) + row * a.d, c, a.gr ? dd : 0);
      gx[q].load(static_cast<const Y*>(a.gx) + row * a.d, c, a.gx ? dd : 0);
    }
  }
};

// 1 + w (1 without a weight) of a chunk.
template <bool VEC>
__device__ __forceinline__ void load_gain(const Vec& w, int64_t c, int64_t d, float (&v)[kVN]) {
  if (w.p) load_vec<VEC>(w, 0, c, d, v);
#pragma unroll
  for (int u = 0; u < kVN; ++u) v[u] = w.p ? 1.f + v[u] : 1.f;
}

template <bool VEC>
__device__ __forceinline__ void store_gate(const Out& o, int64_t at, int64_t c, int64_t d, const float (&v)[kVN]) {
  if (o.bf16) store_chunk<VEC>(static_cast<uint16_t*>(o.p) + at, c, d, v);
  else store_chunk<VEC>(static_cast<float*>(o.p) + at, c, d, v);
}

// Up to eight waves a row with one chunk a thread (d <= 4096): a row's operands, the parameters and the sums over rows
// stay in registers, some 160 a thread. Wider rows (to 8192) have two chunks a thread and the sums in LDS, each thread its
// own columns (24 bytes an element of the row, 12 to 18 from HBM at a tenth of LDS's rate). 4096 rows, f32 stream,
// bf16 y: 34 us at d = 2048 (4.4 TB/s), 66 at 4096, 126 at 7168 (4.2; sixteen waves of one chunk, with a quarter of the
// registers a thread and the parameters read again for every row, took 166).
template <typename R, typename Y, int W, int NQ, bool VEC, bool FULL>
__global__ __launch_bounds__(Map<W>::THREADS, 2) void norm_residual_backward_kernel(NormArgs a) {
  using M = Map<W>;
  __shared__ float red[2][M::WPB][2];
  constexpr bool LDS_SUMS = NQ > 1;
  extern __shared__ __align__(16) float fold[];  // [RPB][d] (several rows a block), or the sums [3][NQ][2][TPR]
  const int lt = threadIdx.x % M::TPR, sub = threadIdx.x / M::TPR;
  auto col = [&](int q) { return (int64_t)(lt + q * M::TPR) * kVN; };
  const float alpha = a.alpha_ptr ? *a.alpha_ptr : a.alpha;
  const float inv_d = 1.0f / (float)a.d;
  float w1[NQ][kVN], w2[NQ][kVN], gc[NQ][kVN], acc1[NQ][kVN], acc2[NQ][kVN], accg[NQ][kVN];
  float acc_alpha = 0.f;
  float4* sums = reinterpret_cast<float4*>(fold) + lt;
  // v added to this thread's part of sum k in LDS, and cleared
  auto add = [&](int k, int q, float (&v)[kVN]) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float4& at = sums[((k * NQ + q) * 2 + hh) * M::TPR];
      const float4 o = at;
      at = make_float4(o.x + v[4 * hh], o.y + v[4 * hh + 1], o.z + v[4 * hh + 2], o.w + v[4 * hh + 3]);
    }
#pragma unroll
    for (int u = 0; u < kVN; ++u) v[u] = 0.f;
  };
  if constexpr (LDS_SUMS) {
#pragma unroll
    for (int k = 0; k < 6 * NQ; ++k) sums[k * M::TPR] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
#pragma unroll
    for (int u = 0; u < kVN; ++u) {
      acc1[q][u] = acc2[q][u] = accg[q][u] = 0.f;
      gc[q][u] = 1.f;
    }
    load_gain<VEC>(a.w1, col(q), a.d, w1[q]);
    load_gain<VEC>(a.w2, col(q), a.d, w2[q]);
    if (a.gate_kind == GATE_CHANNEL) load_vec<VEC>(a.gate, 0, col(q), a.d, gc[q]);
  }
  const int64_t first = (int64_t)blockIdx.x * M::RPB, step = (int64_t)gridDim.x * M::RPB;
  Row<R, Y, NQ, VEC> cur;
  GateChunk<VEC> gate[NQ];  // FULL: this row's gate
  for (int64_t base = first; base < a.n; base += step) {  // uniform in the block
    const int64_t i = base + sub;
    const bool live = i < a.n;
    cur.load(a, i, col);
    if constexpr (FULL) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) gate[q].load(a.gate, (live ? i : 0) * a.ldg, col(q), live ? a.d : 0);
    }
    const float rho1 = cur.rho1, rho2 = cur.rho2, g_row = FULL ? 1.f : cur.g_row;
    // y rho1, u and r' of a chunk
    auto values = [&](int q, float (&yh)[kVN], float (&uu)[kVN], float (&r)[kVN], float (&h)[kVN]) {
      cur.y[q].get(yh);
      cur.r[q].get(r);
      if constexpr (FULL) gate[q].get(gc[q]);
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        yh[u] *= rho1;
        uu[u] = yh[u] * w1[q][u];
        h[u] = fmaf(gc[q][u] * g_row, uu[u], alpha * r[u]);
      }
    };
    float coef2 = 0.f;
    if (a.gx) {  // (else r' takes no part in its own grad: 0 times an r' that is not finite is left out too)
      float s[1] = {0.f};
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float yh[kVN], uu[kVN], r[kVN], h[kVN], gx[kVN];
        values(q, yh, uu, r, h);
        cur.gx[q].get(gx);
#pragma unroll
        for (int u = 0; u < kVN; ++u) {
          acc2[q][u] = fmaf(gx[u], rho2 * h[u], acc2[q][u]);
          s[0] = fmaf(gx[u] * w2[q][u], h[u], s[0]);
        }
        if (LDS_SUMS) add(1, q, acc2[q]);
        if constexpr (NQ > 1) __builtin_amdgcn_sched_barrier(0);  // (one chunk's values at a time)
      }
      row_sums<W, 1, M::WPB>(s, red, 0);
      coef2 = rho2 * rho2 * rho2 * s[0] * inv_d;
    }
    float s2[2] = {0.f, 0.f};  // du (1 + w1) y rho1, t u
    float h[NQ][kVN];          // du (1 + w1) after this
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      cur.y[q].forget();
      cur.r[q].forget();
      cur.gx[q].forget();
      if constexpr (FULL) gate[q].forget();
      float yh[kVN], uu[kVN], r[kVN], gx[kVN], t[kVN];
      values(q, yh, uu, r, h[q]);
      cur.gx[q].get(gx);
      cur.gr[q].get(t);
      if (a.gx) {
#pragma unroll
        for (int u = 0; u < kVN; ++u) t[u] = fmaf(-coef2, h[q][u], fmaf(rho2, gx[u] * w2[q][u], t[u]));
      }
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        acc_alpha = fmaf(t[u], r[u], acc_alpha);
        uu[u] *= t[u];
        s2[1] += uu[u];
        accg[q][u] += uu[u];
        h[q][u] = gc[q][u] * g_row * t[u];
        acc1[q][u] = fmaf(h[q][u], yh[u], acc1[q][u]);
        h[q][u] *= w1[q][u];
        s2[0] = fmaf(h[q][u], yh[u], s2[0]);
        t[u] *= alpha;
      }
      if (live) {
        store_chunk<VEC>(static_cast<R*>(a.dr) + i * a.d, col(q), a.d, t);
        if (FULL && a.dgate.p) store_gate<VEC>(a.dgate, i * a.d, col(q), a.d, uu);
      }
      if (LDS_SUMS && a.w1.p) add(0, q, acc1[q]);
      if (LDS_SUMS && a.gate_kind == GATE_CHANNEL) add(2, q, accg[q]);
      if constexpr (NQ > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (a.w1.p || a.gate_kind == GATE_ROW) row_sums<W, 2, M::WPB>(s2, red, 1);
    if (live && a.gate_kind == GATE_ROW && a.dgate.p && lt == 0) store_one(a.dgate, i, s2[1]);
    const float coef1 = a.w1.p ? rho1 * s2[0] * inv_d : 0.f;  // (rho1^3 y s = rho1 (y rho1) (s rho1))
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      cur.y[q].forget();
      if (live) {
        float yh[kVN];
        cur.y[q].get(yh);
        if (a.w1.p) {  // (else dy = du)
#pragma unroll
          for (int u = 0; u < kVN; ++u) h[q][u] = fmaf(-coef1, yh[u] * rho1, rho1 * h[q][u]);
        }
        store_chunk<VEC>(static_cast<Y*>(a.dy) + i * a.d, col(q), a.d, h[q]);
      }
      if constexpr (NQ > 1) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (W > 1) {
      // a row with only one of the two sums reuses its slot in the next one
      if (!(a.gx && (a.w1.p || a.gate_kind == GATE_ROW))) __syncthreads();
    }
  }
  // this block's partials; several rows a block: their sums added in order through LDS
  const int64_t P = gridDim.x;
  auto write = [&](float (&acc)[NQ][kVN], int which) {
    float* dst = a.partial + ((int64_t)which * P + blockIdx.x) * a.d;
    if constexpr (LDS_SUMS) {
#pragma unroll
      for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const float4 o = sums[((which * NQ + q) * 2 + hh) * M::TPR];
          acc[q][4 * hh] = o.x;
          acc[q][4 * hh + 1] = o.y;
          acc[q][4 * hh + 2] = o.z;
          acc[q][4 * hh + 3] = o.w;
        }
    }
    if constexpr (M::RPB == 1) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) store_chunk<VEC>(dst, col(q), a.d, acc[q]);
    } else {
      static_assert(NQ == 1 || M::RPB == 1, "rows that share a block have one chunk a thread");
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kVN; ++u)
        if (col(0) + u < a.d) fold[(int64_t)sub * a.d + col(0) + u] = acc[0][u];
      __syncthreads();
      for (int64_t k = threadIdx.x; k < a.d; k += M::THREADS) {
        float tt = 0.f;
#pragma unroll
        for (int q = 0; q < M::RPB; ++q) tt += fold[(int64_t)q * a.d + k];
        dst[k] = tt;
      }
    }
  };
  if (a.w1.p) write(acc1, 0);
  if (a.w2.p) write(acc2, 1);
  if (a.gate_kind == GATE_CHANNEL) write(accg, 2);
  block_alpha<M::WPB>(a, acc_alpha, red);
}

// Wider rows (d > 8192), sixteen waves a row and several chunks a thread: a chunk's operands are read again
// (from L2) for each of the three phases instead of being held, and the sums over rows are kept in this block's
// own partials in memory. Right for any width; about half the rate of the form above.
template <typename R, typename Y, bool VEC>
__global__ __launch_bounds__(Map<kMaxWaves>::THREADS, 4) void norm_residual_wide_backward_kernel(NormArgs a) {
  using M = Map<kMaxWaves>;
  __shared__ float red[2][M::WPB][2];
  const int64_t c0 = (int64_t)threadIdx.x * kVN, cstep = (int64_t)M::TPR * kVN, P = gridDim.x;
  const float alpha = a.alpha_ptr ? *a.alpha_ptr : a.alpha;
  const float inv_d = 1.0f / (float)a.d;
  float acc_alpha = 0.f;
  float* part[3] = {a.w1.p ? a.partial + (int64_t)blockIdx.x * a.d : nullptr,
                    a.w2.p ? a.partial + (P + blockIdx.x) * a.d : nullptr,
                    a.gate_kind == GATE_CHANNEL ? a.partial + (2 * P + blockIdx.x) * a.d : nullptr};
  bool fresh = true;  // this block's first row: its partials are written, not added to
  auto add = [&](float* p, int64_t c, const float (&v)[kVN]) {
    if (!p) return;
#pragma unroll
    for (int u = 0; u < kVN; ++u)
      if (c + u < a.d) p[c + u] = fresh ? v[u] : p[c + u] + v[u];
  };
  for (int64_t i = blockIdx.x; i < a.n; i += P) {  // (each block has a row, but for the one of a launch without rows)
    float rho1 = 1.f, rho2 = 0.f;
    // y rho1, u, r' and r of a chunk, and its gains
    float y[kVN], uu[kVN], h[kVN], r[kVN], gx[kVN], w1[kVN], w2[kVN], g[kVN], t[kVN];
    Row<R, Y, 1, VEC> row;
    auto chunk = [&](int64_t c) {
      row.load(a, i, [&](int) { return c; });
      rho1 = row.rho1;
      rho2 = row.rho2;
      row.y[0].get(y);
      row.r[0].get(r);
      row.gx[0].get(gx);
      row.gr[0].get(t);
      load_gain<VEC>(a.w1, c, a.d, w1);
      load_gain<VEC>(a.w2, c, a.d, w2);
      if (a.gate_kind == GATE_CHANNEL) load_vec<VEC>(a.gate, 0, c, a.d, g);
      else if (a.gate_kind == GATE_FULL) load_vec<VEC>(a.gate, i * a.ldg, c, a.d, g);
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        if (a.gate_kind == GATE_NONE || a.gate_kind == GATE_ROW) g[u] = row.g_row;
        y[u] *= rho1;
        uu[u] = y[u] * w1[u];
        h[u] = fmaf(g[u], uu[u], alpha * r[u]);
      }
    };
    float s[1] = {0.f};
    for (int64_t c = c0; c < a.d; c += cstep) {
      chunk(c);
      float v[kVN];
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        v[u] = a.gx ? gx[u] * (rho2 * h[u]) : 0.f;  // (no dx: 0, also where r' is not finite)
        s[0] = fmaf(gx[u] * w2[u], h[u], s[0]);
      }
      add(part[1], c, v);
    }
    row_sums<kMaxWaves, 1, M::WPB>(s, red, 0);
    const float coef2 = a.gx ? rho2 * rho2 * rho2 * s[0] * inv_d : 0.f;
    auto grad = [&](int64_t c) {  // t, the whole grad of r'
      chunk(c);
      if (!a.gx) return;
#pragma unroll
      for (int u = 0; u < kVN; ++u) t[u] = fmaf(-coef2, h[u], fmaf(rho2, gx[u] * w2[u], t[u]));
    };
    float s2[2] = {0.f, 0.f};
    for (int64_t c = c0; c < a.d; c += cstep) {
      grad(c);
      float v[kVN];
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        acc_alpha = fmaf(t[u], r[u], acc_alpha);
        uu[u] *= t[u];
        s2[1] += uu[u];
        h[u] = g[u] * t[u];
        v[u] = h[u] * y[u];
        s2[0] = fmaf(h[u] * w1[u], y[u], s2[0]);
        t[u] *= alpha;
      }
      add(part[0], c, v);
      add(part[2], c, uu);
      store_chunk<VEC>(static_cast<R*>(a.dr) + i * a.d, c, a.d, t);
      if (a.gate_kind == GATE_FULL && a.dgate.p) store_gate<VEC>(a.dgate, i * a.d, c, a.d, uu);
    }
    row_sums<kMaxWaves, 2, M::WPB>(s2, red, 1);
    if (a.gate_kind == GATE_ROW && a.dgate.p && threadIdx.x == 0) store_one(a.dgate, i, s2[1]);
    const float coef1 = a.w1.p ? rho1 * s2[0] * inv_d : 0.f;
    for (int64_t c = c0; c < a.d; c += cstep) {
      grad(c);
#pragma unroll
      for (int u = 0; u < kVN; ++u) {
        h[u] = rho1 * w1[u] * (g[u] * t[u]);
        if (a.w1.p) h[u] = fmaf(-coef1, y[u], h[u]);
      }
      store_chunk<VEC>(static_cast<Y*>(a.dy) + i * a.d, c, a.d, h);
    }
    fresh = false;
  }
  if (fresh) {  // no rows: sums of nothing
    const float zero[kVN] = {};
    for (int64_t c = c0; c < a.d; c += cstep) {
#pragma unroll
      for (int k = 0; k < 3; ++k) add(part[k], c, zero);
    }
  }
  block_alpha<M::WPB>(a, acc_alpha, red);
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
// Waves of a row in the backward, and its blocks. More of them hide more of each row's waits (up to three of four
// waves fit on a CU, one of eight), fewer leave less to the sum of their partials: 16384 rows of 2048 (f32 stream) 126 us
// with 768, 134 with 512, 220 with 256; 4096 rows 42, 40, 48; 1024 rows 28, 24, 22; 4096 rows of 4096 87 with 512, 76
// with 256.
int back_waves(int64_t d) {
  const int w = row_waves(d);
  return w == kMaxWaves && d <= (int64_t)kMaxWaves * 64 * kVN ? kMaxWaves / 2 : w;
}
int partials(int64_t n, int64_t d) {
  const int w = back_waves(d);
  const int64_t want = cdiv(n > 0 ? n : 1, w < 4 ? 4 / w : 1), most = w >= 8 || want <= 1024 ? 256 : want <= 4096 ? 512 : 768;
  return (int)(want < most ? want : most);
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
// What both passes read has 16-byte rows of whole chunks.
bool operands_vec(const NormArgs& a, int r_dtype, int y_dtype, int gate_dtype) {
  return a.d % kVN == 0 && vec_ok(a.r, a.ldr, r_dtype) && vec_ok(a.y, a.ldy, y_dtype) && aligned16(a.w1.p) &&
         aligned16(a.w2.p) &&
         (a.gate_kind == GATE_FULL ? vec_ok(a.gate.p, a.ldg, gate_dtype) : a.gate_kind == GATE_ROW || aligned16(a.gate.p));
}

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
  a.w1 = Vec{w1, pb};
  a.w2 = Vec{w2, pb};
  a.gate = Vec{gate, gb};
  a.gate_kind = gate_kind;
  a.ldg = ldg;
  a.alpha_ptr = alpha_ptr;
  a.alpha = alpha;
  return a;
}

// The forward's operands of n rows from row `first`; bytes of an element of R and Y.
NormArgs rows_from(NormArgs a, int64_t first, int64_t n, size_t r_size, size_t y_size) {
  auto on = [](const void* p, int64_t bytes) { return p ? static_cast<const char*>(p) + bytes : nullptr; };
  auto to = [](void* p, int64_t bytes) { return p ? static_cast<char*>(p) + bytes : nullptr; };
  a.n = n;
  a.r = on(a.r, first * a.ldr * (int64_t)r_size);
  a.y = on(a.y, first * a.ldy * (int64_t)y_size);
  if (a.gate_kind == GATE_ROW || a.gate_kind == GATE_FULL)
    a.gate.p = on(a.gate.p, first * (a.gate_kind == GATE_ROW ? 1 : a.ldg) * (a.gate.bf16 ? 2 : 4));
  a.r_out = to(a.r_out, first * a.d * (int64_t)r_size);
  a.x = to(a.x, first * a.d * (int64_t)y_size);
  if (a.rho1) a.rho1 += first;
  if (a.rho2) a.rho2 += first;
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
  const bool vec = operands_vec(a, r_dtype, y_dtype, gate_dtype) && aligned16(R_out) && aligned16(X);
  a.r_out = R_out;
  a.x = X;
  a.rho1 = rstd_post;
  a.rho2 = rstd_next;
  hipStream_t s = as_stream(stream);
  with_types(r_dtype, y_dtype, [&](auto rt, auto yt) {
    with_map(d, [&](auto w, auto nq) {
      using M = FwdMap<decltype(w)::value>;
      constexpr int W = decltype(w)::value, NQ = decltype(nq)::value;
      auto kern = vec ? norm_residual_kernel<decltype(rt), decltype(yt), W, NQ, true>
                      : norm_residual_kernel<decltype(rt), decltype(yt), W, NQ, false>;
      constexpr int64_t step = kMaxLaunchThreads / M::THREADS * M::RPB;  // rows of a launch
      for (int64_t first = 0; first < n; first += step) {
        const NormArgs part = rows_from(a, first, n - first < step ? n - first : step, sizeof(rt), sizeof(yt));
        hipLaunchKernelGGL(kern, dim3((unsigned)cdiv(part.n, M::RPB)), dim3(M::THREADS), 0, s, part);
      }
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
  const bool vec = operands_vec(a, r_dtype, y_dtype, gate_dtype) && aligned16(dR) && aligned16(dY) &&
                   aligned16(dR_out) && aligned16(dX) && (gate_kind != GATE_FULL || aligned16(dgate));
  a.rho1 = const_cast<float*>(rstd_post);
  a.rho2 = const_cast<float*>(rstd_next);
  a.gr = dR_out;
  a.gx = dX;
  a.dr = dR;
  a.dy = dY;
  a.dgate = Out{gate_kind == GATE_ROW || gate_kind == GATE_FULL ? dgate : nullptr, gate_dtype == ZMOE_DTYPE_BF16};
  a.partial = static_cast<float*>(workspace);
  const int P = partials(n, d);
  bool prepared = true;
  hipStream_t s = as_stream(stream);
  with_types(r_dtype, y_dtype, [&](auto rt, auto yt) {
    if (d > (int64_t)kMaxWaves * 64 * kVN) {
      auto kern = vec ? norm_residual_wide_backward_kernel<decltype(rt), decltype(yt), true>
                      : norm_residual_wide_backward_kernel<decltype(rt), decltype(yt), false>;
      hipLaunchKernelGGL(kern, dim3((unsigned)P), dim3(Map<kMaxWaves>::THREADS), 0, s, a);
      return;
    }
    with_map(d, [&](auto w, auto nq) {
      if constexpr (decltype(nq)::value == 1) {
        // sixteen waves of one chunk become eight of two
        constexpr int NQ = decltype(w)::value == kMaxWaves ? 2 : 1, W = decltype(w)::value / NQ;
        using M = Map<W>;
        using RT = decltype(rt);
        using YT = decltype(yt);
        auto kern = gate_kind == GATE_FULL ? (vec ? norm_residual_backward_kernel<RT, YT, W, NQ, true, true>
                                                  : norm_residual_backward_kernel<RT, YT, W, NQ, false, true>)
                                           : (vec ? norm_residual_backward_kernel<RT, YT, W, NQ, true, false>
                                                  : norm_residual_backward_kernel<RT, YT, W, NQ, false, false>);
        const size_t lds = NQ > 1 ? (size_t)M::TPR * 6 * NQ * sizeof(float4)  // 96 KB
                                  : (M::RPB > 1 ? (size_t)M::RPB * (size_t)d * sizeof(float) : 0);  // <= 8 KB
        if (NQ > 1 && prepare(kern, (int)lds) != ZMOE_OK) {
          prepared = false;
          return;
        }
        hipLaunchKernelGGL(kern, dim3((unsigned)P), dim3(M::THREADS), lds, s, a);
      }
    });
  });
  if (!prepared) return ZMOE_ERR_HIP;
  rc = check_launch("norm_residual_backward");
  if (rc) return rc;
  Reduce red{};
  red.partial = a.partial;
  red.P = P;
  red.d = d;
  const int pb = w_dtype == ZMOE_DTYPE_BF16;
  red.out[0] = Out{w_post ? dw_post : nullptr, pb};
  red.out[1] = Out{w_next ? dw_next : nullptr, pb};
  red.out[2] = Out{gate_kind == GATE_CHANNEL ? dgate : nullptr, gate_dtype == ZMOE_DTYPE_BF16};
  red.dalpha = dscale;
  if (red.out[0].p || red.out[1].p || red.out[2].p || dscale) {
    hipLaunchKernelGGL(norm_residual_reduce_kernel, dim3((unsigned)cdiv(d, 64), 4), dim3(64 * kRedWaves), 0, s, red);
    rc = check_launch("norm_residual_backward sums");
  }
  return rc;
}
