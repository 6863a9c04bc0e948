// Products in 8-bit floating point (OCP e4m3) with a power-of-two scale for each block of 128, dense
// and grouped by expert, the quantisers in front of them and the SwiGLU between two of them.
//
// A block of values v (1 x 128 along an activation row, 128 x 128 of a weight; the last one of a row or
// column is shorter) is held as q s with a = max |v| over its finite values,
//   s = 2^c, c the least whole number >= -127 with a <= 448 s,   q = e4m3(v / s), nearest even,
// 448 being e4m3's largest value; inf and NaN become e4m3's NaN. s is stored as the E8M0 byte c + 127.
// v / s is exact in f32 (short of f32's own underflow, where e4m3 has 0 anyway), so a block has one
// quantised form. gfx950's scaled MFMA (v_mfma_scale_f32_16x16x128_f8f6f4) takes E8M0 bytes as an
// operand: both scales of a product are applied inside the matrix unit, at no cost in vector
// instructions, and sums run on through the whole depth in its f32 accumulators. (An arbitrary f32
// scale would cost a vector FMA for every output and 128 of depth.)
#include <type_traits>
#include <utility>

#include "zmoe_tiles.h"

namespace zmoe {
namespace {

constexpr int kBlk = 128;  // values of one scale along the depth, and bytes of an LDS row
constexpr uint32_t kNaN8 = 0x7f;

typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef int v8i32_t __attribute__((ext_vector_type(8)));

__host__ __device__ inline int64_t blocks_of(int64_t n) { return (n + kBlk - 1) / kBlk; }
// Bytes of one row of scales: a whole number of dwords.
__host__ __device__ inline int64_t scale_pitch(int64_t K) { return (blocks_of(K) + 3) / 4 * 4; }

// E8M0 byte of the least power of two s >= 2^-127 with a <= 448 s (448 = 1.75 * 2^8), a finite, >= 0.
__device__ __forceinline__ int scale_code(float a) {
  const int bits = __float_as_int(a);
  const int c = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return c > 0 ? c : 0;
}
// Byte of the power of two that puts a into [2^14, 2^15) (the least is 2^-126).
__device__ __forceinline__ int half_code(float a) {
  const int c = (__float_as_int(a) >> 23) - 14;
  return c > 1 ? c : 1;
}
// 2^-c of that byte (code <= 247: the exponent field stays normal).
__device__ __forceinline__ float scale_inverse(int code) { return __int_as_float((254 - code) << 23); }

constexpr uint32_t kInfBits = 0x7f800000u;  // magnitudes from here on: inf, NaN
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }
__device__ __forceinline__ float finite_abs(float v) { return finite(v) ? fabsf(v) : 0.f; }

// Four values, already divided by their scale, to e4m3 bytes. Non-finite ones become NaN (the
// conversion itself would depend on the wave's overflow mode).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  return (uint32_t)w;
}
__device__ __forceinline__ uint32_t quantize4(const float (&v)[4], float inv) {
  uint32_t w = pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (!finite(v[u])) w = (w & ~(0xffu << (8 * u))) | (kNaN8 << (8 * u));
  return w;
}

// Largest of v over 16 consecutive lanes, in every one of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
  v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));  // 7 - lane within 8
  return max(v, dpp(v, std::integral_constant<int, 0x140>{}));  // 15 - lane within 16
}

// How rows can be loaded: in 16-byte chunks, in 4-byte pairs (16-bit elements), one by one.
enum Width { W_ONE = 0, W_PAIR = 1, W_CHUNK = 2 };
int row_width(const void* p, int64_t stride, int size) {
  if (aligned16(p) && stride % (16 / size) == 0) return W_CHUNK;
  return size == 2 && (reinterpret_cast<uintptr_t>(p) & 3u) == 0 && stride % 2 == 0 ? W_PAIR : W_ONE;
}

// Eight elements from column c of a row, zeros past K.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t c, int64_t K, int width, float (&v)[8]) {
  constexpr int VN = 16 / sizeof(T);
  if (width == W_CHUNK && c + 8 <= K) {
#pragma unroll
    for (int q = 0; q < 8 / VN; ++q) unpack_chunk(*reinterpret_cast<const uint4*>(row + c + q * VN), &v[q * VN], T{});
  } else if (sizeof(T) == 2 && width != W_ONE) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t at = c + 2 * q;
      w[q] = at + 1 < K ? *reinterpret_cast<const uint32_t*>(row + at)
                        : (at < K ? (uint32_t)row[at] : 0u);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = __uint_as_float(w[q] << 16);
      v[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c + u < K ? to_f32(row[c + u]) : 0.f;
  }
}

// ------------------------------------------------------------------ activations
// Sixteen lanes hold one block of 128 of a row, eight values each: one load of 16 (bf16) or 32 bytes,
// the largest magnitude by four lane exchanges, 8 bytes written by each lane. Bound by HBM (2 or 4
// bytes read, 1 written): 8192 x 7168 bf16 in 33 us (5.3 TB/s); two or four blocks a thread are 6-20% slower.
// Optionally row i is X[rows[i] / row_div] times row_scale[rows[i]] (the grouped, routing-weighted rows of an
// output gradient, never written anywhere in 16 bits).
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ X, int64_t ldx, int64_t x_rows,
                                                            const int64_t* __restrict__ rows, int row_div,
                                                            const float* __restrict__ row_scale, uint32_t total,
                                                            int64_t K, int nb, int width, uint8_t* __restrict__ Q,
                                                            uint8_t* __restrict__ S, int64_t pitch) {
  const uint32_t g = blockIdx.x * 16 + threadIdx.x / 16;  // (row, block)
  if (g >= total) return;  // whole groups of 16 lanes
  const uint32_t i = g / (uint32_t)nb, b = g - i * (uint32_t)nb;
  const int lane = threadIdx.x & 15;
  int64_t src = i;
  float sc = 1.f;
  if (rows != nullptr) {
    const int64_t slot = rows[i];
    src = slot < 0 ? -1 : slot / row_div;
    if (src >= x_rows) src = -1;
    if (src < 0) sc = 0.f;  // an index out of range: a row of zeros
    else if (row_scale != nullptr) sc = row_scale[slot];
  } else if (row_scale != nullptr) {
    sc = row_scale[i];
  }
  const int64_t c = (int64_t)b * kBlk + lane * 8;
  float v[8];
  load8(X + (src < 0 ? 0 : src) * ldx, c, src < 0 ? 0 : K, width, v);
  if (row_scale != nullptr) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] *= sc;
  }
  uint32_t a = 0;  // largest magnitude, as bits: inf and NaN show
#pragma unroll
  for (int u = 0; u < 8; ++u) a = max(a, __float_as_uint(v[u]) & 0x7fffffffu);
  const bool odd = __builtin_amdgcn_ballot_w64(a >= kInfBits) != 0;
  if (odd) {
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) m = fmaxf(m, finite_abs(v[u]));
    a = __float_as_uint(m);
  }
  const int code = scale_code(__uint_as_float(max16(a)));
  const float inv = scale_inverse(code);
  const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
  uint2 w;
  if (odd) w = make_uint2(quantize4(lo, inv), quantize4(hi, inv));
  else w = make_uint2(pack_e4m3(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv),
                      pack_e4m3(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv));
  *reinterpret_cast<uint2*>(Q + (int64_t)g * kBlk + lane * 8) = w;
  if (lane == 0) S[(int64_t)i * pitch + b] = (uint8_t)code;
}

// ------------------------------------------------------------------ weights
// One workgroup per 128 x 128 block: eight rows of eight columns a thread, the block's largest magnitude through LDS.
// With Qt the block is also written transposed (8 x 8 bytes in registers, the rest through LDS): W^T's blocks are W's,
// so one scale serves both, and the input gradient's product reads rows of W^T with the depth contiguous. Bound by HBM:
// 64 x 1536 x 2048 bf16 with both forms in 160 us (5.0 TB/s), f32 in 229 (5.3), 16 x 1030 x 510 in 16.
template <typename T, bool TRANS>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const T* __restrict__ W, int64_t se, int64_t sn,
                                                              int64_t N, int64_t K, int width, uint8_t* __restrict__ Q,
                                                              uint8_t* __restrict__ S, uint8_t* __restrict__ Qt,
                                                              uint8_t* __restrict__ St) {
  __shared__ uint32_t red[4];
  constexpr int TP = kBlk + 16;  // pitch of the transposed block, rows still 16-byte aligned
  __shared__ __align__(16) uint8_t tile[TRANS ? kBlk * TP : 16];
  const int64_t kb = blockIdx.x, nb = blockIdx.y, e = blockIdx.z;
  const int t = threadIdx.x, row0 = (t >> 4) * 8, col = (t & 15) * 8;
  float v[8][8];
  uint32_t a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t n = nb * kBlk + row0 + j;
    load8(W + e * se + (n < N ? n : 0) * sn, kb * kBlk + col, n < N ? K : 0, width, v[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int u = 0; u < 8; ++u) a = max(a, __float_as_uint(v[j][u]) & 0x7fffffffu);
  const bool odd = __builtin_amdgcn_ballot_w64(a >= kInfBits) != 0;  // this wave holds values that are not finite
  if (odd) {
    float f = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int u = 0; u < 8; ++u) f = fmaxf(f, finite_abs(v[j][u]));
    a = __float_as_uint(f);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = max(a, (uint32_t)__shfl_xor((int)a, o, 64));
  if ((t & 63) == 0) red[t >> 6] = a;
  __syncthreads();
  const int code = scale_code(__uint_as_float(max(max(red[0], red[1]), max(red[2], red[3]))));
  const float inv = scale_inverse(code);
  const int64_t nbs = blocks_of(N), kbs = blocks_of(K);
  if (t == 0) {
    S[(e * nbs + nb) * scale_pitch(K) + kb] = (uint8_t)code;
    if (TRANS) St[(e * kbs + kb) * scale_pitch(N) + nb] = (uint8_t)code;
  }
  uint2 w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t n = nb * kBlk + row0 + j;
    const float lo[4] = {v[j][0], v[j][1], v[j][2], v[j][3]}, hi[4] = {v[j][4], v[j][5], v[j][6], v[j][7]};
    if (odd) w[j] = make_uint2(quantize4(lo, inv), quantize4(hi, inv));
    else w[j] = make_uint2(pack_e4m3(lo[0] * inv, lo[1] * inv, lo[2] * inv, lo[3] * inv),
                           pack_e4m3(hi[0] * inv, hi[1] * inv, hi[2] * inv, hi[3] * inv));
    if (n < N) *reinterpret_cast<uint2*>(Q + ((e * N + n) * kbs + kb) * kBlk + col) = w[j];
  }
  if constexpr (TRANS) {
    // columns 4 c .. 4 c + 3 of rows 4 r .. 4 r + 3: byte pairs of two rows, then of two pairs
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t out[4][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = c ? w[4 * r + j].y : w[4 * r + j].x;
        const uint32_t p01 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);
        const uint32_t q01 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
        const uint32_t p23 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
        const uint32_t q23 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
        out[0][r] = __builtin_amdgcn_perm(p23, p01, 0x05040100u);
        out[1][r] = __builtin_amdgcn_perm(p23, p01, 0x07060302u);
        out[2][r] = __builtin_amdgcn_perm(q23, q01, 0x05040100u);
        out[3][r] = __builtin_amdgcn_perm(q23, q01, 0x07060302u);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        *reinterpret_cast<uint2*>(tile + (col + 4 * c + u) * TP + row0) = make_uint2(out[u][0], out[u][1]);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int kr = (t >> 3) + 32 * q, ch = (t & 7) * 16;
      const int64_t k = kb * kBlk + kr;
      if (k < K)
        *reinterpret_cast<uint4*>(Qt + ((e * K + k) * nbs + nb) * kBlk + ch) =
            *reinterpret_cast<const uint4*>(tile + kr * TP + ch);
    }
  }
}

// ------------------------------------------------------------------ products
// C[i, :] = A(i, :) B_e^T for the sorted rows i of expert e (or all rows of one weight), A rows and
// B rows of K / 128 blocks, one 128-byte line each. A stage is one block of the depth: BM + BN lines in
// LDS (the geometry of 64 bf16 elements), one 16 x 16 x 128 MFMA per 16 x 16 outputs. The weight rows
// are the MFMA's first operand, so a lane ends up with 4 consecutive output columns of one row.
// F8_HALF: rows that a sum over a token's k slots reads next, as f16 with a power-of-two scale for each 64 columns:
// 16 bits like bf16, but within 2^-11 of each value (bf16: 2^-8), so that the sum has its own rounding only.
enum Fp8Epi { F8_STORE_BF16 = 0, F8_STORE_F32 = 1, F8_GLU = 2, F8_HALF = 3, F8_GLU_EXACT = 4 };
constexpr bool is_glu(int epi) { return epi == F8_GLU || epi == F8_GLU_EXACT; }
// F8_GLU_EXACT: the SwiGLU's sums are rounded to e4m3 next, where an error of a few 2^-13 (a scaled MFMA's, of its largest
// terms) turns one value in some thousand to its neighbour, up to 2^-3 away: 0.0023 of the result's norm over many rows,
// where bf16's own rounding is 0.0017, and up to 0.018 of a single row of a narrow expert, whatever the launch's size. Terms
// taken to bf16 (exact) and added in f32 do not: 0.0017. They run at bf16's matrix rate, so that what they cost is the
// only reason against them, and that grows with the launch. One row in each of 32 experts of 2048 -> 2 x 768: 18.4 -> 20 us;
// 128 such experts of 4 rows 72 -> 80, of 21 rows 75 -> 84, of 32 rows 79 -> 94, of 128 rows 110 -> 149, of 2048 rows
// 799 -> 1529; 16384 rows skewed over 64 experts of 7168 -> 2 x 2048 619 -> 1009. Rows are independent: a larger
// batch called in parts of up to kExactValues has sums in f32 too.
constexpr int64_t kExactValues = 1 << 21;  // activations of a launch up to which it adds in f32
constexpr int kHalfCols = 64;  // columns of one scale: a wave's

struct Fp8Params {
  const uint8_t* a;
  const uint8_t* as;
  int64_t lda, a_pitch;    // bytes between rows of A and of its scales (few unquantised rows: K, elements between them)
  const int64_t* a_rows;   // A row of sorted row i = a_rows[i] / a_div (null: i)
  int a_div;
  int64_t a_bytes;         // bytes of A
  const uint8_t* b;
  const uint8_t* bs;
  int64_t b_estride, bs_estride, bs_pitch;
  uint32_t b_bytes;        // bytes of one expert's weights
  void* c;
  int64_t ldc;             // elements (GLU: bytes of a row of Aq)
  const int64_t* c_rows;   // output row of sorted row i = c_rows[i] (null: i)
  uint8_t* cs;             // GLU: the activations' scales; HALF: the rows'
  int64_t cs_pitch;
  int vec_c;               // rows of C take 16-byte stores
  const int64_t* offsets;  // inclusive expert ends [E] (null: one weight, ns_m rows)
  int nk, N, E, n_tiles, n_major;
  int half;                // GLU: pairs f
  int ns_m;                // rows of a dense launch (0: grouped)
  static constexpr int ns_sym = 0;
};

template <int BM, int BN, int NW>
struct Grid8 {
  static constexpr int GN = BN / 64, GM = NW / GN;
  static constexpr int WM = BM / GM, MF = WM / 16, NF = 4;
  static_assert(GM * GN == NW && WM % 16 == 0, "waves of 64 columns");
};

constexpr int kScaleStages = 64;  // stages whose scales are in LDS at once

template <int BM, int BN, int NW, int NS>
struct Lds8 {
  static constexpr int kStage = (BM + BN) * kBlk;
  static constexpr int kPitch = 64 * 2 + 16;  // staged output rows, bf16
  static constexpr int stages = NS * kStage;
  static constexpr int glu = BM * kBlk + 4 * BM * 4;  // quantised tile, row maxima of four waves
  static constexpr int kRows = Grid8<BM, BN, NW>::WM < 64 ? Grid8<BM, BN, NW>::WM : 64;  // rows a wave stages at once
  static constexpr int staging = NW * kRows * kPitch;
  static constexpr int ops = stages > glu ? (stages > staging ? stages : staging) : (glu > staging ? glu : staging);
  static constexpr int a_scales = ops;
  static constexpr int b_scales = a_scales + kScaleStages * BM;
  static constexpr int dst = b_scales + kScaleStages * 2;
  static constexpr int total = dst + BM * 4;
  static_assert(total <= 163840, "LDS of one CU");
};

template <int OFF>
__device__ __forceinline__ v4i32_t ds_read128(uint32_t addr) {
  v4i32_t v;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
  return v;
}
// MF scale bytes of this lane's rows (one per 16-row fragment), from `addr`
template <int MF>
struct AScale {
  uint32_t w[(MF + 3) / 4];
  __device__ __forceinline__ void read(uint32_t addr) {
    if constexpr (MF == 8) {
      v2i32_t v;
      asm volatile("ds_read_b64 %0, %1" : "=v"(v) : "v"(addr));
      w[0] = (uint32_t)v[0];
      w[1] = (uint32_t)v[1];
    } else if constexpr (MF == 4) {
      asm volatile("ds_read_b32 %0, %1" : "=v"(w[0]) : "v"(addr));
    } else if constexpr (MF == 2) {
      asm volatile("ds_read_u16 %0, %1" : "=v"(w[0]) : "v"(addr));
    } else {
      static_assert(MF == 1, "1, 2, 4 or 8 fragments");
      asm volatile("ds_read_u8 %0, %1" : "=v"(w[0]) : "v"(addr));
    }
  }
  __device__ __forceinline__ void tie() {
    asm volatile("" : "+v"(w[0]));
    if constexpr (MF == 8) asm volatile("" : "+v"(w[1]));
  }
};

// 32 bytes of a fragment row: lane (r = lane % 16, g = lane / 16) holds chunks g and g + 4 of row r.
// Both operands use this order, so which depths the instruction takes them for does not matter.
struct Frag8 {
  v4i32_t lo, hi;
  __device__ __forceinline__ v8i32_t value() const { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }
  __device__ __forceinline__ void tie() {
    asm_tie(lo);
    asm_tie(hi);
  }
};

// Eight e4m3 values times the power of two of E8M0 byte `code`, in bf16: exact (but for values below 2^-126).
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8v_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8v_t to_bf16x8(int lo, int hi, uint32_t code) {
  const float s = __uint_as_float(code << 23);
  const bf16x2v_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, s, false),
                  b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)lo, s, true),
                  c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, s, false),
                  d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)hi, s, true);
  return bf16x8v_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int... I, typename F>
__device__ __forceinline__ void unrolled(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F f) {
  unrolled(std::make_integer_sequence<int, N>{}, f);
}

// One stage of the wave's MF x 4 fragments with their sums at f32's precision: bf16 MFMAs of 32 depths. between(i) is
// called 16 times, between the MFMAs.
template <int MF, typename Between>
__device__ __forceinline__ void mma_exact(f32x4_t (&acc)[MF][4], const Frag8 (&fa)[MF], const Frag8 (&fb)[4],
                                          const AScale<MF>& sa, uint32_t sb, Between between) {
  unrolled<4>([&](auto h) {
    auto part = [&](const Frag8& f, uint32_t code) {
      const v4i32_t& v = h < 2 ? f.lo : f.hi;
      return to_bf16x8(v[2 * (h & 1)], v[2 * (h & 1) + 1], code);
    };
    bf16x8v_t a[MF];
    unrolled<MF>([&](auto m) { a[m] = part(fa[m], (sa.w[m / 4] >> (8 * (m & 3))) & 0xffu); });
    unrolled<4>([&](auto n) {
      const bf16x8v_t b = part(fb[n], (sb >> (8 * (n / 2))) & 0xffu);
      unrolled<MF>([&](auto m) { acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a[m], acc[m][n], 0, 0, 0); });
      between(std::integral_constant<int, h * 4 + n>{});
    });
  });
}

__device__ __forceinline__ int swizzle8(int row) { return (row & 7) ^ ((row >> 3) & 1); }

// Largest magnitude of v and m, as bits (two instructions for two values, and inf and NaN show).
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const f32x4_t& v) {
#pragma unroll
  for (int u = 0; u < 4; ++u) m = max(m, __float_as_uint(v[u]) & 0x7fffffffu);
  return m;
}
// Largest over the four lanes that hold one row (lane % 16).
__device__ __forceinline__ uint32_t max_rows4(uint32_t v) {
  auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max((uint32_t)a[0], (uint32_t)a[1]);
  a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max((uint32_t)a[0], (uint32_t)a[1]);
}

// decode_rows_tile, each wave for itself: no LDS and no barrier in the chain of loads that a tile begins with.
template <int BM, typename P>
__device__ __forceinline__ bool decode_rows_wave(const P& p, RowsTile& t) {
  if (p.ns_m > 0) {
    const int nm = (p.ns_m + BM - 1) / BM, logical = xcd_logical_tile(nm * p.n_tiles);
    if (logical < 0) return false;
    expert_tile_order(logical, p.n_tiles, nm, t.nt, t.mt);
    t.e = 0;
    t.row0 = (int64_t)t.mt * BM;
    t.rows = min(BM, p.ns_m - t.mt * BM);
    return true;
  }
  // a lane counts the row tiles of its ept consecutive experts (rows are below 2^31: the ends' low words)
  const int lane = (int)threadIdx.x & 63, ept = (p.E + 63) / 64, e0 = lane * ept;
  const int* ends = reinterpret_cast<const int*>(p.offsets);
  auto end_of = [&](int e) { return e >= 0 ? ends[2 * (e < p.E ? e : p.E - 1)] : 0; };
  int local = 0, singles = 0;
  for (int q0 = 0; q0 < ept; q0 += 4) {
    int end[5];
#pragma unroll
    for (int q = 0; q < 5; ++q) end[q] = end_of(e0 + q0 + q - 1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = q0 + q < ept && end[q + 1] > end[q] ? (end[q + 1] - end[q] + BM - 1) / BM : 0;
      local += n;
      singles += __builtin_popcountll(__builtin_amdgcn_ballot_w64(n == 1));
    }
  }
  int run = local;  // inclusive sums over the lanes
  auto add = [&](auto ctrl, auto rows) {
    run += __builtin_amdgcn_update_dpp(0, run, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
  add(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  add(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // the row before's last lane, the lower half's
  add(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  const int total = __builtin_amdgcn_readlane(run, 63) * p.n_tiles;
  const int logical = 4 * singles > p.E ? slab_logical_tile(total) : xcd_logical_tile(total);  // (as there)
  if (logical < 0) return false;
  const uint64_t later = __builtin_amdgcn_ballot_w64(run * p.n_tiles > logical);
  const int owner = __builtin_ctzll(later);  // (logical < total: some lane's sum is past it)
  int rest = logical - (__builtin_amdgcn_readlane(run, owner) - __builtin_amdgcn_readlane(local, owner)) * p.n_tiles;
  int e = owner * ept, beg = end_of(e - 1), end = end_of(e);
  auto tiles_of = [&] { return end > beg ? (end - beg + BM - 1) / BM : 0; };
  while (rest >= tiles_of() * p.n_tiles) {  // (ends at the lane's last expert at the latest)
    rest -= tiles_of() * p.n_tiles;
    beg = end;
    end = end_of(++e);
  }
  int inner, outer;
  const int nm = tiles_of();
  expert_tile_order(rest, p.n_major ? nm : p.n_tiles, p.n_major ? p.n_tiles : nm, inner, outer);
  t.e = e;
  t.nt = p.n_major ? outer : inner;
  t.mt = p.n_major ? inner : outer;
  t.row0 = (int64_t)beg + (int64_t)t.mt * BM;
  t.rows = min(BM, end - (int)t.row0);
  return true;
}

// The lines this wave loads of each stage's operand: 8 rows an instruction (1 KB of LDS), lane i the
// chunk (i % 8) ^ swizzle(row) of row i / 8.
template <int ROWS, int NW>
struct Lines8 {
  static constexpr int NQ = ROWS / (8 * NW);
  static_assert(NQ >= 1 && NQ * 8 * NW == ROWS, "whole instructions for every wave");
  uint32_t off[NQ];
  __device__ __forceinline__ static int row_of(int q) {
    return 8 * ((int)(threadIdx.x >> 6) * NQ + q) + (int)((threadIdx.x & 63) >> 3);
  }
  __device__ __forceinline__ void set(int q, uint32_t row_off) {
    const int c = (int)(threadIdx.x & 7) ^ swizzle8(row_of(q));
    off[q] = row_off == kOOB ? kOOB : row_off + 16u * (uint32_t)c;
  }
};

// The K loop of 256 x 256 tiles on eight waves, 128 x 64 outputs each: two buffers, every instruction placed. A stage
// is four steps of 32 of the wave's rows (two fragments against the four of B, 8 MFMAs, 256 cycles of the matrix
// unit). A step reads the next one's two A fragments while its MFMAs run; the fourth, after the one barrier of a stage
// (this wave's loads of the next stage are in, everyone is done reading this one), reads the next stage's first A
// fragments, its scales and, each as soon as its last MFMA is issued, its B fragments into the registers that
// become free. The loads of the stage after the next go out four in that step and four in the next one, one every
// other MFMA: issued together they hold a wave for ~70 cycles each, with its partner on the SIMD in the same phase.
// Waits count the LDS reads outstanding (they return in order). acc[m][n] as in the ring loop. GLU: B fragments 2 and 3
// take the second scale.
template <bool GLU, int BM, int STAGE, int LPS, typename Dma, typename Fill>
__device__ __forceinline__ void piped_loop(int nst, int c0, uint32_t lds0, uint32_t a_frag, uint32_t b_frag,
                                           uint32_t as_lane, uint32_t bs_lane, f32x4_t (&acc)[8][4], Dma dma, Fill fill) {
  static_assert(LPS == 8, "eight loads a stage");
  Frag8 fa[2][2], fb[4];
  AScale<8> sa, sa_next;
  uint32_t sb, sb_next;
  // LDS reads: half h of A fragment m, of B fragment n, the scales of stage st
  auto read_a = [&](uint32_t base, auto f, auto m, auto h) {
    const uint32_t at = (base + a_frag) ^ (h ? 64u : 0u);
    if constexpr (h == 0) fa[f][m & 1].lo = ds_read128<m * 2048>(at);
    else fa[f][m & 1].hi = ds_read128<m * 2048>(at);
  };
  auto read_b = [&](uint32_t base, auto n) {
    fb[n].lo = ds_read128<n * 2048>(base + b_frag);
    fb[n].hi = ds_read128<n * 2048>((base + b_frag) ^ 64u);
  };
  auto read_scales = [&](int st) {
    sa_next.read(as_lane + (uint32_t)(st * BM));
    if constexpr (GLU) asm volatile("ds_read_u16 %0, %1" : "=v"(sb_next) : "v"(bs_lane + 2u * (uint32_t)st));
    else asm volatile("ds_read_u8 %0, %1" : "=v"(sb_next) : "v"(bs_lane + 2u * (uint32_t)st));
  };
  auto mma = [&](auto m, auto n) {
    acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[n].value(), fa[(m >> 1) & 1][m & 1].value(), acc[m][n],
                                                                0, 0, GLU ? n / 2 : 0, (int)sb, m & 3, (int)sa.w[m / 4]);
  };
  auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
  using std::integral_constant;
  const integral_constant<int, 0> c0_{};
  const integral_constant<int, 1> c1_{};
#pragma unroll
  for (int q = 0; q < LPS / 2; ++q) dma(q, 1, c0 + 1, nst > 1);
  fill();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the scales are in LDS)
  __builtin_amdgcn_s_waitcnt(vm_wait(LPS / 2));
  asm volatile("s_barrier" ::: "memory");
  read_scales(0);
  read_a(lds0, c0_, c0_, c0_);
  read_a(lds0, c0_, c0_, c1_);
  read_a(lds0, c0_, c1_, c0_);
  read_a(lds0, c0_, c1_, c1_);
  unrolled<4>([&](auto n) { read_b(lds0, n); });
  // step 0 of stage st: B fragment n is in once at most the reads after its own are out; the second half of the
  // next stage's loads; at its end the A fragments of step 1 are in
  auto step0 = [&](int st) {
    const int buf = st & 1;
    const uint32_t base = lds0 + (uint32_t)(buf * STAGE);
    __builtin_amdgcn_s_setprio(1);
    unrolled<4>([&](auto n) {
      // allowed: the later B fragments' reads, and the A reads issued so far in this step
      asm_wait_lgkm<2 * (3 - n) + (n == 0 ? 0 : n == 1 ? 2 : 4)>();
      if constexpr (n == 0) {
        sa_next.tie();
        asm volatile("" : "+v"(sb_next));
        sa = sa_next;
        sb = sb_next;
        fa[0][0].tie();
        fa[0][1].tie();
      }
      fb[n].tie();
      fence();
      mma(c0_, n);
      dma(LPS / 2 + n, buf ^ 1, c0 + st + 1, st + 1 < nst);
      fence();
      mma(c1_, n);
      if constexpr (n < 2) {
        read_a(base, c1_, integral_constant<int, 2 + n>{}, c0_);
        read_a(base, c1_, integral_constant<int, 2 + n>{}, c1_);
      }
      fence();
    });
    __builtin_amdgcn_s_setprio(0);
    asm_wait_lgkm<0>();
    fa[1][0].tie();
    fa[1][1].tie();
  };
  // steps 1 and 2
  auto steps12 = [&](int st) {
    const uint32_t base = lds0 + (uint32_t)((st & 1) * STAGE);
    unrolled<2>([&](auto t) {
      constexpr int m0 = 2 + 2 * t;  // this step's fragments; the next step's: m0 + 2
      fence();
      unrolled<4>([&](auto n) {
        mma(integral_constant<int, m0>{}, n);
        if constexpr (n < 2) read_a(base, integral_constant<int, t>{}, integral_constant<int, m0 + 2 + n>{}, c0_);
        fence();
        mma(integral_constant<int, m0 + 1>{}, n);
        if constexpr (n < 2) read_a(base, integral_constant<int, t>{}, integral_constant<int, m0 + 2 + n>{}, c1_);
        fence();
      });
      asm_wait_lgkm<0>();
      fa[t][0].tie();
      fa[t][1].tie();
    });
  };
  // step 3 of a stage with one after it
  auto step3 = [&](int st) {
    const int buf = st & 1;
    const uint32_t next = lds0 + (uint32_t)((buf ^ 1) * STAGE);
    __builtin_amdgcn_s_waitcnt(vm_wait(0));
    asm volatile("s_barrier" ::: "memory");
    fence();
    __builtin_amdgcn_s_setprio(1);
    read_scales(st + 1);
    unrolled<4>([&](auto n) {
      mma(integral_constant<int, 6>{}, n);
      dma(n, buf, c0 + st + 2, st + 2 < nst);
      fence();
      mma(integral_constant<int, 7>{}, n);
      if constexpr (n == 0) {
        read_a(next, c0_, c0_, c0_);
        read_a(next, c0_, c0_, c1_);
        read_a(next, c0_, c1_, c0_);
        read_a(next, c0_, c1_, c1_);
      }
      read_b(next, n);
      fence();
    });
  };
  // The loop closes where no LDS read is out: a register copy that the compiler puts on its back edge must not
  // meet one whose data is still coming.
  step0(0);
  for (int st = 0; st + 1 < nst; ++st) {
    steps12(st);
    step3(st);
    step0(st + 1);
  }
  steps12(nst - 1);
  unrolled<4>([&](auto n) {
    mma(integral_constant<int, 6>{}, n);
    mma(integral_constant<int, 7>{}, n);
  });
  __builtin_amdgcn_s_setprio(0);
}

// The K loop of tiles that share a CU: 128 x 256 on four waves (128 x 64 outputs a wave, two workgroups a CU), 64 x 256
// and 128 x 128 (64 x 64, three). One LDS buffer: a stage's fragments go to registers at once, and the next stage's
// loads go out, one behind each MFMA, when every wave has its own (spread over the last MFMAs instead, with the A
// fragments read between the first ones: 1-2% slower). What a wave waits for is covered by the other workgroups.
template <int EPI, int BM, int LPS, int MF, typename Dma, typename Fill>
__device__ __forceinline__ void single_loop(int nst, int c0, uint32_t lds0, uint32_t a_frag, uint32_t b_frag,
                                            uint32_t as_lane, uint32_t bs_lane, f32x4_t (&acc)[MF][4], Dma dma, Fill fill) {
  constexpr bool GLU = is_glu(EPI);
  Frag8 fa[MF], fb[4];
  AScale<MF> sa;
  uint32_t sb;
  auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
  fill();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  for (int st = 0; st < nst; ++st) {
    __builtin_amdgcn_s_waitcnt(vm_wait(0));
    asm volatile("s_barrier" ::: "memory");
    fence();
    sa.read(as_lane + (uint32_t)(st * BM));
    if constexpr (GLU) asm volatile("ds_read_u16 %0, %1" : "=v"(sb) : "v"(bs_lane + 2u * (uint32_t)st));
    else asm volatile("ds_read_u8 %0, %1" : "=v"(sb) : "v"(bs_lane + 2u * (uint32_t)st));
    unrolled<4>([&](auto n) {
      fb[n].lo = ds_read128<n * 2048>(lds0 + b_frag);
      fb[n].hi = ds_read128<n * 2048>((lds0 + b_frag) ^ 64u);
    });
    unrolled<MF>([&](auto m) {
      fa[m].lo = ds_read128<m * 2048>(lds0 + a_frag);
      fa[m].hi = ds_read128<m * 2048>((lds0 + a_frag) ^ 64u);
    });
    asm_wait_lgkm<0>();
    sa.tie();
    asm volatile("" : "+v"(sb));
#pragma unroll
    for (int n = 0; n < 4; ++n) fb[n].tie();
#pragma unroll
    for (int m = 0; m < MF; ++m) fa[m].tie();
    asm volatile("s_barrier" ::: "memory");
    fence();
    if constexpr (EPI == F8_GLU_EXACT) {
      mma_exact<MF>(acc, fa, fb, sa, sb, [&](auto i) {
        if constexpr (i < LPS) dma(i, 0, c0 + st + 1, st + 1 < nst);
        fence();
      });
    } else unrolled<MF>([&](auto m) {
      unrolled<4>([&](auto n) {
        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[n].value(), fa[m].value(), acc[m][n], 0, 0,
                                                                    GLU ? n / 2 : 0, (int)sb, m & 3, (int)sa.w[m / 4]);
        if constexpr (m * 4 + n < LPS) dma(m * 4 + n, 0, c0 + st + 1, st + 1 < nst);
        fence();
      });
    });
  }
}

template <int BM, int BN, int NW, int NS, int EPI>
__global__ __launch_bounds__(NW * 64, NS > 1 ? 1 : (BM * BN <= 128 * 128 && EPI != F8_GLU_EXACT ? 3 : 2))
void fp8_rows_kernel(Fp8Params p) {
  extern __shared__ __align__(128) char smem[];
  using G = Grid8<BM, BN, NW>;
  using L = Lds8<BM, BN, NW, NS>;
  constexpr int MF = G::MF, NF = G::NF;
  constexpr int NT = NW * 64;
  constexpr bool PIPE = BM == 256 && BN == 256 && NW == 8 && NS == 2;
  static_assert(!is_glu(EPI) || BN == 256, "one block of 128 pairs a tile");

  RowsTile tile;
  if (!decode_rows_wave<BM>(p, tile)) return;  // uniform per workgroup
  const int e = tile.e, nt = tile.nt, rows = tile.rows;
  const int64_t row0 = tile.row0;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = (int)threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const int gm = wave / G::GN, gn = wave % G::GN;
  lds_char* lds = (lds_char*)(smem);
  const uint32_t lds0 = lds_addr(lds);

  // Before the loop a tile waits for memory three times in a row (the expert ends, its rows' numbers, their lines and
  // scales), so nothing else stands between: each lane reads the numbers of the rows that it loads itself, the
  // weight's lines go out before they are in, the scales before A's lines, and the scales' LDS writes come last.
  // Row numbers are below 2^31: the low words of the int64 entries.
  auto row_no = [&](const int64_t* list, int rl) {  // (rows past the tile's: its first)
    rl = rl < rows ? rl : 0;
    return list ? reinterpret_cast<const int*>(list)[2 * (row0 + rl)] : rl;
  };
  auto a_row = [&](int rl) {
    const int r = row_no(p.a_rows, rl);
    return p.a_rows ? (int)((uint32_t)r / (uint32_t)p.a_div) : r;
  };
  int* dst_table = reinterpret_cast<int*>(smem + L::dst);

  // A from its first row (gathered) or from this tile's (contiguous rows: no limit on their number)
  const char* a_base = reinterpret_cast<const char*>(p.a) + (p.a_rows ? 0 : row0 * p.lda);
  const int64_t a_left = p.a_bytes - (p.a_rows ? 0 : row0 * p.lda);
  const uint32_t a_bytes = a_left < 0x7fff0000 ? (uint32_t)a_left : 0x7fff0000u;
  const uint8_t* as_base = p.as + (p.a_rows ? 0 : row0 * p.a_pitch);
  const char* b_base = reinterpret_cast<const char*>(p.b) + (int64_t)e * p.b_estride;

  Lines8<BM, NW> la;
  Lines8<BN, NW> lb;
  constexpr int NQA = Lines8<BM, NW>::NQ, NQB = Lines8<BN, NW>::NQ, LPS = NQA + NQB;
#pragma unroll
  for (int q = 0; q < NQB; ++q) {
    const int rl = lb.row_of(q);
    int n;
    bool ok;
    if constexpr (is_glu(EPI)) {  // 64-row pair blocks [up 32 | gate 32] of the tile's 128 pairs
      const int jj = nt * kBlk + (rl >> 6) * 32 + (rl & 31);
      ok = jj < p.half;
      n = (rl & 32) ? p.half + jj : jj;
    } else {
      n = nt * BN + rl;
      ok = n < p.N;
    }
    lb.set(q, ok ? (uint32_t)((int64_t)n * ((int64_t)p.nk * kBlk)) : kOOB);
  }
  // load q of this wave's LPS of stage kt into buffer buf (zeros when !on)
  auto dma = [&](int q, int buf, int kt, bool on) {
    const int64_t k0 = (int64_t)kt * kBlk, room = (q < NQA ? (int64_t)a_bytes : (int64_t)p.b_bytes) - k0;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc((q < NQA ? a_base : b_base) + k0, on && room > 0 ? (uint32_t)room : 0u);
    lds_char* st = lds + buf * L::kStage;
    if (q < NQA) buf_to_lds(rs, st + (wave * NQA + q) * 1024, la.off[q < NQA ? q : 0]);
    else buf_to_lds(rs, st + BM * kBlk + (wave * NQB + q - NQA) * 1024, lb.off[q < NQA ? 0 : q - NQA]);
  };
  auto issue = [&](int buf, int kt, bool on) {
#pragma unroll
    for (int q = 0; q < LPS; ++q) dma(q, buf, kt, on);
  };
#pragma unroll
  for (int q = NQA; q < LPS; ++q) dma(q, 0, 0, true);
#pragma unroll
  for (int q = 0; q < NQA; ++q) {
    const int rl = la.row_of(q);
    la.set(q, rl < rows ? (uint32_t)((int64_t)a_row(rl) * p.lda) : kOOB);
  }
  constexpr int TPR = NT / BM, SW = kScaleStages / 4 / TPR;  // threads of a row, words of scales a thread takes at most
  const int scales_row = a_row((int)threadIdx.x % BM);

  f32x4_t acc[MF][NF];
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int n = 0; n < NF; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const uint32_t frag_off = (uint32_t)(r16 * kBlk + ((g4 ^ swizzle8(r16)) << 4));
  const uint32_t a_frag = (uint32_t)(gm * G::WM * kBlk) + frag_off;
  const uint32_t b_frag = (uint32_t)((BM + gn * 64) * kBlk) + frag_off;
  const uint32_t as_lane = lds0 + L::a_scales + (uint32_t)((gm * 16 + r16) * MF);
  const uint32_t bs_lane = lds0 + L::b_scales + (is_glu(EPI) ? 0u : (uint32_t)(gn / 2));
  for (int c0 = 0; c0 < p.nk; c0 += kScaleStages) {
    const int nst = p.nk - c0 < kScaleStages ? p.nk - c0 : kScaleStages;
    const int nd = (nst + 3) / 4;
    int tid = (int)threadIdx.x;
    asm volatile("" : "+v"(tid));  // (nothing that follows from it is worth a register throughout the loop)
    const int srow = tid % BM, spart = tid / BM;
    uint32_t sw[SW], bsw = 0;
    int dst_row = 0;
#pragma unroll
    for (int j = 0; j < SW; ++j)
      if (spart + TPR * j < nd)
        sw[j] = *reinterpret_cast<const uint32_t*>(as_base + (int64_t)scales_row * p.a_pitch + c0 + 4 * (spart + TPR * j));
    if (tid < 2 * nst) {
      const int64_t nb = is_glu(EPI) ? (tid & 1 ? blocks_of(p.half) : 0) + nt : (int64_t)nt * (BN / kBlk) + (tid & 1);
      const int64_t last = is_glu(EPI) ? 2 * blocks_of(p.half) - 1 : blocks_of(p.N) - 1;
      bsw = p.bs[(int64_t)e * p.bs_estride + (nb < last ? nb : last) * p.bs_pitch + c0 + (tid >> 1)];
    }
    if (c0 == 0) dst_row = row_no(p.c_rows, srow);
    if (c0 > 0) {
#pragma unroll
      for (int q = NQA; q < LPS; ++q) dma(q, 0, c0, true);
    }
#pragma unroll
    for (int q = 0; q < NQA; ++q) dma(q, 0, c0, true);
    // scales are kept as [stage][rows in fragment order]: row gm WM + 16 m + r at (gm 16 + r) MF + m
    // (asm: the compiler would have an LDS write wait for every load to LDS)
    auto fill = [&] {
      const uint32_t at = lds0 + L::a_scales + (uint32_t)(((srow / G::WM) * 16 + (srow & 15)) * MF + (srow % G::WM) / 16) +
                          (uint32_t)(spart * 4 * BM);
      unrolled<SW>([&](auto j) {
        if (spart + TPR * j < nd) {
          const uint32_t to = at, w = sw[j];
          unrolled<4>([&](auto u) {
            const uint32_t to_ = to, v = w >> (8 * u);
            asm volatile("ds_write_b8 %0, %1 offset:%2" ::"v"(to_), "v"(v), "n"((TPR * decltype(j)::value * 4 + u) * BM)
                         : "memory");
          });
        }
      });
      if (tid < 2 * nst)
        asm volatile("ds_write_b8 %0, %1" ::"v"(lds0 + L::b_scales + (uint32_t)tid), "v"(bsw) : "memory");
      if (c0 == 0 && tid < BM)
        asm volatile("ds_write_b32 %0, %1" ::"v"(lds0 + L::dst + 4u * (uint32_t)tid), "v"(dst_row) : "memory");
    };
    if constexpr (NS == 1) {
      single_loop<EPI, BM, LPS, MF>(nst, c0, lds0, a_frag, b_frag, as_lane, bs_lane, acc, dma, fill);
    } else if constexpr (PIPE) {
      piped_loop<is_glu(EPI), BM, L::kStage, LPS>(nst, c0, lds0, a_frag, b_frag, as_lane, bs_lane, acc, dma, fill);
    } else {
#pragma unroll
      for (int i = 1; i < NS - 1; ++i) issue(i, c0 + i, i < nst);
      fill();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");

      int cur = 0;
      for (int st = 0; st < nst; ++st) {
        __builtin_amdgcn_s_waitcnt(vm_wait((NS - 2) * LPS));  // this wave's loads of stage st are in
        asm volatile("s_barrier" ::: "memory");               // everyone's are, and the buffer before is read
        issue(cur == 0 ? NS - 1 : cur - 1, c0 + st + NS - 1, st + NS - 1 < nst);
        const uint32_t base = lds0 + (uint32_t)(cur * L::kStage);
        AScale<MF> sa;
        uint32_t sb;
        sa.read(as_lane + (uint32_t)(st * BM));
        if constexpr (is_glu(EPI)) asm volatile("ds_read_u16 %0, %1" : "=v"(sb) : "v"(bs_lane + 2u * (uint32_t)st));
        else asm volatile("ds_read_u8 %0, %1" : "=v"(sb) : "v"(bs_lane + 2u * (uint32_t)st));
        Frag8 fb[NF];
        unrolled<NF>([&](auto n) {
          fb[n].lo = ds_read128<n * 2048>(base + b_frag);
          fb[n].hi = ds_read128<n * 2048>((base + b_frag) ^ 64u);
        });
        constexpr int HF = MF < 4 ? MF : 4, STEPS = MF / HF;
        Frag8 fa[2][HF];
        auto read_a = [&](auto s) {
          unrolled<HF>([&](auto m) {
            fa[s & 1][m].lo = ds_read128<(s * HF + m) * 2048>(base + a_frag);
            fa[s & 1][m].hi = ds_read128<(s * HF + m) * 2048>((base + a_frag) ^ 64u);
          });
        };
        read_a(std::integral_constant<int, 0>{});
        unrolled<STEPS>([&](auto s) {
          if constexpr (s + 1 < STEPS) {
            read_a(std::integral_constant<int, s + 1>{});
            asm_wait_lgkm<2 * HF>();  // (in order: at most the next step's reads are out)
          } else {
            asm_wait_lgkm<0>();
          }
          if constexpr (s == 0) {
            sa.tie();
            asm volatile("" : "+v"(sb));
#pragma unroll
            for (int n = 0; n < NF; ++n) fb[n].tie();
          }
#pragma unroll
          for (int m = 0; m < HF; ++m) fa[s & 1][m].tie();
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (EPI == F8_GLU_EXACT) {
            mma_exact<MF>(acc, fa[0], fb, sa, sb, [](auto) {});
          } else unrolled<HF>([&](auto m) {
            unrolled<NF>([&](auto n) {
              constexpr int f = s * HF + m;
              acc[f][n] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                  fb[n].value(), fa[s & 1][m].value(), acc[f][n], 0, 0, is_glu(EPI) ? n / 2 : 0, (int)sb, f & 3,
                  (int)sa.w[f / 4]);
            });
          });
          __builtin_amdgcn_sched_barrier(0);
        });
        cur = cur == NS - 1 ? 0 : cur + 1;
      }
    }
    __builtin_amdgcn_s_waitcnt(vm_wait(0));  // loads past the end (zeros) are done before LDS is reused
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }

  // ---- outputs: acc[m][n][u] is row gm WM + 16 m + r, column gn 64 + 16 n + 4 g + u of the tile
  if constexpr (EPI == F8_STORE_F32) {
    float* C = static_cast<float*>(p.c);
    unrolled<MF>([&](auto m) {
      const int rl = gm * G::WM + 16 * m + r16;
      if (rl < rows) {
        float* out = C + (p.c_rows ? 0 : row0 * p.ldc) + (int64_t)dst_table[rl] * p.ldc;
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          const int col = nt * BN + gn * 64 + 16 * n + 4 * g4;
          if (p.vec_c && col + 4 <= p.N) {
            *reinterpret_cast<float4*>(out + col) = make_float4(acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (col + u < p.N) out[col + u] = acc[m][n][u];
          }
        }
      }
    });
  } else if constexpr (EPI == F8_STORE_BF16) {
    // up to 64 rows at a time through this wave's own staging area, then whole 128-byte lines
    char* st = smem + wave * L::kRows * L::kPitch;
    uint16_t* C = static_cast<uint16_t*>(p.c) + (p.c_rows ? 0 : row0 * p.ldc);
    constexpr int MS = L::kRows / 16;
    const int col0 = nt * BN + gn * 64;
    unrolled<MF / MS>([&](auto s) {
#pragma unroll
      for (int h = 0; h < MS; ++h)
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          const f32x4_t v = acc[s * MS + h][n];
          *reinterpret_cast<uint2*>(st + (16 * h + r16) * L::kPitch + (16 * n + 4 * g4) * 2) =
              make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int it = 0; it < 16 * MS / 8; ++it) {
        const int rr = it * 8 + (lane >> 3), ch = lane & 7;
        const int rl = gm * G::WM + 16 * MS * s + rr, col = col0 + ch * 8;
        const uint4 v = *reinterpret_cast<const uint4*>(st + rr * L::kPitch + ch * 16);
        if (rl < rows && col < p.N) {
          uint16_t* out = C + (int64_t)dst_table[rl] * p.ldc + col;
          if (p.vec_c && col + 8 <= p.N) {
            *reinterpret_cast<uint4*>(out) = v;
          } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (col + u < p.N) out[u] = (uint16_t)(w[u / 2] >> (16 * (u & 1)));
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    });
  } else if constexpr (EPI == F8_HALF) {
    // a row's 64 columns of this wave are in four lanes: the power of two that puts the largest into
    // [2^14, 2^15) (f16 ends at 65504; values down to 2^-28 of the largest keep all 11 bits), then as the bf16 store
    char* st = smem + wave * L::kRows * L::kPitch;
    uint16_t* C = static_cast<uint16_t*>(p.c);
    constexpr int MS = L::kRows / 16;
    const int cb = nt * (BN / kHalfCols) + gn;
    uint32_t top[MF], all = 0;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      top[m] = 0;
#pragma unroll
      for (int n = 0; n < NF; ++n) top[m] = max_bits(top[m], acc[m][n]);
      all = top[m] > all ? top[m] : all;
    }
    if (__builtin_amdgcn_ballot_w64(all >= kInfBits)) {  // rare: the largest finite values
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        float a = 0.f;
#pragma unroll
        for (int n = 0; n < NF; ++n)
#pragma unroll
          for (int u = 0; u < 4; ++u) a = fmaxf(a, finite_abs(acc[m][n][u]));
        top[m] = __float_as_uint(a);
      }
    }
    unrolled<MF / MS>([&](auto s) {
#pragma unroll
      for (int h = 0; h < MS; ++h) {
        constexpr int m0 = s * MS;
        const int code = half_code(__uint_as_float(max_rows4(top[m0 + h])));
        const float inv = scale_inverse(code);
        const int rl = gm * G::WM + 16 * (m0 + h) + r16;
#pragma unroll
        for (int n = 0; n < NF; ++n) {
          const f32x4_t v = acc[m0 + h][n];
          f16x4_t w;
#pragma unroll
          for (int u = 0; u < 4; ++u) w[u] = (_Float16)(v[u] * inv);
          *reinterpret_cast<uint2*>(st + (16 * h + r16) * L::kPitch + (16 * n + 4 * g4) * 2) = __builtin_bit_cast(uint2, w);
        }
        if (g4 == 0 && rl < rows && cb < p.cs_pitch)
          p.cs[((p.c_rows ? 0 : row0) + dst_table[rl]) * p.cs_pitch + cb] = (uint8_t)code;
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int it = 0; it < 16 * MS / 8; ++it) {
        const int rr = it * 8 + (lane >> 3), ch = lane & 7;
        const int rl = gm * G::WM + 16 * MS * s + rr;
        const uint4 v = *reinterpret_cast<const uint4*>(st + rr * L::kPitch + ch * 16);
        if (rl < rows && cb < p.cs_pitch)
          *reinterpret_cast<uint4*>(C + ((p.c_rows ? 0 : row0) + dst_table[rl]) * p.ldc + cb * kHalfCols + ch * 8) = v;
      }
      __builtin_amdgcn_wave_barrier();
    });
  } else {
    // a = silu(gate) up from the f32 sums; a row's 128 pairs of this tile are one block: its largest
    // magnitude over this wave's 32 pairs (four lanes a row), then over the four waves through LDS
    uint32_t* red = reinterpret_cast<uint32_t*>(smem + BM * kBlk);  // [BM][4]
    uint32_t top[MF], all = 0;
    unrolled<MF>([&](auto m) {
      top[m] = 0;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[m][n][u] *= silu_f(acc[m][2 + n][u]);
        top[m] = max_bits(top[m], acc[m][n]);
      }
      all = top[m] > all ? top[m] : all;
    });
    const bool odd = __builtin_amdgcn_ballot_w64(all >= kInfBits) != 0;  // this wave holds values that are not finite
    unrolled<MF>([&](auto m) {
      if (odd) {
        float a = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int u = 0; u < 4; ++u) a = fmaxf(a, finite_abs(acc[m][n][u]));
        top[m] = __float_as_uint(a);
      }
      const uint32_t a = max_rows4(top[m]);
      if (g4 == 0) red[(gm * G::WM + 16 * m + r16) * 4 + gn] = a;
    });
    __syncthreads();
    unrolled<MF>([&](auto m) {
      const int rl = gm * G::WM + 16 * m + r16;
      const uint4 r = *reinterpret_cast<const uint4*>(red + rl * 4);
      const uint32_t a = max(max(r.x, r.y), max(r.z, r.w));
      const int code = scale_code(__uint_as_float(a));
      const float inv = scale_inverse(code);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float v[4] = {acc[m][n][0], acc[m][n][1], acc[m][n][2], acc[m][n][3]};
        *reinterpret_cast<uint32_t*>(smem + rl * kBlk + gn * 32 + 16 * n + 4 * g4) =
            odd ? quantize4(v, inv) : pack_e4m3(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      }
      if (gn == 0 && g4 == 0 && rl < rows) p.cs[(row0 + rl) * p.cs_pitch + nt] = (uint8_t)code;
    });
    __syncthreads();
    uint8_t* C = static_cast<uint8_t*>(p.c) + row0 * p.ldc + (int64_t)nt * kBlk;
    for (int idx = (int)threadIdx.x; idx < rows * 8; idx += NT)
      *reinterpret_cast<uint4*>(C + (int64_t)(idx >> 3) * p.ldc + (idx & 7) * 16) =
          *reinterpret_cast<const uint4*>(smem + (idx >> 3) * kBlk + (idx & 7) * 16);
  }
}

// ------------------------------------------------------------------ sums over slots
// out[t] = add[t] + sum_j g[t, j] Y[t k + j] of F8_HALF rows (g null: 1), one rounding. A thread has eight columns;
// the k rows' loads (compiled for k up to 8) are all issued before the first is used. Bound by HBM: 32768 x 8 rows of
// 2048 in 230 us (5.2 TB/s), 261 right behind the product that wrote them. (Rows left in the products' order and read
// through the inverse permutation: the product 702 -> 670 us, the sum 243, but 60 -> 65 and 277 -> 270 for 16384 x 4:
// not worth a second form.)
template <typename T, int KF>
__global__ __launch_bounds__(256) void combine_half_kernel(const uint16_t* __restrict__ Y, const uint8_t* __restrict__ S,
                                                           int64_t ldy, int64_t pitch, const float* __restrict__ g,
                                                           const T* __restrict__ add, int64_t T_, int k_rt, int64_t N,
                                                           T* __restrict__ out, const int64_t* __restrict__ out_rows,
                                                           int64_t out_total, int vec, uint32_t chunks) {
  const int k = KF > 0 ? KF : k_rt;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t t = idx / chunks;
  if (t >= T_) return;
  const int64_t c = (idx - t * chunks) * 8;
  const int64_t orow = out_rows ? out_rows[t] : t;
  if (orow < 0 || orow >= out_total) return;
  float acc[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u] = 0.f;
  auto one = [&](const uint4& y, int code, float w) {
    const f16x8_t h = __builtin_bit_cast(f16x8_t, y);
    const float sc = __int_as_float(code << 23);  // (code >= 1: a normal number)
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u] = fmaf(w, (float)h[u] * sc, acc[u]);
  };
  const uint16_t* y0 = Y + t * k * ldy + c;
  const uint8_t* s0 = S + t * k * pitch + c / kHalfCols;
  if constexpr (KF > 0) {
    uint4 y[KF];
    int code[KF];
#pragma unroll
    for (int j = 0; j < KF; ++j) {
      y[j] = *reinterpret_cast<const uint4*>(y0 + j * ldy);
      code[j] = s0[j * pitch];
    }
#pragma unroll
    for (int j = 0; j < KF; ++j) one(y[j], code[j], g ? g[t * KF + j] : 1.f);
  } else {
    for (int j = 0; j < k; ++j) one(*reinterpret_cast<const uint4*>(y0 + j * ldy), s0[j * pitch], g ? g[t * k + j] : 1.f);
  }
  if (add) {
    float v[8];
    load8(add + t * N, c, N, vec ? W_CHUNK : W_ONE, v);
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u] += v[u];
  }
  T* o = out + orow * N + c;
  if (vec && c + 8 <= N) {
    constexpr int VN = 16 / sizeof(T);
#pragma unroll
    for (int q = 0; q < 8 / VN; ++q) *reinterpret_cast<uint4*>(o + q * VN) = pack_chunk(&acc[q * VN], T{});
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (c + u < N) o[u] = from_f32<T>(acc[u]);
  }
}

// ------------------------------------------------------------------ a few rows against one weight
// At most 32 rows read the weight once and hardly compute: a workgroup takes 16 columns, its eight waves share out
// the depth, and each wave loads its part of the weight straight into the matrix instruction's registers, up to four
// blocks of 128 ahead, with no LDS and no barrier before the one sum over the waves (in their order).
// One row, 2048 -> 1536: 4.3 us, 4096 -> 4096: 5.0, 16384 -> 4096: 13.5 (5.0 TB/s, the copy rate); 32 rows 5.5, 9.6
// and 30.8. Tiles of 32 x 128 that walk the whole depth: 8.9, 14.4, 48 for one row, 9.1, 14.7, 49 for 32. At 64 rows
// the two are level (8.0 and 9.1, 16.0 and 15.1, 52 and 49), as every workgroup reads all rows here.
constexpr int kFewWaves = 8;
constexpr int kCus = 256;

// What a lane of a fragment holds of a block of a row before it is quantised: values 16 g .. 16 g + 15 and 64 more on.
template <typename T>
struct Raw8 {
  static constexpr int VN = 16 / sizeof(T);
  uint4 w[32 / VN];
  __device__ __forceinline__ void load(const T* __restrict__ row, int64_t c, int64_t K) {  // K in whole eights
#pragma unroll
    for (int q = 0; q < 32 / VN; ++q) {
      const int64_t at = c + (q * VN & 15) + (q * VN & 16) * 4;
      w[q] = at < K ? *reinterpret_cast<const uint4*>(row + at) : make_uint4(0, 0, 0, 0);
    }
  }
  // The block's scale (its four lanes are this row's) and the lane's part of it: quantize_rows_kernel's bytes.
  __device__ __forceinline__ int quantize(Frag8& f) const {
    float v[32];
#pragma unroll
    for (int q = 0; q < 32 / VN; ++q) unpack_chunk(w[q], &v[q * VN], T{});
    uint32_t a = 0;
#pragma unroll
    for (int u = 0; u < 32; ++u) a = max(a, __float_as_uint(v[u]) & 0x7fffffffu);
    const bool odd = __builtin_amdgcn_ballot_w64(a >= kInfBits) != 0;
    if (odd) {
      float m = 0.f;
#pragma unroll
      for (int u = 0; u < 32; ++u) m = fmaxf(m, finite_abs(v[u]));
      a = __float_as_uint(m);
    }
    const int code = scale_code(__uint_as_float(max_rows4(a)));
    const float inv = scale_inverse(code);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float x[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      const int b = (int)(odd ? quantize4(x, inv) : pack_e4m3(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv));
      if (q < 4) f.lo[q] = b;
      else f.hi[q - 4] = b;
    }
    return code;
  }
};

// X: uint8_t for quantised rows, or the type of rows (at most 16 of them) that each wave quantises for itself as it goes,
// in registers: its lanes hold whole blocks. (One bf16 row 2048 -> 1536: 5.6 us, 6.4 with a launch of the quantiser;
// 16 rows 4096 -> 4096 9.8 and 9.7, in one call less; one row 16384 -> 4096 24.8 and 16.3, as every workgroup quantises the
// rows again.)
template <int MF, int U, int EPI, typename X>
__global__ __launch_bounds__(kFewWaves * 64) void fp8_few_kernel(Fp8Params p) {
  constexpr bool RAW = !std::is_same<X, uint8_t>::value;
  static_assert(!RAW || MF == 1, "16 rows");
  __shared__ float part[kFewWaves][16][20];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int lane = (int)threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const int col0 = (int)blockIdx.x * 16, rows = p.ns_m;
  const int each = (p.nk + kFewWaves - 1) / kFewWaves, k0 = wave * each;
  const int cnt = p.nk - k0 < each ? p.nk - k0 : each;  // (may be below 1)

  // rows and columns past the end repeat the last one: their outputs are not stored
  const int n = col0 + r16 < p.N ? col0 + r16 : p.N - 1;
  const uint8_t *a[MF], *as[MF], *b = p.b + ((int64_t)n * p.nk + k0) * kBlk + 16 * g4;
  const uint8_t* bs = p.bs + (int64_t)(col0 / kBlk) * p.bs_pitch + k0;
  const X* x = reinterpret_cast<const X*>(p.a) + (r16 < rows ? r16 : rows - 1) * p.a_pitch;  // RAW: K is lda
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const int r = 16 * m + r16 < rows ? 16 * m + r16 : rows - 1;
    a[m] = p.a + (int64_t)r * p.lda + (int64_t)k0 * kBlk + 16 * g4;
    as[m] = p.as + (int64_t)r * p.a_pitch + k0;
  }
  f32x4_t acc[MF];
#pragma unroll
  for (int m = 0; m < MF; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto load = [](const uint8_t* q) { return *reinterpret_cast<const v4i32_t*>(q); };
  for (int i = 0; i < cnt; i += U) {
    Frag8 fb[U], fa[U][MF];
    int sb[U], sa[U][MF];
    Raw8<std::conditional_t<RAW, X, float>> raw[RAW ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = i + u < cnt ? i + u : cnt - 1;
      sb[u] = bs[kb];
      fb[u].lo = load(b + (int64_t)kb * kBlk);
      fb[u].hi = load(b + (int64_t)kb * kBlk + 64);
      if constexpr (RAW) {
        raw[u].load(x, (int64_t)(k0 + kb) * kBlk + 16 * g4, p.lda);
      } else {
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          fa[u][m].lo = load(a[m] + (int64_t)kb * kBlk);
          fa[u][m].hi = load(a[m] + (int64_t)kb * kBlk + 64);
          sa[u][m] = as[m][kb];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads first
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u < cnt) {
        if constexpr (RAW) sa[u][0] = raw[u].quantize(fa[u][0]);
#pragma unroll
        for (int m = 0; m < MF; ++m)
          acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[u].value(), fa[u][m].value(), acc[m], 0, 0, 0,
                                                                   sb[u], 0, sa[u][m]);
      }
  }
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (m) __syncthreads();
    *reinterpret_cast<f32x4_t*>(&part[wave][r16][4 * g4]) = acc[m];
    __syncthreads();
    if (threadIdx.x < 256) {
      const int r = (int)threadIdx.x >> 4, c = (int)threadIdx.x & 15;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWaves; ++w) v += part[w][r][c];
      if (16 * m + r < rows && col0 + c < p.N) {
        const int64_t at = (int64_t)(16 * m + r) * p.ldc + col0 + c;
        if constexpr (EPI == F8_STORE_F32) static_cast<float*>(p.c)[at] = v;
        else static_cast<uint16_t*>(p.c)[at] = bf16_bits(v);
      }
    }
  }
}

// ------------------------------------------------------------------ host side
// Row tiles of a launch, at most: an expert has at least one row in each, and at most one that is not full.
int64_t row_tiles(const Fp8Params& p, int64_t R, int bm) {
  const int64_t most = cdiv(R, bm) + (p.offsets ? (R < p.E ? R : p.E) : 0);
  return most < R ? most : R;
}

template <int BM, int BN, int NW, int NS, int EPI>
int launch8(Fp8Params p, int64_t R, hipStream_t s) {
  auto kern = fp8_rows_kernel<BM, BN, NW, NS, EPI>;
  constexpr int lds = Lds8<BM, BN, NW, NS>::total;
  int rc = prepare(kern, lds);
  if (rc) return rc;
  p.n_tiles = (int)(is_glu(EPI) ? blocks_of(p.half) : cdiv(p.N, BN));
  const int64_t mt = row_tiles(p, R, BM);
  const int64_t total = cdiv(mt * p.n_tiles, (int64_t)kXcds * kSlab) * kXcds * kSlab;  // either tile mapping
  ZMOE_REQUIRE(mt * p.n_tiles < (int64_t)0x7fffff00, ZMOE_ERR_SHAPE, "fp8 product: too many tiles");
  hipLaunchKernelGGL(kern, dim3((unsigned)total), dim3(NW * 64), lds, s, p);
  return check_launch("fp8 rows kernel");
}

template <int MF, int U, int EPI, typename X = uint8_t>
int launch_few(const Fp8Params& p, hipStream_t s) {
  auto kern = fp8_few_kernel<MF, U, EPI, X>;
  hipLaunchKernelGGL(kern, dim3((unsigned)cdiv(p.N, 16)), dim3(kFewWaves * 64), 0, s, p);
  return check_launch("fp8 few rows kernel");
}

// The tile. Wider ones read the operands less often (a 128-deep step of 256 x 256 is 64 KB for 16.8 MFLOP, of 64 x 128
// 24 KB for 2.1), narrower ones leave less of a short expert's last tile empty and put more workgroups on the 256 CUs.
// Measured in us, bf16 or f16 rows out unless GLU:
//  - A launch whose workgroups are on the CUs all at once takes the narrowest tile with which they are, its stages loaded
//    well ahead. 4096 -> 4096: 128 rows 15.5 (32 x 128), 19.0 (64 x 128); 1000 rows 25.8 (64 x 128), 33.3 (128 x 128);
//    2048 rows 50 (64 x 128), 39 (128 x 128), 47 (128 x 256). GLU, 2048 -> 2 x 768: 1000 rows 13.9 (32 x 256), 16.4
//    (64 x 256); 4000 rows 40, 22.5, 26.7 (128 x 256). One row for each of 32 experts: GLU 18.4 (32) and 22.9 (64), back
//    11.3 (64 x 128) and 13.7 (64 x 256).
//  - Experts of some tens of rows stream their weights: 64 x 256, three workgroups a CU. 128 experts of 2048 -> 2 x 768
//    (GLU) and back: 4 rows each 73 (76.6 with 32 x 256, 87 with 128 x 256) and 34.4 (38.6 with 64 x 128, 39.6); 32 each 79
//    (98, 94) and 37.3 (41.5, 42.3); 64 each 88 and 92.6, back 44.3 and 44.5; 126 each 109 and 119, back 70 and 66.
//    Of exact sums (two workgroups a CU): 4 rows each 79.5 with 32 x 256 and 82.3 with 64 x 256, 12 each 83 and 88.6,
//    21 each 95 and 84.
//  - Else 128 x 256, two workgroups a CU (one's prologue and epilogue run under the other's loop), or 256 x 256 for experts
//    of six or more such tiles, whose last one, half empty on average, then costs less than a tenth. 8192 x 7168 -> 4096:
//    189 and 175; 262144 rows over 128 experts, 2048 -> 2 x 768 (GLU): 815 and 797; 65536 rows over 128 experts: 244
//    and 263, over 64, 1536 -> 2048: 274 and 281; 16384 rows skewed over 64 experts, 7168 -> 2 x 2048 (GLU): 605 and
//    668, back 356 and 404. The depth moves this little: 2048 rows for each of 64 experts, f16 rows out, 768 -> 2048: 371
//    and 364, 1536 -> 2048: 544 and 533, 2048 -> 1536: 504 and 487, 7168 -> 1536: 1413 and 1341.
// Rows per expert are R / E: the host does not know which experts have rows, so skewed routing runs on tiles that are
// narrower than its large experts would take.
template <int EPI>
int dispatch8(const Fp8Params& p, int64_t R, hipStream_t s) {
  const int64_t per = R / p.E;
  const int n = is_glu(EPI) ? 2 * p.half : p.N;
  const auto fits = [&](int bm, int bn, int per_cu) { return row_tiles(p, R, bm) * cdiv(n, bn) <= per_cu * kCus; };
  if constexpr (is_glu(EPI)) {
    const bool exact = R * p.half <= kExactValues;
    if (fits(32, 256, 1) || (exact && per <= 16)) return launch8<32, 256, 4, 4, F8_GLU_EXACT>(p, R, s);
    if (exact) return launch8<64, 256, 4, 1, F8_GLU_EXACT>(p, R, s);
    if (per <= 128 || fits(64, 256, 3)) return launch8<64, 256, 4, 1, EPI>(p, R, s);
  } else {
    if constexpr (EPI != F8_HALF) {
      if (!p.offsets && R <= 16) return launch_few<1, 4, EPI>(p, s);
      if (!p.offsets && R <= 32) return launch_few<2, 2, EPI>(p, s);
    }
    if (fits(32, 128, 1)) return launch8<32, 128, 4, 4, EPI>(p, R, s);
    if (fits(64, 128, 2)) return launch8<64, 128, 4, 3, EPI>(p, R, s);
    if (p.offsets && per <= 64) return launch8<64, 256, 4, 1, EPI>(p, R, s);
    if (fits(128, 128, 3)) return launch8<128, 128, 4, 1, EPI>(p, R, s);
  }
  if (per >= 1536) return launch8<256, 256, 8, 2, EPI>(p, R, s);
  return launch8<128, 256, 4, 1, EPI>(p, R, s);
}

constexpr int64_t kMaxSpan8 = 0x7fff0000LL;  // bytes that a buffer resource addresses
constexpr int64_t kMaxRows8 = 0x7fffffffLL;

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int quantize_checks(const char* name, int64_t n, int64_t K, int dtype) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "%s: dtype %d", name, dtype);
  ZMOE_REQUIRE(n >= 0 && n < kMaxRows8 && K >= 1 && K < (1 << 30), ZMOE_ERR_SHAPE, "%s: bad sizes (%lld x %lld)", name,
               (long long)n, (long long)K);
  return ZMOE_OK;
}

}  // namespace
}  // namespace zmoe

using namespace zmoe;

extern "C" int zmoe_fp8_scale_pitch(int64_t K, int64_t* pitch) {
  ZMOE_REQUIRE(K >= 1 && K < (1 << 30), ZMOE_ERR_SHAPE, "fp8_scale_pitch: K=%lld", (long long)K);
  ZMOE_REQUIRE(pitch, ZMOE_ERR_NULL, "fp8_scale_pitch: null pointer");
  *pitch = scale_pitch(K);
  return ZMOE_OK;
}

extern "C" int zmoe_fp8_quantize_rows(const void* X, int64_t x_stride, int64_t x_rows, const int64_t* rows,
                                      int row_div, const float* row_scale, int64_t n, int64_t K, int dtype, void* Q,
                                      void* S, void* stream) {
  int rc = quantize_checks("fp8_quantize_rows", n, K, dtype);
  if (rc) return rc;
  ZMOE_REQUIRE(x_rows >= 0 && x_stride >= K && row_div >= 1, ZMOE_ERR_SHAPE,
               "fp8_quantize_rows: bad row stride, row count or divisor");
  ZMOE_REQUIRE(rows || n <= x_rows, ZMOE_ERR_SHAPE, "fp8_quantize_rows: more rows than X has");
  if (n == 0) return ZMOE_OK;
  ZMOE_REQUIRE(Q && S && (X || x_rows == 0), ZMOE_ERR_NULL, "fp8_quantize_rows: null pointer");
  ZMOE_REQUIRE(aligned16(Q) && aligned4(S), ZMOE_ERR_ALIGN, "fp8_quantize_rows: Q on 16, S on 4 bytes");
  const int64_t nb = blocks_of(K);
  ZMOE_REQUIRE(n * nb < (int64_t)0x7fffffff, ZMOE_ERR_SHAPE, "fp8_quantize_rows: too many blocks");
  const int width = row_width(X, x_stride, dtype_size(dtype));
  hipStream_t s = as_stream(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    const int64_t step = kMaxLaunchThreads / 256 * 16 / nb;  // rows of a launch
    for (int64_t i = 0; i < n; i += step) {
      const int64_t m = n - i < step ? n - i : step;
      // rows in order: X and the scales from row i; listed ones: the list
      hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3((unsigned)cdiv(m * nb, 16)), dim3(256), 0, s,
                         static_cast<const T*>(X) + (rows ? 0 : i * x_stride), x_stride, rows ? x_rows : x_rows - i,
                         rows ? rows + i : nullptr, row_div, row_scale && !rows ? row_scale + i : row_scale,
                         (uint32_t)(m * nb), K, (int)nb, width, static_cast<uint8_t*>(Q) + i * nb * kBlk,
                         static_cast<uint8_t*>(S) + i * scale_pitch(K), scale_pitch(K));
    }
  };
  if (dtype == ZMOE_DTYPE_BF16) go(uint16_t{});
  else go(float{});
  return check_launch("fp8_quantize_rows");
}

extern "C" int zmoe_fp8_quantize_weight(const void* W, int64_t w_stride_e, int64_t w_stride_n, int64_t E, int64_t N,
                                        int64_t K, int dtype, void* Q, void* S, void* Qt, void* St, void* stream) {
  int rc = quantize_checks("fp8_quantize_weight", N, K, dtype);
  if (rc) return rc;
  ZMOE_REQUIRE(N >= 1 && E >= 1 && E <= 65535 && w_stride_n >= K && w_stride_e >= 0, ZMOE_ERR_SHAPE,
               "fp8_quantize_weight: bad sizes or strides");
  ZMOE_REQUIRE(W && Q && S && (!Qt == !St), ZMOE_ERR_NULL, "fp8_quantize_weight: null pointer");
  ZMOE_REQUIRE(aligned16(Q) && aligned4(S) && aligned16(Qt) && aligned4(St), ZMOE_ERR_ALIGN,
               "fp8_quantize_weight: values on 16, scales on 4 bytes");
  ZMOE_REQUIRE(blocks_of(N) <= 65535, ZMOE_ERR_SHAPE, "fp8_quantize_weight: too many rows");
  const int size = dtype_size(dtype), wn = row_width(W, w_stride_n, size), we = row_width(W, w_stride_e, size);
  const int width = wn < we ? wn : we;
  const dim3 grid((unsigned)blocks_of(K), (unsigned)blocks_of(N), (unsigned)E);
  hipStream_t s = as_stream(stream);
  uint8_t *q = static_cast<uint8_t*>(Q), *sc = static_cast<uint8_t*>(S), *qt = static_cast<uint8_t*>(Qt),
          *st = static_cast<uint8_t*>(St);
  auto go = [&](auto t, auto trans) {
    using T = decltype(t);
    hipLaunchKernelGGL((quantize_weight_kernel<T, decltype(trans)::value>), grid, dim3(256), 0, s,
                       static_cast<const T*>(W), w_stride_e, w_stride_n, N, K, width, q, sc, qt, st);
  };
  if (dtype == ZMOE_DTYPE_BF16) {
    if (Qt) go(uint16_t{}, std::true_type{});
    else go(uint16_t{}, std::false_type{});
  } else {
    if (Qt) go(float{}, std::true_type{});
    else go(float{}, std::false_type{});
  }
  return check_launch("fp8_quantize_weight");
}

namespace {
// What both products check of A (rows of K values), its gather and B ([rows_b, K] per expert); fills them in.
int product_operands(const char* name, const void* Xq, const void* Xs, int64_t M, const void* Wq, const void* Ws,
                     int64_t K, int64_t rows_b, int64_t blocks_b, int E, const int64_t* offsets, Fp8Params& p) {
  ZMOE_REQUIRE(Xq && Xs && Wq && Ws, ZMOE_ERR_NULL, "%s: null pointer", name);
  ZMOE_REQUIRE(aligned16(Xq) && aligned4(Xs) && aligned16(Wq) && aligned4(Ws), ZMOE_ERR_ALIGN,
               "%s: values on 16, scales on 4 bytes", name);
  const int64_t nk = blocks_of(K);
  p.a = static_cast<const uint8_t*>(Xq);
  p.as = static_cast<const uint8_t*>(Xs);
  p.lda = nk * kBlk;
  p.a_pitch = scale_pitch(K);
  p.a_bytes = M * p.lda;
  p.b = static_cast<const uint8_t*>(Wq);
  p.bs = static_cast<const uint8_t*>(Ws);
  p.b_estride = rows_b * p.lda;
  p.bs_pitch = scale_pitch(K);
  p.bs_estride = blocks_b * p.bs_pitch;
  ZMOE_REQUIRE(p.b_estride <= kMaxSpan8, ZMOE_ERR_SHAPE, "%s: one expert's weights span more than 2 GiB", name);
  ZMOE_REQUIRE(!p.a_rows || p.a_bytes <= kMaxSpan8, ZMOE_ERR_SHAPE, "%s: gathered rows span more than 2 GiB", name);
  ZMOE_REQUIRE(256 * p.lda <= kMaxSpan8, ZMOE_ERR_SHAPE, "%s: K too large", name);
  p.b_bytes = (uint32_t)p.b_estride;
  p.nk = (int)nk;
  p.E = E;
  p.offsets = offsets;
  return ZMOE_OK;
}
}  // namespace

namespace {
// Both forms of the product; half: Y in f16 with scales Ys, else out_dtype.
int scatter2scatter8(const char* name, const void* Xq, const void* Xs, int64_t M, const void* Wq, const void* Ws,
                     const int64_t* sorted_scattered_idxs, const int64_t* expert_offsets, int64_t K, int64_t N, int E,
                     int k, int x_grouped, int y_grouped, int out_dtype, bool half, void* Y, void* Ys, int64_t y_stride,
                     void* stream) {
  ZMOE_REQUIRE(half || dtype_ok(out_dtype), ZMOE_ERR_DTYPE, "%s: dtype %d", name, out_dtype);
  ZMOE_REQUIRE(M >= 0 && K >= 1 && N >= 1 && K < (1 << 30) && N < (1 << 30) && E >= 1 && E <= kGemmMaxE && k >= 1,
               ZMOE_ERR_SHAPE, "%s: bad sizes (M=%lld K=%lld N=%lld E=%d k=%d)", name, (long long)M, (long long)K,
               (long long)N, E, k);
  ZMOE_REQUIRE(M < kMaxRows8 && M * (x_grouped ? 1 : k) < kMaxRows8, ZMOE_ERR_SHAPE, "%s: rows must be below 2^31", name);
  ZMOE_REQUIRE(expert_offsets || (E == 1 && x_grouped && y_grouped), ZMOE_ERR_NULL,
               "%s: no expert_offsets only for one weight and rows in order", name);
  ZMOE_REQUIRE(half || y_stride >= N, ZMOE_ERR_SHAPE, "%s: row stride of Y", name);
  const int64_t R = x_grouped ? M : M * k;
  if (R == 0) return ZMOE_OK;
  ZMOE_REQUIRE((x_grouped && y_grouped) || sorted_scattered_idxs, ZMOE_ERR_NULL,
               "%s: sorted_scattered_idxs required unless x_grouped and y_grouped", name);
  ZMOE_REQUIRE(Y && (!half || Ys), ZMOE_ERR_NULL, "%s: null pointer", name);
  ZMOE_REQUIRE(half ? aligned16(Y) : (reinterpret_cast<uintptr_t>(Y) % dtype_size(out_dtype)) == 0, ZMOE_ERR_ALIGN,
               "%s: Y's alignment", name);
  Fp8Params p{};
  p.a_rows = x_grouped ? nullptr : sorted_scattered_idxs;
  p.a_div = k;
  int rc = product_operands(name, Xq, Xs, M, Wq, Ws, K, N, blocks_of(N), E, expert_offsets, p);
  if (rc) return rc;
  p.c = Y;
  p.c_rows = y_grouped ? nullptr : sorted_scattered_idxs;
  p.N = (int)N;
  p.n_major = x_grouped ? 1 : 0;
  p.ns_m = expert_offsets ? 0 : (int)M;
  hipStream_t s = as_stream(stream);
  if (half) {
    p.cs = static_cast<uint8_t*>(Ys);
    p.cs_pitch = cdiv(N, kHalfCols);
    p.ldc = p.cs_pitch * kHalfCols;
    return dispatch8<F8_HALF>(p, R, s);
  }
  p.ldc = y_stride;
  p.vec_c = aligned16(Y) && y_stride % (16 / dtype_size(out_dtype)) == 0;
  return out_dtype == ZMOE_DTYPE_BF16 ? dispatch8<F8_STORE_BF16>(p, R, s) : dispatch8<F8_STORE_F32>(p, R, s);
}
}  // namespace

extern "C" int zmoe_fp8_scatter2scatter(const void* Xq, const void* Xs, int64_t M, const void* Wq, const void* Ws,
                                        const int64_t* sorted_scattered_idxs, const int64_t* expert_offsets, int64_t K,
                                        int64_t N, int E, int k, int x_grouped, int y_grouped, int out_dtype, void* Y,
                                        int64_t y_stride, void* stream) {
  return scatter2scatter8("fp8_scatter2scatter", Xq, Xs, M, Wq, Ws, sorted_scattered_idxs, expert_offsets, K, N, E, k,
                          x_grouped, y_grouped, out_dtype, false, Y, nullptr, y_stride, stream);
}

extern "C" int zmoe_fp8_linear_few(const void* X, int64_t x_stride, int64_t M, const void* Wq, const void* Ws, int64_t K,
                                   int64_t N, int dtype, void* Y, int64_t y_stride, void* stream) {
  int rc = quantize_checks("fp8_linear_few", M, K, dtype);
  if (rc) return rc;
  ZMOE_REQUIRE(M <= 16 && K % 8 == 0 && N >= 1 && N < (1 << 30) && x_stride >= K &&
                   x_stride % (16 / dtype_size(dtype)) == 0 && y_stride >= N,
               ZMOE_ERR_SHAPE, "fp8_linear_few: at most 16 rows in whole 16-byte chunks (M=%lld K=%lld N=%lld)",
               (long long)M, (long long)K, (long long)N);
  if (M == 0) return ZMOE_OK;
  ZMOE_REQUIRE(X && Y, ZMOE_ERR_NULL, "fp8_linear_few: null pointer");
  ZMOE_REQUIRE(aligned16(X) && (reinterpret_cast<uintptr_t>(Y) % dtype_size(dtype)) == 0, ZMOE_ERR_ALIGN,
               "fp8_linear_few: X on 16 bytes, Y on its elements");
  Fp8Params p{};
  rc = product_operands("fp8_linear_few", X, Ws, M, Wq, Ws, K, N, blocks_of(N), 1, nullptr, p);
  if (rc) return rc;
  p.as = nullptr;
  p.lda = K;
  p.a_pitch = x_stride;
  p.c = Y;
  p.ldc = y_stride;
  p.N = (int)N;
  p.ns_m = (int)M;
  hipStream_t s = as_stream(stream);
  return dtype == ZMOE_DTYPE_BF16 ? launch_few<1, 4, F8_STORE_BF16, uint16_t>(p, s)
                                  : launch_few<1, 2, F8_STORE_F32, float>(p, s);
}

extern "C" int zmoe_fp8_scatter2scatter_half(const void* Xq, const void* Xs, int64_t M, const void* Wq, const void* Ws,
                                             const int64_t* sorted_scattered_idxs, const int64_t* expert_offsets,
                                             int64_t K, int64_t N, int E, int k, int x_grouped, int y_grouped, void* Y,
                                             void* Ys, void* stream) {
  return scatter2scatter8("fp8_scatter2scatter_half", Xq, Xs, M, Wq, Ws, sorted_scattered_idxs, expert_offsets, K, N, E,
                          k, x_grouped, y_grouped, 0, true, Y, Ys, 0, stream);
}

extern "C" int zmoe_combine_half(const void* Y, const void* Ys, const float* gates, const void* addend, int64_t T, int k,
                                 int64_t N, int dtype, const int64_t* out_rows, int64_t out_total, void* out,
                                 void* stream) {
  ZMOE_REQUIRE(dtype_ok(dtype), ZMOE_ERR_DTYPE, "combine_half: dtype %d", dtype);
  ZMOE_REQUIRE(T >= 0 && T < kMaxRows8 && k >= 1 && T * k < kMaxRows8 && N >= 1 && N < (1 << 30) && out_total >= 0,
               ZMOE_ERR_SHAPE, "combine_half: bad sizes");
  if (T == 0) return ZMOE_OK;
  ZMOE_REQUIRE(Y && Ys && out, ZMOE_ERR_NULL, "combine_half: null pointer");
  ZMOE_REQUIRE(aligned16(Y), ZMOE_ERR_ALIGN, "combine_half: Y on 16 bytes");
  const int64_t chunks = cdiv(N, 8), pitch = cdiv(N, kHalfCols), blocks = cdiv(T * chunks, 256);
  ZMOE_REQUIRE(launch_fits(blocks, 256), ZMOE_ERR_SHAPE, "combine_half: too many elements");
  const int vec = aligned16(out) && aligned16(addend) && N % (16 / dtype_size(dtype)) == 0;
  auto go = [&](auto tt, auto kf) {
    using TT = decltype(tt);
    hipLaunchKernelGGL((combine_half_kernel<TT, decltype(kf)::value>), dim3((unsigned)blocks), dim3(256), 0,
                       as_stream(stream), static_cast<const uint16_t*>(Y), static_cast<const uint8_t*>(Ys),
                       pitch * kHalfCols, pitch, gates, static_cast<const TT*>(addend), T, k, N, static_cast<TT*>(out),
                       out_rows, out_rows ? out_total : T, vec, (uint32_t)chunks);
  };
  auto by_k = [&](auto tt) {
    if (k == 8) go(tt, std::integral_constant<int, 8>{});
    else if (k == 4) go(tt, std::integral_constant<int, 4>{});
    else if (k == 2) go(tt, std::integral_constant<int, 2>{});
    else go(tt, std::integral_constant<int, 0>{});
  };
  if (dtype == ZMOE_DTYPE_BF16) by_k(uint16_t{});
  else by_k(float{});
  return check_launch("combine_half");
}

extern "C" int zmoe_fp8_glu_w1_forward(const void* Xq, const void* Xs, int64_t T, const void* W1q, const void* W1s,
                                       const int64_t* sorted_scattered_idxs, const int64_t* expert_offsets, int64_t d,
                                       int64_t f, int E, int k, void* Aq, void* As, void* stream) {
  ZMOE_REQUIRE(T >= 0 && d >= 1 && f >= 1 && d < (1 << 30) && f < (1 << 29) && E >= 1 && E <= kGemmMaxE && k >= 1,
               ZMOE_ERR_SHAPE, "fp8_glu_w1_forward: bad sizes");
  ZMOE_REQUIRE(T < kMaxRows8 && T * k < kMaxRows8, ZMOE_ERR_SHAPE, "fp8_glu_w1_forward: T*k must be below 2^31");
  const int64_t R = T * k;
  if (R == 0) return ZMOE_OK;
  ZMOE_REQUIRE(expert_offsets ? sorted_scattered_idxs != nullptr : (E == 1 && k == 1), ZMOE_ERR_NULL,
               "fp8_glu_w1_forward: no expert_offsets only for one weight, else sorted_scattered_idxs too");
  ZMOE_REQUIRE(Aq && As, ZMOE_ERR_NULL, "fp8_glu_w1_forward: null pointer");
  ZMOE_REQUIRE(aligned16(Aq) && aligned4(As), ZMOE_ERR_ALIGN, "fp8_glu_w1_forward: values on 16, scales on 4 bytes");
  Fp8Params p{};
  p.a_rows = expert_offsets ? sorted_scattered_idxs : nullptr;
  p.a_div = k;
  int rc = product_operands("fp8_glu_w1_forward", Xq, Xs, T, W1q, W1s, d, 2 * f, 2 * blocks_of(f), E, expert_offsets, p);
  if (rc) return rc;
  p.c = Aq;
  p.ldc = blocks_of(f) * kBlk;
  p.cs = static_cast<uint8_t*>(As);
  p.cs_pitch = scale_pitch(f);
  p.half = (int)f;
  p.N = (int)(2 * f);
  p.n_major = 0;
  p.ns_m = expert_offsets ? 0 : (int)T;
  return dispatch8<F8_GLU>(p, R, as_stream(stream));
}
