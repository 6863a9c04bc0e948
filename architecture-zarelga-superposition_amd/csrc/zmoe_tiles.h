// Tile machinery shared by the grouped GEMM kernels (gemm.hip, fp8.hip): the mapping of workgroups
// to (expert, m-tile, n-tile), loads from HBM straight into LDS, and LDS fragment reads that the
// compiler does not order behind them.
#pragma once

#include <mutex>
#include <unordered_set>

#include "zmoe_internal.h"

namespace zmoe {

constexpr int kGemmMaxE = 1024;
constexpr int kXcds = 8;

// ------------------------------------------------------------------ block scan
template <int NT = 256>
__device__ __forceinline__ int block_exclusive_scan(int v, int* tmp, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int base = 0, tot = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    const int t = tmp[w];
    if (w < wave) base += t;
    tot += t;
  }
  *total = tot;
  return base + x - v;
}

// Logical tile of this workgroup under the XCD-aware mapping, or -1.
__device__ __forceinline__ int xcd_logical_tile(int total) {
  const int xcd = blockIdx.x % kXcds, slot = blockIdx.x / kXcds;
  const int chunk = (total + kXcds - 1) / kXcds;
  const int logical = xcd * chunk + slot;
  return (slot < chunk && logical < total) ? logical : -1;
}

// Logical tile under slabs of kSlab consecutive tiles (the workgroups one XCD holds at
// once) dealt to the XCDs in turn. The weight-grad launches always map this way: a
// weight-grad tile's cost grows with its expert's rows, so xcd_logical_tile's contiguous
// per-XCD ranges (equal tile counts) leave the XCD that holds a popular expert with most
// of the work when routing is skewed: 2.4x the mean at C4's Zipf(1.1) popularity, dW1 +
// dW2 13.0 -> 10.1 ms with slabs. A slab still keeps 32 concurrent tiles of one expert on
// one XCD (same time as the contiguous ranges at C3; slabs of 8 time the same at C4, of 1
// are 3-11% slower at C3). A launch of at most 8 slabs (the dense split-K grads) takes one
// slab of ceil(total / 8) tiles per XCD, i.e. the contiguous ranges, so no XCD sits idle.
// The launches round their grids up to whole slabs on every XCD.
constexpr int kSlab = 32;
// Tile order within one expert, for position `loc` of its ninner x nouter tiles: the
// inner index (the tiles sharing the outer operand block) runs fastest, in serpentine order
// (backwards on odd outer steps, so the tiles either side of a turn share a block too:
// 0.3-0.8% per launch). An expert with at least 2 * kBand inner tiles takes its inner index
// in bands of kBand, the outer index reversed on odd bands, so that the ~32 tiles an XCD
// runs at once span about kBand x 4 tiles instead of one or two outer steps of 16-32:
// a one-expert 262144 x 2048 x 2048 GEMM with one n-tile per column of 32 read X once per
// XCD (8.86 GB from HBM for 1.08 GB of operands; banded 3.23 GB, 2.02 -> 1.84 ms), and
// C4's W1 forward (16 pair-column tiles) read each expert's weights once per two m-tiles
// (banded 4.46 -> 4.30 ms).
constexpr int kBand = 8;
__device__ __forceinline__ void expert_tile_order(int loc, int ninner_all, int nouter, int& inner, int& outer) {
  const int band = ninner_all >= 2 * kBand ? kBand : ninner_all;
  const int b = loc / (band * nouter), lb = loc - b * band * nouter;
  const int ninner = min(band, ninner_all - b * band);
  const int outer0 = lb / ninner, in0 = lb % ninner;
  outer = (b & 1) ? nouter - 1 - outer0 : outer0;
  inner = b * band + ((outer0 & 1) ? ninner - 1 - in0 : in0);
}
__host__ __device__ __forceinline__ int slab_size(int64_t total) {
  const int64_t per_xcd = (total + kXcds - 1) / kXcds;
  return per_xcd < kSlab ? (int)(per_xcd > 0 ? per_xcd : 1) : kSlab;
}
__device__ __forceinline__ int slab_logical_tile(int total, int b = -1) {
  if (b < 0) b = (int)blockIdx.x;
  const int slab = slab_size(total);
  const int xcd = b % kXcds, slot = b / kXcds;
  const int logical = ((slot / slab) * kXcds + xcd) * slab + slot % slab;
  return logical < total ? logical : -1;
}

struct RowsTile {
  int e, nt, rows, mt;  // mt: m-tile index within the expert (symmetric launches)
  int64_t row0;
};

// Map this workgroup to (expert, m-tile, n-tile) of a rows launch; false if it has no tile. P holds
// offsets (inclusive expert ends), E, n_tiles, n_major, ns_m and ns_sym.
template <int BM, int NT = 256, typename P>
__device__ __forceinline__ bool decode_rows_tile(const P& p, char* smem, RowsTile& t) {
  if (p.ns_m > 0) {
    // equal experts: no offsets to read; symmetric ones run the upper-triangle tiles (nt >= mt)
    const int nm = (p.ns_m + BM - 1) / BM;
    const int per = p.ns_sym ? nm * (nm + 1) / 2 : nm * p.n_tiles;
    const int logical = xcd_logical_tile(p.E * per);
    if (logical < 0) return false;
    t.e = logical / per;
    int r = logical % per;
    if (p.ns_sym) {
      int mt = 0;
      while (r >= nm - mt) {
        r -= nm - mt;
        ++mt;
      }
      t.mt = mt;
      t.nt = mt + r;
    } else {
      expert_tile_order(r, p.n_tiles, nm, t.nt, t.mt);
    }
    t.row0 = (int64_t)t.e * p.ns_m + (int64_t)t.mt * BM;
    t.rows = min(BM, p.ns_m - t.mt * BM);
    return true;
  }
  // One pass over the expert ends: each thread counts the m-tiles of its experts, a
  // block scan places them, and the thread whose expert holds this workgroup's m-tile
  // posts (expert, first row, rows) to LDS. The offsets are read once, so the decode
  // costs one global round trip.
  int64_t* found = reinterpret_cast<int64_t*>(smem);  // [0] expert, [1] first row, [2] rows, [3] n-tile
  int* tmp = reinterpret_cast<int*>(smem + 32);
  const int ept = (p.E + NT - 1) / NT;  // <= 4
  const int e0 = threadIdx.x * ept;
  int64_t ebeg[4] = {0, 0, 0, 0}, eend[4] = {0, 0, 0, 0};
  int ntl[4] = {0, 0, 0, 0};
  int local = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int e = e0 + q;
    if (q < ept && e < p.E) {
      ebeg[q] = e ? p.offsets[e - 1] : 0;
      eend[q] = p.offsets[e];
      const int64_t c = eend[q] > ebeg[q] ? eend[q] - ebeg[q] : 0;
      ntl[q] = (int)((c + BM - 1) / BM);
      local += ntl[q];
    }
  }
  // experts whose rows fit one m-tile, per wave (ballots: no LDS round trips)
  int single = 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) single += __builtin_popcountll(__builtin_amdgcn_ballot_w64(ntl[q] == 1));
  int* single_w = tmp + 16;  // per-wave counts; the scan's barrier orders them before the reads
  if ((threadIdx.x & 63) == 0) single_w[threadIdx.x >> 6] = single;
  // expert e owns ntl_e * n_tiles consecutive logical tiles, its m-tiles outer (tiles
  // sharing A rows run together) or its n-tiles outer (tiles sharing B columns do)
  int ttiles;
  int run = block_exclusive_scan<NT>(local * p.n_tiles, tmp, &ttiles);
  int singles = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) singles += single_w[w];
  // Skewed routing, with over a quarter of the experts in a single m-tile: their tiles
  // stream a whole weight block for a few rows (HBM-bound) beside the compute-bound tiles
  // of the popular experts, and slabs give every XCD its share of both (C4: W1 forward 6%,
  // W1 input grad 4% faster). Otherwise each XCD keeps whole experts (1% faster at C3).
  const int logical = 4 * singles > p.E ? slab_logical_tile(ttiles) : xcd_logical_tile(ttiles);
  if (logical < 0) return false;  // uniform per workgroup
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int tiles_e = ntl[q] * p.n_tiles;
    if (logical >= run && logical < run + tiles_e) {  // (ntl[q] is 0 past the last expert)
      int in2, outer;
      expert_tile_order(logical - run, p.n_major ? ntl[q] : p.n_tiles, p.n_major ? p.n_tiles : ntl[q], in2, outer);
      const int mt = p.n_major ? in2 : outer;
      const int64_t r0 = ebeg[q] + (int64_t)mt * BM;
      found[0] = e0 + q;
      found[1] = r0;
      found[2] = min((int64_t)BM, eend[q] - r0);
      found[3] = p.n_major ? outer : in2;
    }
    run += tiles_e;
  }
  __syncthreads();
  t.e = (int)found[0];
  t.row0 = found[1];
  t.rows = (int)found[2];
  t.nt = (int)found[3];
  t.mt = 0;
  __syncthreads();  // the decode area is dead; LDS becomes operand stages
  return true;
}

// ------------------------------------------------------------------ HBM -> LDS loads
typedef __attribute__((address_space(3))) char lds_char;
typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef short v8i16_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16;
typedef __attribute__((address_space(3))) uint4 lds_uint4;

constexpr uint32_t kOOB = 0x80000000u;  // any offset >= num_records reads zero

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void buf_to_lds(__amdgpu_buffer_rsrc_t r, lds_char* dst, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)dst, 16, voff, 0, 0, 0);
}

// s_waitcnt immediate that waits until at most n vector-memory ops are outstanding.
constexpr int vm_wait(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// ------------------------------------------------------------------ LDS fragment reads
// Fragment reads are inline asm: LLVM's waitcnt pass makes any LDS read it cannot
// disambiguate (the ds_read_tr intrinsic carries no alias info) wait for every
// in-flight LDS-DMA load, which would serialise the stage pipeline. Being asm,
// these reads are invisible to that pass, so the K loops issue their own
// lgkmcnt waits and ties the fragment registers to them with empty asm (data
// dependencies keep every MFMA after the wait that covers its operands).
typedef int v4i32_t __attribute__((ext_vector_type(4)));
typedef int v2i32_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t lds_addr(const lds_char* p) { return (uint32_t)(uintptr_t)p; }

__device__ __forceinline__ v4i32_t asm_ds_read_b128(uint32_t addr) {
  v4i32_t v;
  asm volatile("ds_read_b128 %0, %1" : "=v"(v) : "v"(addr));
  return v;
}
__device__ __forceinline__ v2i32_t asm_ds_read_tr16(uint32_t addr) {
  v2i32_t v;
  asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(v) : "v"(addr));
  return v;
}
template <int N>
__device__ __forceinline__ void asm_wait_lgkm() {
  asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(N < 15 ? N : 15));
}
__device__ __forceinline__ void asm_tie(v4i32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ void asm_tie(v2i32_t& v) { asm volatile("" : "+v"(v)); }

// ------------------------------------------------------------------ host side
// One attribute call per kernel (keyed by the kernel's address: instantiations share a
// function type), under a lock, since callers may launch from several host threads.
template <typename K>
int prepare(K kernel, int lds_bytes) {
  static std::mutex mu;
  static std::unordered_set<const void*> done;
  const void* key = reinterpret_cast<const void*>(kernel);
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(key)) return ZMOE_OK;
  hipError_t e = hipFuncSetAttribute(key, hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
  if (e != hipSuccess) return set_error(ZMOE_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  done.insert(key);
  return ZMOE_OK;
}

}  // namespace zmoe
