// Products of many rows with affine 4-bit weights on the 5th-generation tensor cores
// (sm_100a): y = x W^T for one weight matrix, or one per expert over rows sorted by expert.
//
// Roles swapped so that ragged row counts cost what they are: the MMA's 128 M rows are weight
// rows and its N columns are rows of x, any multiple of 16 up to 192, so an expert with 40
// rows pays for 48. Weights become the A operand in TENSOR memory: a dequantizer thread owns
// one weight row, turns a group of 64 codes into 16-bit values in registers and stores them
// to its lane, so dequantized weights touch neither HBM nor shared memory. Rows of x are the
// B operand in shared memory, by TMA (128-byte swizzle).
//
//   * Persistent CTAs, one per SM. A tile is (expert, up to 192 of its rows, 128 weight rows);
//     an expert's rows are cut into equal tiles. Every CTA takes a contiguous range of the
//     tiles, equally many (a tile takes the dequantizers about the same time whatever its rows),
//     computed by each CTA from the offsets: nothing is counted through memory, and
//     neighbouring tiles share rows of x in L2.
//   * Warps: 0 issues the MMAs, 1 loads rows of x (TMA), 2 packed codes (TMA), 3 scales, 4-19
//     dequantize (four warpgroups: the two halves of 128 K values, two such in turn), 20-23
//     store results.
//   * Tensor memory: two accumulators of 192 columns (a tile's results are stored while the
//     next one accumulates) and four A stages of 32 columns (64 K values each).
//   * Gated activation: 16 gate rows and the 16 up rows of the same outputs share a warp's 32
//     lanes, so the epilogue exchanges them with one shuffle per two values.
//
// Rounding: a weight is rounded once to x's type, round(scale * code + bias) by a fused
// multiply-add, the value mx.dequantize gives; sums are fp32. The kernel for few rows rounds no
// weight: relative to the exact product the results are off by 2.2e-3 (bf16, the output's own
// rounding included) against its 1.7e-3, of a gated product by 2.7e-3 against 1.7e-3; in f16 by
// 2.8e-4 and 3.4e-4 against 2.1e-4. A choice, which the documents of the calls state: weights in
// two terms need twice the MMAs, and those alone take 2048 rows through 5120x2048 from 32.6 to 54.6
// us, 16384 expert rows from 143 to 210 and 1332 from 39 to 53 (measured with every MMA issued
// twice), for an error that stays below the result's own rounding in all but the gated products.
//
// What bounds it, measured: 128 experts of 1536x2048 at 16384 rows, 143 us: the tensor pipe is
// busy 47% of the time, the ALU pipe with dequantizing 52% (its warps wait for
// freed A stages about as often as the MMAs wait for full ones), HBM at 1.8 TB/s. 2048 rows through
// 5120x2048: 32.6 us, 1320 TFLOP/s, tensor pipe 62 to 76%. Run without a pause both are at the
// card's power limit (1540 MHz): 168 and 40 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "matmul_internal.h"
#include "qkv_common.cuh"
#include "qkv_internal.h"
#include "tc_common.cuh"

namespace qkv {

namespace {

constexpr int kWarps = 24;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxTok = 192;           // rows of x in a tile
constexpr int kBoxRows = 32;           // rows of x are copied in multiples of this
constexpr int kAStages = 4;            // of 64 K values, in tensor memory
constexpr int kACol = 2 * kMaxTok;     // first A column
constexpr int kMaxBStages = 8;         // of 128 K values
constexpr int kBBytes = 144 * 1024;    // shared memory of the B stages
constexpr int kSlots = 4;              // prefetched stages of packed codes, two per turn
constexpr int kSlotBytes = 128 * 64;   // 128 weight rows x 64 bytes: 128 K values
constexpr int kScaleGroups = 16;       // groups of a staged piece of scales and biases
constexpr int kScalePitch = 48;        // bytes of a row of a piece
constexpr int kScaleBytes = 2 * 128 * kScalePitch;  // one piece: 128 rows of both
// barriers, in shared memory: pairs of full and free by stage
constexpr int kBarA = 0, kBarFreed = kBarA + kAStages, kBarB = kBarFreed + kAStages, kBarC = kBarB + 2 * kMaxBStages,
              kBarS = kBarC + 2 * kSlots;
constexpr int kBarAcc = kBarS + 4, kBarFin = kBarAcc + 4, kBars = kBarFin + 1;
constexpr int kMaxExperts = 1024;

struct TcArgs {
  CUtensorMap codes;  // (E * N, K/2) bytes; boxes of 128 rows, or of 16 gate or up rows
  CUtensorMap x[kMaxTok / kBoxRows];  // (x_rows, K); boxes of 1, 2, ... times kBoxRows rows
  MatmulArgs a;
  int tok;       // most rows of x per tile (a multiple of 16)
  int b_stages;
  int n_tiles;   // tiles of 128 weight rows
  bool gathered; // rows of x by gather_rows_kernel just before
};

struct Split {
  int n;    // row tiles of an expert
  int per;  // rows of each (a multiple of 16; the last may have fewer)
};
__host__ __device__ inline Split split_rows(int count, int tok) {
  if (count <= 0) return {0, 16};
  const int n = (count + tok - 1) / tok;
  const int per = ((count + n - 1) / n + 15) / 16 * 16;
  return {(count + per - 1) / per, per};
}
__host__ __device__ inline int stage_rows(int tok) { return (tok + kBoxRows - 1) / kBoxRows * kBoxRows; }
template <typename T>
struct Conv;
template <>
struct Conv<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128 + code, exact
  static __device__ __forceinline__ uint32_t sub(uint32_t a) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(kMagic));
    return d;
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
};
template <>
struct Conv<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;  // 1024 + code, exact
  static __device__ __forceinline__ uint32_t sub(uint32_t a) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(kMagic));
    return d;
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
};

// a 16-bit value in both halves
__device__ __forceinline__ uint32_t lds_u16x2(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
  return v * 0x10001u;
}
__device__ __forceinline__ void lds_v4(uint32_t at, uint32_t* v) {
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// 1 for one lane of a converged warp, the same each time
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(p));
  return p;
}

// A value that all lanes have, in a uniform register. The loops that issue MMAs and copies count
// to such values and call no function (which would not preserve the registers): their operands
// then stay in uniform registers, instead of being moved there for every instruction (16384
// expert rows 3% slower with loops that the compiler takes for divergent).
__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return __reduce_max_sync(0xffffffffu, v);
}

// Barrier waits by shared address: one poll inline, a wait that lasts out of line (but for the
// warps that issue), bounded as every wait of the library. (try_wait without a time limit: with one it is a loop of its own,
// which took a third of all instructions; sleeping between the polls gained nothing.)
__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// a poll that never suspends
__device__ __forceinline__ uint32_t test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int* status, int where) {
  unsigned long long t0 = 0;
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (poll(bar, parity)) return true;
    if ((i & 15) == 15) {
      const unsigned long long t = global_ns();
      if (!t0) t0 = t;
      if (t - t0 > kSpinNanos) break;
    }
  }
  flag_device_error(status, where);
  return false;
}
// a converged warp, which stays converged
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status, int where) {
  if (__all_sync(0xffffffffu, poll(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_long(bar, parity, status, where));
}
// the same without a call
__device__ __forceinline__ bool wait_inline(uint32_t bar, uint32_t parity, int* status, int where) {
  unsigned long long t0 = 0;
  for (uint32_t i = 1; !__all_sync(0xffffffffu, poll(bar, parity)); ++i) {
    if (i & 255) continue;
    const unsigned long long t = global_ns();
    if (!t0) t0 = t;
    if (__any_sync(0xffffffffu, t - t0 > kSpinNanos || i >= kSpinLimit)) {
      flag_device_error(status, where);
      return false;
    }
  }
  return true;
}
// three barriers, their polls in flight together
__device__ __forceinline__ bool wait_three(uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2,
                                           uint32_t b3, uint32_t p3, int* status, int where) {
  const bool r1 = poll(b1, p1), r2 = poll(b2, p2), r3 = poll(b3, p3);
  if (__all_sync(0xffffffffu, r1 & r2 & r3)) return true;
  return wait_inline(b1, p1, status, where) && wait_inline(b2, p2, status, where + 10) &&
         wait_inline(b3, p3, status, where + 11);
}
// The following act for the threads whose `on` is not 0, by predicate: a branch around them
// costs over a hundred clocks of convergence bookkeeping.
__device__ __forceinline__ void arrive(uint32_t bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar),
      "r"(on)
      : "memory");
}
__device__ __forceinline__ void arrive_tx(uint32_t bar, uint32_t bytes, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes), "r"(on)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          bar),
      "r"(on)
      : "memory");
}
// tile of `map` at (column, row) into shared memory
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int col, int row,
                                          uint32_t bar, uint32_t on) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(bar), "r"(on)
      : "memory");
}
// four MMAs of 16 K values: A from tensor memory, B's descriptor by halves
__device__ __forceinline__ void mma4(uint32_t acc, uint32_t at, uint32_t blo, uint32_t bhi,
                                     uint32_t idesc, uint32_t accumulate, uint32_t on) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 d;\n\tmov.b64 d, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, p;\n\t}" ::"r"(acc),
        "r"(at + s * 8), "r"(blo + s * 2), "r"(bhi), "r"(idesc), "r"(s ? 1u : accumulate), "r"(on)
        : "memory");
}

// Walks this CTA's tiles: expert, row tile, weight tile (fastest).
struct Cursor {
  const int* off;
  int E, tok, n_tiles;
  int e, seg, j;
  Split s;
  int row_begin, row_end;

  __device__ __forceinline__ void set_expert() {
    const int lo = __shfl_sync(0xffffffffu, off[e], 0), hi = __shfl_sync(0xffffffffu, off[e + 1], 0);
    row_begin = lo;
    row_end = hi;
    s = split_rows(hi - lo, tok);
  }
  __device__ __forceinline__ int row0() const { return row_begin + seg * s.per; }
  __device__ __forceinline__ int row1() const { return min(row_end, row0() + s.per); }
  __device__ __forceinline__ void next() {
    if (++j == n_tiles) {
      j = 0;
      if (++seg == s.n) {
        seg = 0;
        do {
          if (++e >= E) return;
          set_expert();
        } while (s.n == 0);
      }
    }
  }
};

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) matmul_tc_kernel(const __grid_constant__ TcArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t bars[kBars];
  __shared__ uint32_t tmem_sh;
  __shared__ int start_sh[3];
  __shared__ long long range_sh[2];
  const MatmulArgs& a = p.a;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* codes = smem + kBBytes;
  uint8_t* scales = codes + kSlots * kSlotBytes;     // two pieces
  int* off = (int*)(scales + 2 * kScaleBytes);       // E + 1 clamped offsets
  // broadcast, so that the compiler knows it for uniform: every branch it takes for divergent
  // costs over a hundred clocks of convergence bookkeeping (measured)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int steps = a.K / 64;  // K steps of one group

  // ---- set-up: barriers, tensor memory, this CTA's range of tiles --------------------------
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAStages; ++i) {
      mbar_init(&bars[kBarA + i], 4);
      mbar_init(&bars[kBarFreed + i], 1);
    }
    for (int i = 0; i < kMaxBStages; ++i) {
      mbar_init(&bars[kBarB + 2 * i], 1);
      mbar_init(&bars[kBarB + 2 * i + 1], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars[kBarC + 2 * i], 1);
      mbar_init(&bars[kBarC + 2 * i + 1], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kBarS + 2 * i], 32);
      mbar_init(&bars[kBarS + 2 * i + 1], 16);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kBarAcc + 2 * i], 1);
      mbar_init(&bars[kBarAcc + 2 * i + 1], 4);
    }
    mbar_init(&bars[kBarFin], 1);
    fence_mbar_init();
  }
  // Tensor memory is taken after the kernel before has ended and before the next one may be set
  // up: neither can hold columns that this one waits for while it waits for this one.
  wait_for_kernel_before();
  if (warp == 0) {
    tc::tmem_alloc(&tmem_sh, 512);
    tc::tmem_relinquish();
  }
  for (int e = threadIdx.x; e <= a.E; e += kThreads)
    off[e] = a.offsets ? min(max(a.offsets[e], 0), a.R) : (e ? a.R : 0);
  __syncthreads();
  if (warp == 3) {
    // the number of tiles, then the first one of this CTA's share
    long long total = 0;
    for (int e = lane; e < a.E; e += 32) {
      const Split s = split_rows(off[e + 1] - off[e], p.tok);
      total += (long long)s.n * p.n_tiles;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const long long lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
    long long base = 0;
    bool found = false;
    for (int e0 = 0; e0 < a.E && !found; e0 += 32) {
      const int e = e0 + lane;
      Split s = {0, 16};
      if (e < a.E) s = split_rows(off[e + 1] - off[e], p.tok);
      const long long mine = (long long)s.n * p.n_tiles;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const long long begin = base + sum - mine;
      const long long first = lo > begin ? lo - begin : 0;  // tile of this expert
      const bool here = first < mine;
      const unsigned m = __ballot_sync(0xffffffffu, here);
      if (m) {
        found = true;
        if (lane == __ffs(m) - 1) {
          start_sh[0] = e;
          start_sh[1] = (int)(first / p.n_tiles);
          start_sh[2] = (int)(first % p.n_tiles);
          range_sh[0] = begin + first;
          range_sh[1] = hi;
        }
      }
      base += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (!found && lane == 0) {
      start_sh[0] = a.E;
      range_sh[0] = range_sh[1] = 0;
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  allow_next_kernel();
  const uint32_t tmem = tmem_sh;
  Cursor cur;
  cur.off = off;
  cur.E = a.E;
  cur.tok = p.tok;
  cur.n_tiles = p.n_tiles;
  cur.e = __shfl_sync(0xffffffffu, start_sh[0], 0);
  cur.seg = __shfl_sync(0xffffffffu, start_sh[1], 0);
  cur.j = __shfl_sync(0xffffffffu, start_sh[2], 0);
  if (cur.e < a.E) cur.set_expert();
  const int n_out = GATED ? a.N / 2 : a.N;
  // weight row of row r of tile j (clamped into the matrix; what is past it is not stored)
  auto weight_row = [&](int e, int j, int r) -> long long {
    const int n = GATED ? min(j * 64 + (r >> 5) * 16 + (r & 15), n_out - 1) + (r >> 4 & 1) * n_out
                        : min(j * 128 + r, n_out - 1);
    return (long long)e * a.N + n;
  };
  // a B stage is two tiles of 64 K values
  const int half_bytes = stage_rows(p.tok) * 128;
  // full barrier of B stage i at bar_b + 16 i, its free barrier 8 bytes on; the others alike.
  // A double step (128 K values) has a turn, 0 or 1 in alternation from every tile's first: two
  // A stages (one per half; full barriers by stage, freed barriers by turn), two warpgroups and
  // two stages of codes, which count the double steps of their turn.
  const uint32_t bar_a = smem_u32(bars), bar_freed = bar_a + 8 * kBarFreed, bar_b = bar_a + 8 * kBarB, bar_c = bar_a + 8 * kBarC;
  const uint32_t bar_s = bar_a + 8 * kBarS, bar_acc = bar_a + 8 * kBarAcc, bar_fin = bar_a + 8 * kBarFin;
  const uint32_t one = elect_one();
  const uint32_t mine = uniform((uint32_t)(range_sh[1] - range_sh[0]));  // tiles of this CTA
  bool ok = true;

  if (warp >= 4 && warp < 20) {
    // ------------------------------------------------------------------ dequantizers
    // half h of the double steps of a turn; tensor memory lanes 32q..32q+31
    const int h = (warp >> 2) - 1 & 1, turn = (warp >> 2) - 1 >> 1, q = warp & 3;
    const uint32_t my_row = smem_u32(codes) + turn * 2 * kSlotBytes + (q * 32 + lane) * 64;
    const uint32_t at0 = my_row + (((2 * h) ^ (lane >> 1 & 3)) << 4);
    const uint32_t at1 = my_row + (((2 * h + 1) ^ (lane >> 1 & 3)) << 4);
    const uint32_t my_scales =
        smem_u32(scales) + (q * 32 + lane) * kScalePitch + (2 * turn + h) * 2;
    const uint32_t my_a = tmem + kACol + turn * 64 + h * 32 + ((uint32_t)(q * 32) << 16);
    const uint32_t my_full = bar_a + 8 * (turn * 2 + h), my_freed = bar_freed + 8 * turn;
    const uint32_t my_codes = bar_c + 32 * turn;
    uint32_t n = 0, piece = 0;  // double steps of this turn, pieces of scales so far
    for (uint32_t tile = 0; tile < mine && ok; ++tile) {
      for (int k0 = 0; k0 < steps; k0 += kScaleGroups, ++piece) {
        const uint32_t s_bar = bar_s + 16 * (piece & 1);
        uint32_t sat = my_scales + (piece & 1) * kScaleBytes;
        ok = wait_warp(s_bar, piece >> 1 & 1, a.status, 71);
        if (!ok) break;
#pragma unroll 1
        for (int k = k0 + 2 * turn; k < min(k0 + kScaleGroups, steps); k += 4, ++n, sat += 8) {
          // (half 1 of an odd last step converts what is not multiplied, to keep the count)
          const uint32_t slot = n & 1;
          ok = wait_warp(my_codes + 16 * slot, n >> 1 & 1, a.status, 67);
          if (!ok) break;
          const uint32_t s2 = lds_u16x2(sat), b2 = lds_u16x2(sat + 128 * kScalePitch);
          uint32_t out[32], wv[8];
          lds_v4(at0 + slot * kSlotBytes, wv);
          lds_v4(at1 + slot * kSlotBytes, wv + 4);
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            // byte c of a word holds codes 2c and 2c + 1: its low nibble and, from the word
            // shifted by four, its high one go to the two halves
            const uint32_t up = wv[w] >> 4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t pair = prmt(wv[w], up, 0x0400u + 0x0101u * c);
              out[4 * w + c] =
                  Conv<T>::fma(Conv<T>::sub(and_or(pair, 0x000f000fu, Conv<T>::kMagic)), s2, b2);
            }
          }
          // converted before the stage is free, so that it is stored at once
          ok = wait_warp(my_freed, (n & 1) ^ 1, a.status, 60);
          if (!ok) break;
          tc::fence_after_sync();
          tc::st32(my_a, out);
          tc::wait_st();
          tc::fence_before_sync();
          __syncwarp();
          // the codes are freed after their last use, not after their loads: a load that the
          // assembler moved below the arrive would read the stage's next contents
          arrive(my_full, one);
          arrive(my_codes + 16 * slot + 8, one);
        }
        if (!ok) break;
        __syncwarp();
        arrive(s_bar + 8, one);
      }
    }
  } else if (warp >= 20) {
    // ------------------------------------------------------------------ results
    const int q = warp & 3;
    T* out = (T*)a.out;
    for (uint32_t tile = 0; tile < mine; ++tile) {
      const int buf = tile & 1;
      ok = wait_warp(bar_acc + 16 * buf, (tile >> 1) & 1, a.status, 61);
      if (!ok) break;
      tc::fence_after_sync();
      const int row0 = cur.row0(), rows = cur.row1() - row0;
      const int n = GATED ? cur.j * 64 + q * 16 + (lane & 15) : cur.j * 128 + q * 32 + lane;
      const uint32_t acc = tmem + buf * kMaxTok + ((uint32_t)(q * 32) << 16);
      T* o = out + (long long)row0 * n_out + n;
      for (int c0 = 0; c0 < rows; c0 += 16) {
        uint32_t r[16];
        tc::ld16(acc + c0, r);
        tc::wait_ld();
        const bool full = c0 + 16 <= rows;
        if (GATED) {
          const bool hi = lane >= 16;  // lanes 0-15 finish column c, lanes 16-31 column c + 1
          T* oc = o + (long long)(c0 + (hi ? 1 : 0)) * n_out;
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, hi ? r[c] : r[c + 1], 16);
            const float gate = __uint_as_float(hi ? other : r[c]);
            const float up = __uint_as_float(hi ? r[c + 1] : other);
            // (a denominator of at most 2: __fdividef gives 0 for one past 2^126, a gate below
            // -87.3, and a divide that rounds right calls a function, 176 against 144.5 us)
            const float e = expf(-fabsf(gate));
            const T v = Elem<T>::from_f32(gate * __fdividef(gate < 0.f ? e : 1.f, 1.f + e) * up);
            if (n < n_out && (full || c0 + c + (hi ? 1 : 0) < rows)) oc[0] = v;
            oc += 2 * n_out;
          }
        } else {
          T* oc = o + (long long)c0 * n_out;
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const T v = Elem<T>::from_f32(__uint_as_float(r[c]));
            if (n < n_out && (full || c0 + c < rows)) oc[0] = v;
            oc += n_out;
          }
        }
      }
      tc::fence_before_sync();
      __syncwarp();
      arrive(bar_acc + 16 * buf + 8, one);
      cur.next();
    }
  } else if (warp == 3) {
    // ------------------------------------------------------------------ scales and biases
    // A dequantizer lane reading its own row from global memory would cost the load pipe a
    // lookup per lane and stall its warp (34 clocks per load, measured), so this warp stages
    // pieces of 16 groups of the tile's 128 rows.
    const uint32_t base = smem_u32(scales);
    const uintptr_t bits = (uintptr_t)a.scales | (uintptr_t)a.biases;
    const bool wide = steps % 8 == 0 && bits % 16 == 0, pairs = steps % 2 == 0 && bits % 4 == 0;
    uint32_t buf = 0, ph = 1;
    for (uint32_t tile = 0; tile < mine && ok; ++tile) {
      for (int g0 = 0; g0 < steps; g0 += kScaleGroups) {
        ok = wait_warp(bar_s + 16 * buf + 8, ph, a.status, 72);
        if (!ok) break;
        const uint32_t dst = base + buf * kScaleBytes;
        const uint16_t* const arrays[2] = {(const uint16_t*)a.scales, (const uint16_t*)a.biases};
        if (wide) {
          const int g = g0 + (lane & 1) * 8;
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            const int r = (lane >> 1) + 16 * i;
            const long long at = weight_row(cur.e, cur.j, r) * steps + g;
            if (g < steps) {
              cp16(dst + r * kScalePitch + (lane & 1) * 16, arrays[0] + at);
              cp16(dst + (128 + r) * kScalePitch + (lane & 1) * 16, arrays[1] + at);
            }
          }
        } else if (pairs) {
          const int g = g0 + (lane & 7) * 2;
#pragma unroll 8
          for (int i = 0; i < 32; ++i) {
            const int r = (lane >> 3) + 4 * i;
            const long long at = weight_row(cur.e, cur.j, r) * steps + g;
            if (g < steps) {
              cp4(dst + r * kScalePitch + (lane & 7) * 4, arrays[0] + at);
              cp4(dst + (128 + r) * kScalePitch + (lane & 7) * 4, arrays[1] + at);
            }
          }
        } else {
          const int g = min(g0 + (lane & 15), steps - 1);
#pragma unroll 1
          for (int i0 = 0; i0 < 64; i0 += 16) {
            uint16_t v[2][16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const long long at = weight_row(cur.e, cur.j, (lane >> 4) + 2 * (i0 + i)) * steps + g;
              v[0][i] = __ldg(arrays[0] + at);
              v[1][i] = __ldg(arrays[1] + at);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t to = dst + ((lane >> 4) + 2 * (i0 + i)) * kScalePitch + (lane & 15) * 2;
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(to), "h"(v[0][i]) : "memory");
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + 128 * kScalePitch), "h"(v[1][i])
                           : "memory");
            }
          }
        }
        if (wide || pairs)  // when the copies have landed
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar_s + 16 * buf)
                       : "memory");
        else
          arrive(bar_s + 16 * buf, 1);
        buf ^= 1;
        ph ^= buf ^ 1;
      }
      cur.next();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 1) {
    // ------------------------------------------------------------------ rows of x, in order
    const uint32_t base = smem_u32(smem);
    int st = 0, issued = 0;
    uint32_t ph = 1;
    for (uint32_t tile = 0; tile < mine && ok; ++tile) {
      // (What lies past the tile's rows is multiplied, and not stored, or not even that. With
      // `tok` rows for every tile the L2 traffic was 1.8 times as much at 106 rows a tile; with
      // several boxes of 32 rows for each tile this warp was too slow, 163 against 147 us.)
      const int row0 = uniform(cur.row0());
      const int boxes = uniform((cur.row1() - row0 + kBoxRows - 1) / kBoxRows);
      const CUtensorMap* map = &p.x[boxes - 1];
      for (int k = 0; k < steps; k += 2) {
        ok = wait_inline(bar_b + 16 * st + 8, ph, a.status, 62);
        if (!ok) break;
        const uint32_t dst = base + st * 2 * half_bytes, bar = bar_b + 16 * st;
        const bool both = k + 1 < steps;
        arrive_tx(bar, (both ? 2 : 1) * boxes * kBoxRows * 128, one);
        load_tile(dst, map, k * 64, row0, bar, one);
        if (both) load_tile(dst + half_bytes, map, k * 64 + 64, row0, bar, one);
        ++issued;
        if (++st == p.b_stages) {
          st = 0;
          ph ^= 1;
        }
      }
      cur.next();
    }
    // no copy is in flight when the CTA exits, not even after a wait that gave up
    for (int i = min(issued, p.b_stages); i > 0; --i) {
      st = st ? st - 1 : p.b_stages - 1;
      if (st == p.b_stages - 1) ph ^= 1;
      wait_inline(bar_b + 16 * st, ph ^ 1, a.status, 68);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ packed codes
    const uint32_t base = smem_u32(codes);
    uint32_t n[2] = {0, 0};  // double steps of either turn so far
    for (uint32_t tile = 0; tile < mine && ok; ++tile) {
      const int row = uniform(cur.e * a.N + cur.j * (GATED ? 64 : 128));
      for (int k = 0; k < steps && ok; k += 4) {
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
          const int kk = k + 2 * turn;
          if (kk < steps && ok) {
            const uint32_t slot = turn * 2 + (n[turn] & 1);
            const uint32_t dst = base + slot * kSlotBytes, bar = bar_c + 16 * slot;
            ok = wait_inline(bar + 8, (n[turn] >> 1 & 1) ^ 1, a.status, 69);
            if (ok) {
              arrive_tx(bar, kSlotBytes, one);
              if (GATED) {
#pragma unroll
                for (int i = 0; i < 8; ++i)  // 16 gate rows, their 16 up rows, per quarter
                  load_tile(dst + i * 1024, &p.codes, kk * 32,
                            row + (i >> 1) * 16 + (i & 1) * n_out, bar, one);
              } else {
                load_tile(dst, &p.codes, kk * 32, row, bar, one);
              }
              ++n[turn];
            }
          }
        }
      }
      cur.next();
    }
#pragma unroll
    for (int turn = 0; turn < 2; ++turn)
      for (uint32_t i = n[turn] < 2 ? 0 : n[turn] - 2; i < n[turn]; ++i)
        wait_inline(bar_c + 16 * (turn * 2 + (i & 1)), i >> 1 & 1, a.status, 70);
  } else if (warp == 0) {
    // ------------------------------------------------------------------ MMA issuer
    // As few instructions as it takes: an MMA or a commit takes its thread 44 clocks.
    constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
    const uint64_t desc = tc::sdesc_sw128(smem_u32(smem), 16, 1024);
    const uint32_t dlo = (uint32_t)desc, dhi = (uint32_t)(desc >> 32);
    const uint32_t dhalf = (uint32_t)half_bytes >> 4;  // descriptor units of 16 bytes
    const uint32_t bb_end = bar_b + 16 * p.b_stages;
    constexpr uint32_t tm = 0;  // all 512 columns are taken, so they begin at 0
    uint32_t bb = bar_b, blo = dlo;  // full barrier and descriptor of the B stage
    uint32_t bph = 0, aph = 0;  // bit t of aph: phase of turn t
    uint32_t ready = 0;  // the next double step's barriers, tested while this one's MMAs run
    for (uint32_t tile = 0; tile < mine && ok; ++tile) {
      const int rows = uniform(cur.row1() - cur.row0());
      const uint32_t idesc = tc::idesc_f16(kBf, 128, 0, false, false) +
                             ((uint32_t)((rows + 15) / 16 * 2) << 17);
      const uint32_t buf = tile & 1, acc = tm + buf * kMaxTok;
      ok = wait_inline(bar_acc + 16 * buf + 8, (tile >> 1 & 1) ^ 1, a.status, 63);
      uint32_t turn = 0;
      for (int k = 0; k < steps && ok; k += 2) {
        const uint32_t ba = bar_a + 16 * turn, ph = aph >> turn & 1;
        if (!__all_sync(0xffffffffu, ready)) ok = wait_three(bb, bph, ba, ph, ba + 8, ph, a.status, 64);
        if (!ok) break;
        tc::fence_after_sync();
        const bool last = k + 2 >= steps;
        const uint32_t am = tm + kACol + turn * 64, b_free = bb + 8, b_at = blo;
        const uint32_t freed = bar_freed + 8 * turn;
        aph ^= 1u << turn;
        turn = last ? 0 : turn ^ 1;
        bb += 16;
        blo += 2 * dhalf;
        if (bb == bb_end) {
          bb = bar_b;
          blo = dlo;
          bph ^= 1;
        }
        const uint32_t na = bar_a + 16 * turn, nph = aph >> turn & 1;
        mma4(acc, am, b_at, dhi, idesc, k > 0 ? 1u : 0u, one);
        if (k + 1 < steps) mma4(acc, am + 32, b_at + dhalf, dhi, idesc, 1u, one);
        // by now the stages freed by the double step before have been refilled
        ready = test(bb, bph) & test(na, nph) & test(na + 8, nph);
        commit(freed, one);
        commit(b_free, one);
        if (last) commit(bar_acc + 16 * buf, one);
      }
      cur.next();
    }
    // every MMA has completed before tensor memory is freed (one lane, the same each time,
    // issued them all)
    commit(bar_fin, one);
    wait_inline(bar_fin, 0, a.status, 66);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

// The rows of x that `rows` names, one after the other; a bad index gives a row of zeros. The
// product kernel could gather by itself, but four-row TMA loads and 16-byte cp.async both
// brought 32 bytes a clock and SM where its MMAs take 64 (16384 rows of 2048 through 128 experts
// of 1536x2048: 185 us with gathering inside; 13 us for this kernel, which writes 67 MB,
// and 128 for the product).
__global__ void __launch_bounds__(256)
    gather_rows_kernel(const uint4* __restrict__ x, long long ldx, int x_rows,
                       const int* __restrict__ rows, uint4* __restrict__ out, int R, int per_row) {
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  wait_for_previous();
  if (r >= R) return;
  const int from = rows[r];
  const bool in = from >= 0 && from < x_rows;
  const uint4* src = x + (in ? from : 0) * ldx;
  uint4* dst = out + (long long)r * per_row;
  for (int c = threadIdx.x & 31; c < per_row; c += 32)
    dst[c] = in ? src[c] : make_uint4(0, 0, 0, 0);
}

size_t smem_bytes(int E) {
  return 1024 + kBBytes + kSlots * kSlotBytes + 2 * kScaleBytes + (size_t)(E + 1) * sizeof(int);
}

template <typename T, bool GATED>
int launch_tc_t(TcArgs& p, int grid, cudaStream_t st) {
  const size_t smem = smem_bytes(p.a.E);
  static std::atomic<unsigned long long> ready{0};  // devices whose shared memory bound is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return QKV_ECUDA;
  if (dev < 0 || dev >= kMaxDevices || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(matmul_tc_kernel<T, GATED>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_bytes(kMaxExperts)) != cudaSuccess)
      return QKV_ECUDA;
    if (dev >= 0 && dev < kMaxDevices) ready.fetch_or(1ull << dev);
  }
  if (!make_rows_map(&p.codes, p.a.w, 1, p.a.K / 2, (long long)p.a.E * p.a.N, p.a.K / 2, 64,
                     GATED ? 16 : 128))
    return QKV_ECUDA;
  for (int i = 0; i < stage_rows(p.tok) / kBoxRows; ++i)
    if (!make_rows_map(&p.x[i], p.a.x, 2, p.a.K, p.a.x_rows, p.a.ldx * 2, 64, (i + 1) * kBoxRows))
      return QKV_ECUDA;
  return launch(!p.gathered, matmul_tc_kernel<T, GATED>, dim3(grid), kThreads, smem, st, p);
}

}  // namespace

size_t matmul_tc_workspace(int R, int K) { return (size_t)R * K * 2; }

bool matmul_tc_fits(int E, int N) {
  return E <= kMaxExperts && (long long)E * N < (1ll << 31) - 256;  // 32-bit TMA coordinates
}

int launch_matmul_tc(const MatmulArgs& a, cudaStream_t st) {
  const bool gated = a.act == QKV_ACT_SWIGLU;
  const int n_out = gated ? a.N / 2 : a.N;
  const int sms = num_sms();
  TcArgs p;
  p.a = a;
  p.gathered = a.rows != nullptr;
  if (a.rows) {
    const int rc = launch(true, gather_rows_kernel, dim3((a.R + 7) / 8), 256, 0, st, a.x,
                                    a.ldx / 8, a.x_rows, a.rows, a.workspace, a.R, a.K / 8);
    if (rc) return rc;
    p.a.x = a.workspace;
    p.a.ldx = a.K;
    p.a.x_rows = a.R;
    p.a.rows = nullptr;
  }
  p.n_tiles = gated ? (n_out + 63) / 64 : (n_out + 127) / 128;
  // One matrix: the largest row tile, or a smaller one if that takes fewer rounds of tiles.
  // Experts: the counts are on the device, so the largest.
  p.tok = kMaxTok;
  if (!a.offsets) {
    long long best = -1;
    for (int tok = kMaxTok; tok >= 64; tok -= 16) {
      const Split s = split_rows(a.R, tok);
      const long long rounds = ((long long)s.n * p.n_tiles + sms - 1) / sms;
      if (best < 0 || rounds < best) {
        best = rounds;
        p.tok = tok;
      }
    }
  }
  const int most = std::min(a.R, p.tok);
  p.tok = (most + 15) / 16 * 16;
  p.b_stages = std::min(kMaxBStages, kBBytes / (stage_rows(p.tok) * 256));
  long long tiles = (long long)((a.R + p.tok - 1) / p.tok + (a.offsets ? std::min(a.E, a.R) : 0)) * p.n_tiles;
  const int grid = (int)std::min<long long>(tiles, sms);
  if (a.dtype == QKV_BF16)
    return gated ? launch_tc_t<__nv_bfloat16, true>(p, grid, st)
                 : launch_tc_t<__nv_bfloat16, false>(p, grid, st);
  return gated ? launch_tc_t<__half, true>(p, grid, st) : launch_tc_t<__half, false>(p, grid, st);
}

}  // namespace qkv
