// Products of many rows with affine 4-bit weights on the 5th-generation tensor cores
// (sm_100a): y = x W^T for one weight matrix, or one per expert over rows sorted by expert.
//
// Roles swapped so that ragged row counts cost what they are: the MMA's 128 M rows are weight
// rows and its N columns are rows of x, any multiple of 16 up to 192, so an expert with 40
// rows pays for 48. Weights become the A operand in TENSOR memory: a dequantizer thread owns
// one weight row, turns a group of 64 codes into 16-bit values in registers and stores them
// to its lane, so dequantized weights touch neither HBM nor shared memory. Rows of x are the
// B operand in shared memory, gathered row by row with cp.async (128-byte swizzle).
//
//   * Persistent CTAs, one per SM. A tile is (expert, up to 192 of its rows, 128 weight rows);
//     an expert's rows are cut into equal tiles. Every CTA takes a contiguous range of the
//     tiles of equal summed cost, computed by each CTA from the offsets: nothing is counted
//     through memory, and neighbouring tiles share rows of x in L2.
//   * Warps: 0 issues the MMAs, 1 loads rows of x (TMA), 2 packed codes (TMA), 4-11
//     dequantize (two warpgroups, alternate 128 K values), 12-15 store results; 1, 3 and 16-19
//     gather rows of x (TMA, four rows a load).
//   * Tensor memory: two accumulators of 192 columns (a tile's results are stored while the
//     next one accumulates) and four A stages of 32 columns (64 K values each).
//   * Gated activation: 16 gate rows and the 16 up rows of the same outputs share a warp's 32
//     lanes, so the epilogue exchanges them with one shuffle per two values.
//
// Rounding: a weight is rounded once to x's type, round(scale * code + bias) by a fused
// multiply-add, the value mx.dequantize gives; sums are fp32.
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

constexpr int kWarps = 20;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxTok = 192;           // rows of x in a tile
constexpr int kAStages = 2;            // of 128 K values, in tensor memory
constexpr int kACols = 64;             // columns of an A stage
constexpr int kACol = 2 * kMaxTok;     // first A column
constexpr int kMaxBStages = 8;         // of 128 K values
constexpr int kBBytes = 144 * 1024;    // shared memory of the B stages
constexpr int kSlots = 4;              // prefetched spans of packed codes
constexpr int kSlotBytes = 128 * 128;  // 128 weight rows x 128 bytes: 256 K values
// barriers, in shared memory: pairs of full and free by stage
constexpr int kBarA = 0, kBarB = kBarA + 2 * kAStages, kBarC = kBarB + 2 * kMaxBStages;
constexpr int kBarAcc = kBarC + 2 * kSlots, kBarFin = kBarAcc + 4, kBars = kBarFin + 1;
constexpr int kGatherWarps = 6;        // warps 1, 3 and 16-19
constexpr int kMaxExperts = 1024;

struct TcArgs {
  CUtensorMap codes;  // (E * N, K/2) bytes; boxes of 128 rows, or of 16 gate or up rows
  CUtensorMap x;      // (x_rows, K); boxes of `tok` rows, or single rows for gathering
  MatmulArgs a;
  int tok;       // most rows of x per tile (a multiple of 16)
  int b_stages;
  int n_tiles;   // tiles of 128 weight rows
};

// Cost of a tile in units of 16 rows' MMAs: below kMinCost the dequantizers set the pace.
constexpr int kMinCost = 6;
constexpr int kFixCost = 1;

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
__host__ __device__ inline int tile_cost(int per) {
  const int c = per / 16;
  return (c > kMinCost ? c : kMinCost) + kFixCost;
}

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

// tile of `map` at (column, row) into shared memory
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int col, int row,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(bar)
      : "memory");
}
// Scale loads, volatile so that they stay ahead of the span they are loaded under.
__device__ __forceinline__ uint32_t ld_u16(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_u32(const uint16_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ void ld_v4(const uint16_t* p, uint32_t (&v)[4]) {
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "l"(p));
}
__device__ __forceinline__ bool bad_row(const MatmulArgs& a, int r) {
  const int i = __ldg(a.rows + r);
  return i < 0 || i >= a.x_rows;
}
// four rows of `map` (any indices inside it) at a column
__device__ __forceinline__ void load_rows4(uint32_t dst, const CUtensorMap* map, int col,
                                           const int4& r, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w),
      "r"(bar)
      : "memory");
}
// one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(p));
  return p != 0;
}

// Barrier waits by shared address: one poll inline; a wait that lasts suspends in hardware
// until the phase flips (polling would take issue slots from the dequantizers), bounded as
// every wait of the library.
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
__device__ __noinline__ bool wait_long(uint32_t bar, uint32_t parity, int* status, int where) {
  unsigned long long t0 = 0;
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(100000u)
        : "memory");
    if (ok) return true;
    if (i >= 4) {
      const unsigned long long t = global_ns();
      if (!t0) t0 = t;
      if (t - t0 > kSpinNanos) break;
    }
  }
  flag_device_error(status, where);
  return false;
}
// one thread
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, int* status, int where) {
  return poll(bar, parity) || wait_long(bar, parity, status, where);
}
// a converged warp, which stays converged
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, int* status, int where) {
  if (__all_sync(0xffffffffu, poll(bar, parity))) return true;
  return __all_sync(0xffffffffu, wait_long(bar, parity, status, where));
}
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void arrive_tx(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(
          bar),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}
// four MMAs of 16 K values: A from tensor memory, B's descriptor by halves
__device__ __forceinline__ void mma4(uint32_t acc, uint32_t at, uint32_t blo, uint32_t bhi,
                                     uint32_t idesc, uint32_t accumulate) {
#pragma unroll
  for (int s = 0; s < 4; ++s)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 d;\n\tmov.b64 d, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], d, %4, p;\n\t}" ::"r"(acc),
        "r"(at + s * 8), "r"(blo + s * 2), "r"(bhi), "r"(idesc), "r"(s ? 1u : accumulate)
        : "memory");
}

// Walks this CTA's tiles: expert, row tile, weight tile (fastest).
struct Cursor {
  const int* off;
  int E, tok, n_tiles;
  long long pos, end;
  int e, seg, j;
  Split s;
  int cost, row_begin, row_end;

  __device__ __forceinline__ void set_expert() {
    const int lo = off[e], hi = off[e + 1];
    row_begin = lo;
    row_end = hi;
    s = split_rows(hi - lo, tok);
    cost = tile_cost(s.per);
  }
  __device__ __forceinline__ bool valid() const { return e < E && pos < end; }
  __device__ __forceinline__ int row0() const { return row_begin + seg * s.per; }
  __device__ __forceinline__ int row1() const { return min(row_end, row0() + s.per); }
  __device__ __forceinline__ void next() {
    pos += cost;
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

// SB: how scales are read (0 singly, 1 in pairs, 2 eight at a time)
template <typename T, bool GATED, int SB>
__global__ void __launch_bounds__(kThreads, 1) matmul_tc_kernel(const __grid_constant__ TcArgs p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ uint64_t bars[kBars];
  __shared__ uint32_t tmem_sh;
  __shared__ int start_sh[3];
  __shared__ long long range_sh[2];
  const MatmulArgs& a = p.a;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* codes = smem + kBBytes;
  int* off = (int*)(codes + kSlots * kSlotBytes);  // E + 1 clamped offsets
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int steps = a.K / 64;  // K steps of one group

  // ---- set-up: barriers, tensor memory, this CTA's range of tiles --------------------------
  if (threadIdx.x == 0) {
    for (int i = 0; i < kAStages; ++i) {
      mbar_init(&bars[kBarA + 2 * i], 4);
      mbar_init(&bars[kBarA + 2 * i + 1], 1);
    }
    for (int i = 0; i < kMaxBStages; ++i) {
      mbar_init(&bars[kBarB + 2 * i], a.rows ? kGatherWarps : 1);
      mbar_init(&bars[kBarB + 2 * i + 1], 1);
    }
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars[kBarC + 2 * i], 1);
      mbar_init(&bars[kBarC + 2 * i + 1], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[kBarAcc + 2 * i], 1);
      mbar_init(&bars[kBarAcc + 2 * i + 1], 4);
    }
    mbar_init(&bars[kBarFin], 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tc::tmem_alloc(&tmem_sh, 512);
    tc::tmem_relinquish();
  }
  for (int e = threadIdx.x; e <= a.E; e += kThreads)
    off[e] = a.offsets ? min(max(a.offsets[e], 0), a.R) : (e ? a.R : 0);
  __syncthreads();
  if (warp == 3) {
    // total cost, then the first tile that starts inside this CTA's share
    long long total = 0;
    for (int e = lane; e < a.E; e += 32) {
      const Split s = split_rows(off[e + 1] - off[e], p.tok);
      total += (long long)s.n * p.n_tiles * tile_cost(s.per);
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
      const int c = tile_cost(s.per);
      const long long mine = (long long)s.n * p.n_tiles * c;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const long long begin = base + sum - mine;
      // index of the first tile of this expert starting at or after lo
      const long long first = lo > begin ? (lo - begin + c - 1) / c : 0;
      const bool here = first < (long long)s.n * p.n_tiles;
      const unsigned m = __ballot_sync(0xffffffffu, here);
      if (m) {
        found = true;
        if (lane == __ffs(m) - 1) {
          start_sh[0] = e;
          start_sh[1] = (int)(first / p.n_tiles);
          start_sh[2] = (int)(first % p.n_tiles);
          range_sh[0] = begin + first * c;
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
  const uint32_t tmem = tmem_sh;
  Cursor cur;
  cur.off = off;
  cur.E = a.E;
  cur.tok = p.tok;
  cur.n_tiles = p.n_tiles;
  cur.e = start_sh[0];
  cur.seg = start_sh[1];
  cur.j = start_sh[2];
  cur.pos = range_sh[0];
  cur.end = range_sh[1];
  if (cur.e < a.E) cur.set_expert();
  const int n_out = GATED ? a.N / 2 : a.N;
  const int half_bytes = p.tok * 128;  // a B stage is two tiles of 64 K values
  // full barrier of A stage i at bar_a + 16 i, its free barrier 8 bytes on; the others alike
  const uint32_t bar_a = smem_u32(bars), bar_b = bar_a + 8 * kBarB, bar_c = bar_a + 8 * kBarC;
  const uint32_t bar_acc = bar_a + 8 * kBarAcc, bar_fin = bar_a + 8 * kBarFin;
  bool ok = true;

  if (warp >= 4 && warp < 12) {
    // ------------------------------------------------------------------ dequantizers
    const int par = (warp >> 2) - 1, q = warp & 3;  // double step of a span; tensor memory lanes 32q..32q+31
    const int spans = (steps + 3) / 4;
    const uint32_t my_row = smem_u32(codes) + (q * 32 + lane) * 128;
    int slot = 0;
    uint32_t ph = 0;
    uint32_t gs = 0;  // double steps of all tiles so far: A stage gs % 2
    while (cur.valid() && ok) {
      // weight row of this lane (clamped into the matrix; what is past it is not stored)
      const int wn = GATED ? min(cur.j * 64 + q * 16 + (lane & 15), n_out - 1) + (lane >> 4) * n_out
                           : min(cur.j * 128 + q * 32 + lane, n_out - 1);
      const long long wr = (long long)cur.e * a.N + wn;
      const uint16_t* sp = (const uint16_t*)a.scales + wr * steps;
      const uint16_t* bp = (const uint16_t*)a.biases + wr * steps;
      // scales and biases: pairs for this warpgroup's two K steps of a span, loaded a span (or
      // two, sixteen bytes at a time) ahead; a lane reads its own row, so wide loads save L1
      uint32_t cs[4], cb[4], ns[4], nb[4];
      auto load_sb = [&](int span) {
        const int k = span * 4;
        if (SB == 2) {
          if (k < steps) {
            ld_v4(sp + k, ns);
            ld_v4(bp + k, nb);
          }
        } else if (SB == 1) {
          if (k + 2 * par < steps) {
            ns[0] = ld_u32(sp + k + 2 * par);
            nb[0] = ld_u32(bp + k + 2 * par);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int kk = min(k + 2 * par + h, steps - 1);
            ns[h] = ld_u16(sp + kk);
            nb[h] = ld_u16(bp + kk);
          }
        }
      };
      load_sb(0);
      for (int span = 0; span < spans && ok; ++span) {
        uint32_t s2[2], b2[2];  // scale and bias of each step in both halves
        if (SB == 2) {
          if (!(span & 1)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              cs[i] = ns[i];
              cb[i] = nb[i];
            }
            load_sb(span + 2);
          }
          const uint32_t sw = span & 1 ? (par ? cs[3] : cs[2]) : (par ? cs[1] : cs[0]);
          const uint32_t bw = span & 1 ? (par ? cb[3] : cb[2]) : (par ? cb[1] : cb[0]);
          s2[0] = prmt(sw, sw, 0x1010), s2[1] = prmt(sw, sw, 0x3232);
          b2[0] = prmt(bw, bw, 0x1010), b2[1] = prmt(bw, bw, 0x3232);
        } else if (SB == 1) {
          s2[0] = prmt(ns[0], ns[0], 0x1010), s2[1] = prmt(ns[0], ns[0], 0x3232);
          b2[0] = prmt(nb[0], nb[0], 0x1010), b2[1] = prmt(nb[0], nb[0], 0x3232);
          if (span + 1 < spans) load_sb(span + 1);
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s2[h] = prmt(ns[h], ns[h], 0x1010);
            b2[h] = prmt(nb[h], nb[h], 0x1010);
          }
          if (span + 1 < spans) load_sb(span + 1);
        }
        ok = wait_warp(bar_c + 16 * slot, ph, a.status, 67);
        if (!ok) break;
        const int k0 = span * 4 + 2 * par;  // this warpgroup's steps k0 and k0 + 1
        if (k0 < steps) {
          const uint32_t g = gs + span * 2 + par, st = g % kAStages;
          const uint32_t dst = tmem + kACol + st * kACols + ((uint32_t)(q * 32) << 16);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t out[32];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t wv[4];
              const uint32_t at = my_row + slot * kSlotBytes +
                                  (((4 * par + 2 * h + i) ^ (lane & 7)) << 4);
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(wv[0]), "=r"(wv[1]), "=r"(wv[2]), "=r"(wv[3])
                           : "r"(at)
                           : "memory");
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint32_t v[4];
#pragma unroll
                for (int c = 0; c < 4; ++c)
                  v[c] = Conv<T>::fma(
                      Conv<T>::sub(and_or(wv[w] >> (4 * c), 0x000f000fu, Conv<T>::kMagic)), s2[h],
                      b2[h]);
                // (0,4)(1,5)(2,6)(3,7) -> (0,1)(2,3)(4,5)(6,7)
                out[16 * i + 4 * w + 0] = prmt(v[0], v[1], 0x5410);
                out[16 * i + 4 * w + 1] = prmt(v[2], v[3], 0x5410);
                out[16 * i + 4 * w + 2] = prmt(v[0], v[1], 0x7632);
                out[16 * i + 4 * w + 3] = prmt(v[2], v[3], 0x7632);
              }
            }
            // the first half is converted before the stage is free
            if (h == 0) {
              ok = wait_warp(bar_a + 16 * st + 8, ((g / kAStages) & 1) ^ 1, a.status, 60);
              if (!ok) break;
              tc::fence_after_sync();
            }
            // (the second half of an odd last step holds zeros that no MMA reads)
            tc::st32(dst + h * 32, out);
          }
          if (!ok) break;
          tc::wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) arrive(bar_a + 16 * st);
        }
        // after the last use of the words, not after their loads: a load that the assembler
        // moved below this arrive would read the slot's next contents
        __syncwarp();
        if (lane == 0) arrive(bar_c + 16 * slot + 8);
        if (++slot == kSlots) {
          slot = 0;
          ph ^= 1;
        }
      }
      gs += (steps + 1) / 2;
      cur.next();
    }
  } else if (warp >= 12 && warp < 16) {
    // ------------------------------------------------------------------ results
    const int q = warp & 3;
    int tile = 0;
    T* out = (T*)a.out;
    while (cur.valid()) {
      const int buf = tile & 1;
      ok = wait_warp(bar_acc + 16 * buf, (tile >> 1) & 1, a.status, 61);
      if (!ok) break;
      tc::fence_after_sync();
      const int row0 = cur.row0(), rows = cur.row1() - row0;
      const int n = GATED ? cur.j * 64 + q * 16 + (lane & 15) : cur.j * 128 + q * 32 + lane;
      const uint32_t acc = tmem + buf * kMaxTok + ((uint32_t)(q * 32) << 16);
      T* o = out + (long long)row0 * n_out + n;
      bool bad = false;  // whether a row of the tile has an index outside x
      if (a.rows)
        for (int t = lane; t < rows; t += 32) bad |= bad_row(a, row0 + t);
      bad = __any_sync(0xffffffffu, bad);
      for (int c0 = 0; c0 < rows; c0 += 16) {
        uint32_t r[16];
        tc::ld16(acc + c0, r);
        tc::wait_ld();
        if (bad) {
#pragma unroll
          for (int c = 0; c < 16; ++c)
            if (c0 + c < rows && bad_row(a, row0 + c0 + c)) r[c] = 0;
        }
        const bool full = c0 + 16 <= rows;
        if (GATED) {
          const bool hi = lane >= 16;  // lanes 0-15 finish column c, lanes 16-31 column c + 1
          T* oc = o + (long long)(c0 + (hi ? 1 : 0)) * n_out;
#pragma unroll
          for (int c = 0; c < 16; c += 2) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, hi ? r[c] : r[c + 1], 16);
            const float gate = __uint_as_float(hi ? other : r[c]);
            const float up = __uint_as_float(hi ? r[c + 1] : other);
            const T v = Elem<T>::from_f32(__fdividef(gate, 1.f + __expf(-gate)) * up);
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
      if (lane == 0) arrive(bar_acc + 16 * buf + 8);
      ++tile;
      cur.next();
    }
  } else if (warp == 1 && !a.rows) {
    // ------------------------------------------------------------------ rows of x, in order
    if (lane == 0) {
      const uint32_t base = smem_u32(smem);
      int st = 0, issued = 0;
      uint32_t ph = 1;
      while (cur.valid() && ok) {
        const int row0 = cur.row0();
        for (int k = 0; k < steps; k += 2) {
          ok = wait_one(bar_b + 16 * st + 8, ph, a.status, 62);
          if (!ok) break;
          const uint32_t dst = base + st * 2 * half_bytes;
          arrive_tx(bar_b + 16 * st, k + 1 < steps ? 2 * half_bytes : half_bytes);
          load_tile(dst, &p.x, k * 64, row0, bar_b + 16 * st);
          if (k + 1 < steps) load_tile(dst + half_bytes, &p.x, k * 64 + 64, row0, bar_b + 16 * st);
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
        wait_one(bar_b + 16 * st, ph ^ 1, a.status, 68);
      }
    }
  } else if (a.rows && (warp == 1 || warp == 3 || warp >= 16)) {
    // ------------------------------------------------------------------ rows of x, gathered
    // four rows per load; a load instruction takes a thread about 44 clocks, so six warps
    const uint32_t base = smem_u32(smem);
    const int w = warp < 16 ? warp >> 1 : warp - 14;
    int st = 0, issued = 0;
    uint32_t ph = 1;
    while (cur.valid() && ok) {
      const int row0 = cur.row0(), row1 = cur.row1();
      const int n4 = (row1 - row0 + 15) / 16 * 4;
      const int four = w + kGatherWarps * lane;
      const int mine = (n4 - w + kGatherWarps - 1) / kGatherWarps;  // fours of this warp
      int4 idx = make_int4(0, 0, 0, 0);  // (bad and missing rows load row 0)
      if (four < n4) {
        int v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int r = row0 + four * 4 + c;
          v[c] = r < row1 ? a.rows[r] : 0;
          if (v[c] < 0 || v[c] >= a.x_rows) v[c] = 0;
        }
        idx = make_int4(v[0], v[1], v[2], v[3]);
      }
      for (int k = 0; k < steps; k += 2) {
        ok = wait_warp(bar_b + 16 * st + 8, ph, a.status, 62);
        if (!ok) break;
        const uint32_t dst = base + st * 2 * half_bytes + four * 512;
        if (lane == 0) arrive_tx(bar_b + 16 * st, mine * (k + 1 < steps ? 1024 : 512));
        __syncwarp();
        if (four < n4) {
          load_rows4(dst, &p.x, k * 64, idx, bar_b + 16 * st);
          if (k + 1 < steps) load_rows4(dst + half_bytes, &p.x, k * 64 + 64, idx, bar_b + 16 * st);
        }
        ++issued;
        if (++st == p.b_stages) {
          st = 0;
          ph ^= 1;
        }
      }
      cur.next();
    }
    for (int i = min(issued, p.b_stages); i > 0; --i) {
      st = st ? st - 1 : p.b_stages - 1;
      if (st == p.b_stages - 1) ph ^= 1;
      wait_warp(bar_b + 16 * st, ph ^ 1, a.status, 68);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ packed codes
    if (lane == 0) {
      const uint32_t base = smem_u32(codes);
      const int spans = (steps + 3) / 4;
      int slot = 0, issued = 0;
      uint32_t ph = 1;
      while (cur.valid() && ok) {
        const int row = cur.e * a.N + cur.j * (GATED ? 64 : 128);
        for (int span = 0; span < spans; ++span) {
          ok = wait_one(bar_c + 16 * slot + 8, ph, a.status, 69);
          if (!ok) break;
          const uint32_t dst = base + slot * kSlotBytes;
          arrive_tx(bar_c + 16 * slot, kSlotBytes);
          if (GATED) {
#pragma unroll
            for (int i = 0; i < 8; ++i)  // 16 gate rows, their 16 up rows, per quarter
              load_tile(dst + i * 2048, &p.codes, span * 128, row + (i >> 1) * 16 + (i & 1) * n_out,
                        bar_c + 16 * slot);
          } else {
            load_tile(dst, &p.codes, span * 128, row, bar_c + 16 * slot);
          }
          ++issued;
          if (++slot == kSlots) {
            slot = 0;
            ph ^= 1;
          }
        }
        cur.next();
      }
      for (int i = min(issued, kSlots); i > 0; --i) {
        slot = slot ? slot - 1 : kSlots - 1;
        if (slot == kSlots - 1) ph ^= 1;
        wait_one(bar_c + 16 * slot, ph ^ 1, a.status, 70);
      }
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------------ MMA issuer
    // One thread and as few instructions as it takes: an MMA or a commit takes it 44 clocks.
    constexpr bool kBf = std::is_same<T, __nv_bfloat16>::value;
    if (elect_one()) {
      const uint64_t desc = tc::sdesc_sw128(smem_u32(smem), 16, 1024);
      const uint32_t dlo = (uint32_t)desc, dhi = (uint32_t)(desc >> 32);
      const uint32_t dhalf = (uint32_t)half_bytes >> 4;  // descriptor units of 16 bytes
      const uint32_t bb_end = bar_b + 16 * p.b_stages;
      uint32_t bb = bar_b, blo = dlo;  // full barrier and descriptor of the B stage
      uint32_t bph = 0, as = 0, aph = 0, tile = 0;
      while (cur.valid() && ok) {
        const int rows = cur.row1() - cur.row0();
        const uint32_t idesc = tc::idesc_f16(kBf, 128, 0, false, false) +
                               ((uint32_t)((rows + 15) / 16 * 2) << 17);
        const uint32_t buf = tile & 1, acc = tmem + buf * kMaxTok;
        ok = wait_one(bar_acc + 16 * buf + 8, ((tile >> 1) & 1) ^ 1, a.status, 63);
        for (int k = 0; k < steps && ok; k += 2) {
          ok = wait_one(bb, bph, a.status, 64) && wait_one(bar_a + 16 * as, aph, a.status, 65);
          if (!ok) break;
          tc::fence_after_sync();
          const uint32_t am = tmem + kACol + as * kACols;
          mma4(acc, am, blo, dhi, idesc, k > 0 ? 1u : 0u);
          if (k + 1 < steps) mma4(acc, am + 32, blo + dhalf, dhi, idesc, 1u);
          commit(bar_a + 16 * as + 8);
          commit(bb + 8);
          as ^= 1;
          aph ^= as ^ 1;
          bb += 16;
          blo += 2 * dhalf;
          if (bb == bb_end) {
            bb = bar_b;
            blo = dlo;
            bph ^= 1;
          }
        }
        if (ok) commit(bar_acc + 16 * buf);
        ++tile;
        cur.next();
      }
      // every MMA has completed before tensor memory is freed
      commit(bar_fin);
      wait_one(bar_fin, 0, a.status, 66);
    }
    __syncwarp();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == 0) tc::tmem_dealloc(tmem, 512);
}

size_t smem_bytes(int E) {
  return 1024 + kBBytes + kSlots * kSlotBytes + (size_t)(E + 1) * sizeof(int);
}

template <typename T, bool GATED, int SB>
int launch_tc_s(TcArgs& p, int grid, cudaStream_t st) {
  const size_t smem = smem_bytes(p.a.E);
  static std::atomic<unsigned long long> ready{0};  // devices whose shared memory bound is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return QKV_ECUDA;
  if (dev < 0 || dev >= kMaxDevices || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(matmul_tc_kernel<T, GATED, SB>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)smem_bytes(kMaxExperts)) != cudaSuccess)
      return QKV_ECUDA;
    if (dev >= 0 && dev < kMaxDevices) ready.fetch_or(1ull << dev);
  }
  if (!make_rows_map(&p.codes, p.a.w, 1, p.a.K / 2, (long long)p.a.E * p.a.N, p.a.K / 2, 128,
                     GATED ? 16 : 128) ||
      !make_rows_map(&p.x, p.a.x, 2, p.a.K, p.a.x_rows, p.a.ldx * 2, 64, p.a.rows ? 1 : p.tok))
    return QKV_ECUDA;
  matmul_tc_kernel<T, GATED, SB><<<grid, kThreads, smem, st>>>(p);
  return QKV_OK;
}

template <typename T, bool GATED>
int launch_tc_t(TcArgs& p, int grid, cudaStream_t st) {
  const int groups = p.a.K / 64;
  const uintptr_t at = (uintptr_t)p.a.scales | (uintptr_t)p.a.biases;
  if (groups % 8 == 0 && at % 16 == 0) return launch_tc_s<T, GATED, 2>(p, grid, st);
  if (groups % 2 == 0 && at % 4 == 0) return launch_tc_s<T, GATED, 1>(p, grid, st);
  return launch_tc_s<T, GATED, 0>(p, grid, st);
}

}  // namespace

bool matmul_tc_fits(int E, int N) {
  return E <= kMaxExperts && (long long)E * N < (1ll << 31) - 256;  // 32-bit TMA coordinates
}

int launch_matmul_tc(const MatmulArgs& a, cudaStream_t st) {
  const bool gated = a.act == QKV_ACT_SWIGLU;
  const int n_out = gated ? a.N / 2 : a.N;
  const int sms = num_sms();
  TcArgs p;
  p.a = a;
  p.n_tiles = gated ? (n_out + 63) / 64 : (n_out + 127) / 128;
  // One matrix: the row tile that leaves the fewest idle SMs in the last wave. Experts: the
  // counts are on the device, so the largest.
  p.tok = kMaxTok;
  if (!a.offsets) {
    long long best = -1;
    for (int tok = kMaxTok; tok >= 16; tok -= 16) {
      const Split s = split_rows(a.R, tok);
      const long long tiles = (long long)s.n * p.n_tiles;
      const long long cost = (tiles + sms - 1) / sms * tile_cost(s.per);
      if (best < 0 || cost < best) {
        best = cost;
        p.tok = tok;
      }
    }
  }
  const int most = std::min(a.R, p.tok);
  p.tok = (most + 15) / 16 * 16;
  p.b_stages = std::min(kMaxBStages, kBBytes / (p.tok * 256));
  long long tiles = (long long)((a.R + p.tok - 1) / p.tok + (a.offsets ? std::min(a.E, a.R) : 0)) * p.n_tiles;
  const int grid = (int)std::min<long long>(tiles, sms);
  if (a.dtype == QKV_BF16)
    return gated ? launch_tc_t<__nv_bfloat16, true>(p, grid, st)
                 : launch_tc_t<__nv_bfloat16, false>(p, grid, st);
  return gated ? launch_tc_t<__half, true>(p, grid, st) : launch_tc_t<__half, false>(p, grid, st);
}

}  // namespace qkv
