// Products of a few rows with affine 4-bit weights (sm_100a): y = x W^T with
// W[n][k] = scale[n][k/64] * code[n][k] + bias[n][k/64], for one weight matrix or one per
// expert over rows sorted by expert.
//
// Mathematics. Per group g of 64 the codes factor out of the scale:
//     y[m][n] = sum_g scale[n][g] * (sum_k code[n][k] x[m][k]) + bias[n][g] * (sum_k x[m][k])
// so the inner sums run over exact small integers on mma.sync (m16n8k16, fp32 accumulation)
// and nothing of the weight is rounded. The A operand holds 16 weight rows, the B operand up
// to 8 rows of x. Codes enter the MMA without a conversion: in bf16 as 128 + code (the code
// is the low mantissa bits of 128.0; the 128 * sum_k x is taken off with the bias), in f16 as
// the subnormal code * 2^-24 (taken out of the result). sum_k x comes from the same tensor
// pipe with a matrix of ones.
//
// K order. A 32-bit word holds codes k..k+7 LSB-first, and one shift-and-mask yields the pair
// (i, i+4); the MMA sums over k, so x is paired the same way and no code moves.
//
// What bounds it: the packed weights, read once from HBM. A warp owns 16 weight rows and a
// share of the K chunks (256 values, 128 bytes of each row), which it copies into its own ring
// of shared-memory stages with cp.async, whole lines at a time: the load pipe looks up one line
// a clock, and fragments read from global memory directly cost it 8 lines per 256 bytes. Warps
// of a CTA split K until the machine has enough of them to keep HBM busy, and add their sums
// through shared memory in a fixed order. The rows of x stay in shared memory, already paired.
// One row through 131071x2048 (f16): 31 us, 4.9 of 6.6 TB/s; a chunk of 4096 weights takes about
// 290 instructions of a warp, 112 of them the codes' masks and shifts. No unit is full (issue 59%
// of clocks, ALU pipe 57%, HBM 4.5 TB/s under the profiler): of the 6 clocks between two
// instructions of a warp 1.2 go to another warp's turn, 1.1 to fixed latencies, 0.9 to the ALU
// pipe's and 0.3 to a load, so fewer instructions, not more loads in flight, would shorten it. Few
// weights are bound by latency: one row through 5120x2048 5.0 us, of which a launch, the wait for
// x and one chunk's trip are 4. Three CTAs per SM with 80 registers were no faster (32.4 and 5.5).
#include <algorithm>
#include <atomic>

#include "matmul_internal.h"
#include "qkv_common.cuh"
#include "qkv_internal.h"

namespace qkv {

namespace {

constexpr int kWarps = 8;
constexpr int kChunk = 256;  // K values per warp step: four groups, one per lane of a quad

// D = A B or D += A B, m16n8k16 with fp32 sums
#define QKV_MMA16(TYPE)                                                                          \
  static __device__ __forceinline__ void mma0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, \
                                              uint32_t b1) {                                      \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                           \
                 ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"              \
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                 \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));       \
  }                                                                                               \
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,  \
                                             uint32_t b1) {                                       \
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                           \
                 ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"                  \
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])                                 \
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));                 \
  }

template <typename T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128.0 | code
  static constexpr uint32_t kOnes = 0x3f803f80u;
  static constexpr float kUnit = 1.f;  // what a code of 1 counts in the MMA
  // factor of the sum of x beside the scale's sum of codes
  static __device__ __forceinline__ float bias(float s, float b) { return fmaf(-128.f, s, b); }
  QKV_MMA16("bf16")
};
template <>
struct Codes<__half> {
  static constexpr uint32_t kMagic = 0u;  // the code as an f16 subnormal: code * 2^-24
  static constexpr uint32_t kOnes = 0x3c003c00u;
  static constexpr float kUnit = 1.f / 16777216.f;
  static __device__ __forceinline__ float bias(float, float b) { return b; }
  QKV_MMA16("f16")
};
#undef QKV_MMA16

__device__ __forceinline__ uint2 lds_v2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds_v4(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts_v4(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES)
               : "memory");
}

// The expert and the first row of token chunk `id` (chunks of `per` rows, experts in order),
// by a whole warp; false past the last chunk. Offsets are clamped into [0, R], and a
// decreasing pair counts as an empty expert, so bad offsets cannot leave the tensors. (With pairs
// that decrease the other experts can have any part of the R rows each, so chunks are counted in
// 64 bits.)
__device__ __forceinline__ bool find_chunk(const int* __restrict__ offsets, int E, int R, int per,
                                           long long id, int lane, int& expert, int& row0,
                                           int& row1) {
  long long base = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < E) {
      lo = min(max(offsets[e], 0), R);
      hi = min(max(offsets[e + 1], 0), R);
    }
    const int n = hi > lo ? (hi - lo + per - 1) / per : 0;
    long long sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const bool here = id < base + sum && id >= base + sum - n;
    const unsigned m = __ballot_sync(0xffffffffu, here);
    if (m) {
      const int src = __ffs(m) - 1;
      expert = e0 + src;
      const int first = __shfl_sync(0xffffffffu, lo + (int)(id - (base + sum - n)) * per, src);
      const int end = __shfl_sync(0xffffffffu, hi, src);
      row0 = first;
      row1 = min(first + per, end);
      return true;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// How many token chunks there are, by a whole warp.
__device__ __forceinline__ long long count_chunks(const int* __restrict__ offsets, int E, int R,
                                                  int per, int lane) {
  long long n = 0;
  for (int e = lane; e < E; e += 32) {
    const int lo = min(max(offsets[e], 0), R), hi = min(max(offsets[e + 1], 0), R);
    n += hi > lo ? (hi - lo + per - 1) / per : 0;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

constexpr int kStages = 3;                  // of one chunk, per warp
constexpr int kCodeBytes = 16 * 128;        // 16 weight rows
constexpr int kStageBytes = kCodeBytes + 2 * 16 * 8;  // and four scales and biases of each

// Dynamic shared memory of a CTA (8 KiB of sums are static): rows of x, their sums by group and
// a row of zeros, then the rings.
constexpr int kDynamicBytes = 227 * 1024 - 8192 - 256;
inline long long x_bytes(int rows, int K) { return (long long)rows * K * 2 + (long long)K / 64 * 32 + 128; }

// Rows of x in one pass over the weights: eight, or as many as fit beside the rings (0: not one).
// (Two or four tiles of eight rows to a pass were slower at every row count: 2048x4096 at 64 rows
// 15.4 us with one tile, 15.5 and 21.8 with two and four; 12288x2048 at 32 rows 18.8, 17.8, 28.5.)
int rows_per_pass(int R, int K) {
  int per = std::min(8, R);
  while (per > 0 && x_bytes(per, K) + kWarps * kStages * kStageBytes > kDynamicBytes) --per;
  return per;
}

struct RowsArgs {
  MatmulArgs a;
  int wk_count;  // warps that share K
  int tiles;     // of 16 weight rows
  int per;       // rows of x per CTA (at most 8)
};

// GATED: MMA rows 0-7 are gate rows, 8-15 the up rows of the same outputs. SB: how a row's four
// scales of a chunk are copied (8 bytes, 2 x 4, or one by one). GROUPED: with experts.
template <typename T, bool GATED, int SB, bool GROUPED>
__global__ void __launch_bounds__(kWarps * 32, 2) matmul_rows_kernel(const RowsArgs p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float red[2][kWarps][4][32];
  __shared__ int seg[3], sums_of[kWarps];
  __shared__ long long count_of;
  // everything here may come from the kernel before, the weights too
  wait_for_previous();
  const MatmulArgs& a = p.a;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int wk_count = p.wk_count;

  const int wk = warp % wk_count, wn = warp / wk_count, wn_count = kWarps / wk_count;
  const int n_out = GATED ? a.N / 2 : a.N;
  const int G = a.K / 64, chunks = (a.K + kChunk - 1) / kChunk, pieces = a.K / 32;
  const int units = (p.tiles + wn_count - 1) / wn_count;  // of wn_count tiles
  const uint32_t xs = smem_u32(smem);
  const uint32_t sums = xs + (uint32_t)p.per * a.K * 2;  // of each group of each row of x
  const uint32_t zeros = sums + (uint32_t)G * 32;        // what rows past the last read
  const uint32_t ring = zeros + 128 + warp * kStages * kStageBytes;
  // This CTA's units: every gridDim.x-th of its chunk of rows, or with experts an equal run of
  // those of all their chunks, whose number only the device knows.
  int lo = 0, hi = units, id = blockIdx.y;  // units counted from chunk `id`, `from` with experts
  long long from = 0;
  int my_lo = 0, my_hi = 0, my_n = 0, my_id = 0;  // rows, chunks and first chunk of expert threadIdx.x
  const bool few = a.E <= kWarps * 32;            // a thread for every expert
  if (GROUPED) {
    if (threadIdx.x < 3) seg[threadIdx.x] = 0;
    long long all = 0;
    if (few) {
      if ((int)threadIdx.x < a.E) {
        my_lo = min(max(a.offsets[threadIdx.x], 0), a.R);
        my_hi = min(max(a.offsets[threadIdx.x + 1], 0), a.R);
        my_n = my_hi > my_lo ? (my_hi - my_lo + p.per - 1) / p.per : 0;
      }
      int sum = my_n;  // (256 experts' chunks in 32 bits: more rows go to the other kernel)
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (lane == 31) sums_of[warp] = sum;
      __syncthreads();
      my_id = sum - my_n;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        my_id += w < warp ? sums_of[w] : 0;
        all += sums_of[w];
      }
    } else {
      if (warp == 0) {
        const long long n = count_chunks(a.offsets, a.E, a.R, p.per, lane);
        if (lane == 0) count_of = n;
      }
      __syncthreads();
      all = count_of;
    }
    all = __shfl_sync(0xffffffffu, all, 0) * units;
    const long long each = all / gridDim.x, first = blockIdx.x * each;
    const int more = (int)(all - each * gridDim.x), b = blockIdx.x;  // CTAs with one unit more
    from = (first + min(b, more)) / units;
    id = 0;
    lo = (int)(first + min(b, more) - from * units);
    hi = lo + (int)each + (b < more ? 1 : 0);
    if (lo >= hi) return;
    my_id -= (int)from;
  }

  int buf = 0;
  for (int first = 0; first < hi; first += units, ++id) {
    const int unit0 = GROUPED ? max(lo - first, 0) : blockIdx.x;
    const int unit1 = GROUPED ? min(hi - first, units) : units;
    const int step = GROUPED ? 1 : gridDim.x;
    int expert = 0, row0, row1;
    if (GROUPED) {
      if (few) {
        if (id >= my_id && id < my_id + my_n) {
          seg[0] = threadIdx.x;
          seg[1] = my_lo + (id - my_id) * p.per;
          seg[2] = min(my_lo + (id - my_id + 1) * p.per, my_hi);
        }
      } else if (warp == 0) {
        int e = 0, r0 = 0, r1 = 0;
        find_chunk(a.offsets, a.E, a.R, p.per, from + id, lane, e, r0, r1);
        if (lane == 0) {
          seg[0] = e;
          seg[1] = r0;
          seg[2] = r1;
        }
      }
      __syncthreads();  // (and no warp reads the rows of the chunk before)
      expert = __shfl_sync(0xffffffffu, seg[0], 0);
      row0 = __shfl_sync(0xffffffffu, seg[1], 0);
      row1 = __shfl_sync(0xffffffffu, seg[2], 0);
    } else {
      row0 = id * p.per;
      row1 = min(row0 + p.per, a.R);
    }
    const int rows = row1 - row0;

    // ---- the warp's stream of chunks: its tile of every unit, chunks wk, wk + wk_count, ... ----
    // weight row of row r of a tile (clamped into the matrix; what is past it is not stored)
    auto weight_row = [&](int tile, int r) -> long long {
      const int n = GATED ? min(tile * 8 + (r & 7), n_out - 1) + (r >> 3) * n_out
                          : min(tile * 16 + r, n_out - 1);
      return (long long)expert * a.N + n;
    };
    int ld_unit = unit0, ld_c = wk;
    const char* src[4];  // this lane's 16 bytes of rows lane/8 + 4i of the next chunk
    const char* ssrc;    // scales of row lane (biases of row lane - 16)
    auto set_src = [&]() {
      const int ld_tile = min(ld_unit * wn_count + wn, p.tiles - 1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        src[i] = (const char*)a.w + weight_row(ld_tile, (lane >> 3) + 4 * i) * (a.K / 2) + ld_c * 128 +
                 (lane & 7) * 16;
      ssrc = (const char*)(lane < 16 ? a.scales : a.biases) + weight_row(ld_tile, lane & 15) * G * 2 +
             ld_c * 8;
    };
    set_src();
    // rows lane/8 + 4i, a 512-byte step (the swizzle keeps the fragment reads apart); scales
    const uint32_t code_to = ring + (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) & 3) << 1) << 4);
    const uint32_t scale_to = ring + kCodeBytes + lane * 8;
    uint32_t ld_at = 0;  // the stage's offset
    auto load = [&]() {
      if (ld_unit < unit1) {
        if (ld_c * 8 + (lane & 7) < pieces) {
#pragma unroll
          for (int i = 0; i < 4; ++i) cp16(code_to + ld_at + i * 512, src[i]);
        }
        if (SB == 2) {
          cp_small<8>(scale_to + ld_at, ssrc);
        } else if (SB == 1) {
          cp_small<4>(scale_to + ld_at, ssrc);
          if (ld_c * 4 + 2 < G) cp_small<4>(scale_to + ld_at + 4, ssrc + 4);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (ld_c * 4 + j < G) {
              const uint16_t v = __ldg((const uint16_t*)ssrc + j);
              asm volatile("st.shared.u16 [%0], %1;" ::"r"(scale_to + ld_at + 2 * j), "h"(v) : "memory");
            }
        }
        ld_c += wk_count;
        if (ld_c >= chunks) {
          ld_c = wk;
          ld_unit += step;
          set_src();
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) src[i] += wk_count * 128;
          ssrc += wk_count * 8;
        }
      }
      ld_at = ld_at + kStageBytes == kStages * kStageBytes ? 0 : ld_at + kStageBytes;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kStages - 1; ++i) load();

    // ---- rows of x: 128 bytes per (group, row), the 32 bytes of lane t at 32 t, values paired
    // as the codes are, the two halves of odd rows swapped (their reads then share no bank) -----
    for (int i = threadIdx.x; i < rows * G * 4; i += kWarps * 32) {
      const int m = i / (G * 4), q = i - m * (G * 4);  // q = group * 4 + t
      const int r = row0 + m;
      const int from = a.rows ? a.rows[r] : r;
      uint4 u = make_uint4(0, 0, 0, 0), v = u;
      if (from >= 0 && from < a.x_rows) {
        const uint4* at = (const uint4*)((const char*)a.x + ((long long)from * a.ldx + q * 16) * 2);
        u = __ldg(at);
        v = __ldg(at + 1);
      }
      const uint32_t to = xs + ((q >> 2) * rows + m) * 128 + (q & 3) * 32;
      sts_v4(to + (m & 1) * 16, make_uint4(prmt(u.x, u.z, 0x5410), prmt(u.x, u.z, 0x7632),
                                           prmt(u.y, u.w, 0x5410), prmt(u.y, u.w, 0x7632)));
      sts_v4(to + (~m & 1) * 16, make_uint4(prmt(v.x, v.z, 0x5410), prmt(v.x, v.z, 0x7632),
                                            prmt(v.y, v.w, 0x5410), prmt(v.y, v.w, 0x7632)));
    }
    if (threadIdx.x < 8) sts_v4(zeros + threadIdx.x * 16, make_uint4(0, 0, 0, 0));
    __syncthreads();

    // one group of x as B fragments: lane (g, t) holds 16 values of row g
    const uint32_t my_x = (g < rows ? xs + g * 128 : zeros) + t * 32, x_step = g < rows ? rows * 128 : 0;
    auto x_frag = [&](uint32_t at, uint4 (&xv)[2]) {
      xv[0] = lds_v4(at + (g & 1) * 16);
      xv[1] = lds_v4(at + (~g & 1) * 16);
    };
    // sums of x by group, with a matrix of ones, in the unit of the codes' sums
    for (int j = warp; j < G; j += kWarps) {
      const uint32_t ones[4] = {Codes<T>::kOnes, Codes<T>::kOnes, Codes<T>::kOnes, Codes<T>::kOnes};
      uint4 xv[2];
      x_frag(my_x + j * x_step, xv);
      float d[4];
      Codes<T>::mma0(d, ones, xv[0].x, xv[0].y);
      Codes<T>::mma(d, ones, xv[0].z, xv[0].w);
      Codes<T>::mma(d, ones, xv[1].x, xv[1].y);
      Codes<T>::mma(d, ones, xv[1].z, xv[1].w);
      if (g == 0)
        asm volatile("st.shared.v2.f32 [%0], {%1,%2};" ::"r"(sums + j * 32 + t * 8), "f"(d[0] * Codes<T>::kUnit),
                     "f"(d[1] * Codes<T>::kUnit)
                     : "memory");
    }
    __syncthreads();
    uint32_t code_at[4];  // of the chunk's groups
#pragma unroll
    for (int j = 0; j < 4; ++j)
      code_at[j] = ring + g * 128 + (((2 * j + (t >> 1)) ^ (g & 3) << 1) << 4) + (t & 1) * 8;
    // results of a tile: lane (g, t) holds weight rows g and g + 8 for rows 2t and 2t + 1 of x
    auto store = [&](int tile, float (&acc)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] *= 1.f / Codes<T>::kUnit;
      const int nA = GATED ? tile * 8 + g : tile * 16 + g, nB = GATED ? nA : nA + 8;
      T* out = (T*)a.out;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = t * 2 + i;
        if (r >= rows) continue;
        T* o = out + (long long)(row0 + r) * n_out;
        if (GATED) {
          const float gate = acc[i], up = acc[i + 2];
          if (nA < n_out) o[nA] = Elem<T>::from_f32(gate / (1.f + expf(-gate)) * up);
        } else {
          if (nA < n_out) o[nA] = Elem<T>::from_f32(acc[i]);
          if (nB < n_out) o[nB] = Elem<T>::from_f32(acc[i + 2]);
        }
      }
    };
    uint32_t at = 0;  // the stage's offset
    for (int unit = unit0; unit < unit1; unit += step) {
      const int tile = unit * wn_count + wn;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c = wk; c < chunks; c += wk_count) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        load();  // into the stage of the chunk before
        // scales and biases of rows g and g + 8, four groups each
        const uint32_t sat = ring + at + kCodeBytes + g * 8;
        const uint2 sA = lds_v2(sat), sB = lds_v2(sat + 64), bA = lds_v2(sat + 128), bB = lds_v2(sat + 192);
        uint32_t xa = my_x + c * 4 * x_step;
        const uint32_t sum_at = sums + c * 128 + t * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (SB != 2 && c * 4 + j >= G) break;  // (SB 2: whole chunks)
          const uint2 wa = lds_v2(code_at[j] + at), wb = lds_v2(code_at[j] + at + 1024);
          uint32_t f[4][4];  // A fragments of the group's four MMAs
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t u = (i & 2 ? wa.y : wa.x) >> (8 * (i & 1));
            const uint32_t v = (i & 2 ? wb.y : wb.x) >> (8 * (i & 1));
            f[i][0] = and_or(u, 0x000f000fu, Codes<T>::kMagic);
            f[i][1] = and_or(v, 0x000f000fu, Codes<T>::kMagic);
            f[i][2] = and_or(u >> 4, 0x000f000fu, Codes<T>::kMagic);
            f[i][3] = and_or(v >> 4, 0x000f000fu, Codes<T>::kMagic);
          }
          const uint32_t s0 = j < 2 ? sA.x : sA.y, s1 = j < 2 ? sB.x : sB.y;
          const uint32_t b0 = j < 2 ? bA.x : bA.y, b1 = j < 2 ? bB.x : bB.y;
          const int sh = (j & 1) * 16;
          const float q0 = Elem<T>::bits_to_f32((uint16_t)(s0 >> sh));
          const float q1 = Elem<T>::bits_to_f32((uint16_t)(s1 >> sh));
          const float o0 = Codes<T>::bias(q0, Elem<T>::bits_to_f32((uint16_t)(b0 >> sh)));
          const float o1 = Codes<T>::bias(q1, Elem<T>::bits_to_f32((uint16_t)(b1 >> sh)));
          uint4 xv[2];
          x_frag(xa, xv);
          xa += x_step;
          float d[4];
          Codes<T>::mma0(d, f[0], xv[0].x, xv[0].y);
          Codes<T>::mma(d, f[1], xv[0].z, xv[0].w);
          Codes<T>::mma(d, f[2], xv[1].x, xv[1].y);
          Codes<T>::mma(d, f[3], xv[1].z, xv[1].w);
          const uint2 sx = lds_v2(sum_at + j * 32);
          const float sx0 = __uint_as_float(sx.x), sx1 = __uint_as_float(sx.y);
          acc[0] = fmaf(q0, d[0], fmaf(o0, sx0, acc[0]));
          acc[1] = fmaf(q0, d[1], fmaf(o0, sx1, acc[1]));
          acc[2] = fmaf(q1, d[2], fmaf(o1, sx0, acc[2]));
          acc[3] = fmaf(q1, d[3], fmaf(o1, sx1, acc[3]));
        }
        at = at + kStageBytes == kStages * kStageBytes ? 0 : at + kStageBytes;
      }

      if (wk_count > 1) {
        // (two buffers: the reader of this unit's passes the next unit's barrier before anyone
        // writes here again)
        if (wk) {
#pragma unroll
          for (int i = 0; i < 4; ++i) red[buf][warp][i][lane] = acc[i];
        }
        named_bar_sync(1 + wn, wk_count * 32);
        if (!wk) {
          for (int o = 1; o < wk_count; ++o)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] += red[buf][warp + o][i][lane];
        }
        buf ^= 1;
      }
      if (wk == 0 && tile < p.tiles) store(tile, acc);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <typename T, bool GATED, int SB, bool GROUPED>
int launch_rows_s(const RowsArgs& p, dim3 grid, size_t smem, cudaStream_t st) {
  static std::atomic<unsigned long long> ready{0};  // devices whose shared memory bound is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return QKV_ECUDA;
  if (dev < 0 || dev >= kMaxDevices || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(matmul_rows_kernel<T, GATED, SB, GROUPED>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kDynamicBytes) != cudaSuccess)
      return QKV_ECUDA;
    if (dev >= 0 && dev < kMaxDevices) ready.fetch_or(1ull << dev);
  }
  return launch(true, matmul_rows_kernel<T, GATED, SB, GROUPED>, grid, kWarps * 32, smem, st, p);
}

template <typename T, bool GATED, bool GROUPED>
int launch_rows_g(const RowsArgs& p, dim3 grid, size_t smem, cudaStream_t st) {
  const int groups = p.a.K / 64;
  const uintptr_t at = (uintptr_t)p.a.scales | (uintptr_t)p.a.biases;
  if (groups % 4 == 0 && at % 8 == 0) return launch_rows_s<T, GATED, 2, GROUPED>(p, grid, smem, st);
  if (groups % 2 == 0 && at % 4 == 0) return launch_rows_s<T, GATED, 1, GROUPED>(p, grid, smem, st);
  return launch_rows_s<T, GATED, 0, GROUPED>(p, grid, smem, st);
}

template <typename T>
int launch_rows(const MatmulArgs& a, cudaStream_t st) {
  const bool gated = a.act == QKV_ACT_SWIGLU;
  const int n_out = gated ? a.N / 2 : a.N;
  RowsArgs p;
  p.a = a;
  p.tiles = gated ? (n_out + 7) / 8 : (n_out + 15) / 16;
  p.per = rows_per_pass(a.R, a.K);
  if (p.per < 1) return QKV_EUNSUPPORTED;
  long long segs = (a.R + p.per - 1ll) / p.per;
  if (a.offsets) segs = std::min<long long>(a.R, std::min(a.E, a.R) + segs);
  if (!a.offsets && segs > 65535) return QKV_EUNSUPPORTED;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const size_t smem = x_bytes(p.per, a.K) + kWarps * kStages * kStageBytes;
  const int resident = num_sms() * (smem > 104 * 1024 ? 1 : 2);
  // Warps that share K: the number whose longest warp has the least to do. A unit of a CTA costs
  // its chunks and about half a chunk more for the sums (through shared memory when shared).
  // With experts that is a guess: the bound on their chunks counts empty experts too, unless
  // there are few rows.
  const long long guess = !a.offsets || 2ll * a.R <= a.E ? segs : (2 * segs + 2) / 3;
  int best = 0;
  long long best_cost = 0;
  for (int wk = 1; wk <= kWarps && wk <= chunks; wk *= 2) {
    const int units = (p.tiles + kWarps / wk - 1) / (kWarps / wk);
    const long long ctas = std::max(1ll, resident / segs);
    const long long rounds = a.offsets ? (guess * units + resident - 1) / resident
                                       : (units + ctas - 1) / ctas;
    const long long cost = rounds * (4 * ((chunks + wk - 1) / wk) + (wk > 1 ? 2 : 1));
    if (!best || cost < best_cost) {
      best = wk;
      best_cost = cost;
    }
  }
  p.wk_count = best;
  const int units = (p.tiles + kWarps / best - 1) / (kWarps / best);
  if (a.offsets && segs * units > 1ll << 30) return QKV_EUNSUPPORTED;
  const dim3 grid =
      a.offsets ? dim3((unsigned)std::min<long long>(resident, segs * units))
                : dim3((unsigned)std::min<long long>(units, std::max(1ll, resident / segs)),
                       (unsigned)segs);
  if (a.offsets)
    return gated ? launch_rows_g<T, true, true>(p, grid, smem, st)
                 : launch_rows_g<T, false, true>(p, grid, smem, st);
  return gated ? launch_rows_g<T, true, false>(p, grid, smem, st)
               : launch_rows_g<T, false, false>(p, grid, smem, st);
}

}  // namespace

int launch_matmul_rows(const MatmulArgs& a, cudaStream_t st) {
  if (a.dtype == QKV_BF16) return launch_rows<__nv_bfloat16>(a, st);
  return launch_rows<__half>(a, st);
}

// Few rows go to the kernel above, which takes a pass over the weights for every rows_per_pass
// rows; the tcgen05 kernel reads them once, but takes 6 us and 2.6 for every 1024 of K and round of
// 128 x 192 tiles over the SMs, the other 4 and 1 for every 8 million weights of a pass (both
// measured, to 15%).
// us of this and of that kernel at 16, 32, 64 and 96 rows: 2048x4096 6.9 9.1 13.4 18.3, 16.8 17.0
// 17.3 17.8; 5120x2048 8.4 10.9 15.5 19.7, 11.3 11.4 11.8 12.3; 12288x2048 11.5 16.8 27.3 34.6,
// 12.2 12.4 12.8 13.4. At 4, 8, 12 and 16 rows of long K: 8192x14336 (five rows a pass) 22.3 35.2
// 50.4 59.5, 46.3 throughout; 8192x28672 (two) 64.9 114 172 232, 88.0; 5120x28672 49.3 79.8 113
// 143, 86.8; 2048x28672 24.6 39.3 53.8 67.5, 86.2.
// Experts' counts are on the device. With the counts of routed tokens both kernels take the same
// time at about ten rows on average, or earlier where some experts are popular (us of this and of
// that kernel at 8, 10 and 12 rows for each of the experts on average; logits normal, "popular" with
// as much again by expert): 128 of 1536x2048 gated 69.7 82.4 92.9, 83.9 84.3 84.5, popular 68.2 75.7
// 88.5, 62.9 67.4 67.9; 64 of these 40.7 42.7 54.0, 52.0 52.2 52.4, popular 40.2 42.8 52.4, 40.4
// 41.0 46.3; 32 of these 22.5 25.7 30.5, 32.7 32.7 32.8; 128 of 2048x768 39.0 45.3 49.7, 49.2 49.5
// 49.4, popular 38.3 42.4 48.0, 37.2 41.6 40.7; 60 of 2048x1408 39.0 41.6 48.2, 44.1 44.3 44.7.
bool matmul_takes_tc(int R, int E, int N, int K) {
  if (!matmul_tc_fits(E, N)) return false;
  const int per = rows_per_pass(R, K);
  if (per < 1) return true;  // a row of x does not fit shared memory beside the rings above
  if (R > 65528) return true;  // the kernel above has one grid row for every eight at most
  const int experts = std::min(E, R);
  if (R <= (long long)per * experts || (experts > 1 && 4ll * R <= 5ll * per * experts)) return false;
  const long long passes = (R + per - 1ll) / per, sms = num_sms();
  const long long tiles = (N + 127ll) / 128 * ((R + 191ll) / 192);
  return passes * N > 16000000 / K + 20000 * ((tiles + sms - 1) / sms);
}

int launch_matmul(const MatmulArgs& a, cudaStream_t st) {
  if (matmul_takes_tc(a.R, a.E, a.N, a.K)) return launch_matmul_tc(a, st);
  return launch_matmul_rows(a, st);
}

}  // namespace qkv
