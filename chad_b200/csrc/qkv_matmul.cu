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
// the subnormal code * 2^-24 (the scale carries the 2^24). sum_k x comes from the same tensor
// pipe with a matrix of ones.
//
// K order. A 32-bit word holds codes k..k+7 LSB-first, and one shift-and-mask yields the pair
// (i, i+4); the MMA sums over k, so x is paired the same way and no code moves.
//
// What bounds it: the packed weights, read once from HBM. A warp owns 16 weight rows and a
// share of the K chunks (256 values, 128 bytes of each row); warps of a CTA split K until the
// machine has enough of them to keep HBM busy, and add their sums through shared memory in a
// fixed order.
#include <algorithm>

#include "matmul_internal.h"
#include "qkv_common.cuh"
#include "qkv_internal.h"

namespace qkv {

namespace {

constexpr int kWarps = 8;
constexpr int kChunk = 256;  // K values per warp step: four groups, one per lane of a quad

template <typename T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;  // 128.0 | code
  static constexpr uint32_t kOnes = 0x3f803f80u;
  // scale of the accumulated sum, and bias of the x sum
  static __device__ __forceinline__ float scale(float s) { return s; }
  static __device__ __forceinline__ float bias(float s, float b) { return fmaf(-128.f, s, b); }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Codes<__half> {
  static constexpr uint32_t kMagic = 0u;  // the code as an f16 subnormal: code * 2^-24
  static constexpr uint32_t kOnes = 0x3c003c00u;
  static __device__ __forceinline__ float scale(float s) { return s * 16777216.f; }
  static __device__ __forceinline__ float bias(float, float b) { return b; }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    mma16816(d, a, b0, b1);
  }
};

__device__ __forceinline__ uint2 ld_stream(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
               : "=r"(v.x), "=r"(v.y)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint4 ld_x(const void* p) { return __ldg((const uint4*)p); }

// The expert and the first row of token chunk `id` (chunks of `per` rows, experts in order),
// by a whole warp; false past the last chunk. Offsets are clamped into [0, R], and a
// decreasing pair counts as an empty expert, so bad offsets cannot leave the tensors.
__device__ __forceinline__ bool find_chunk(const int* __restrict__ offsets, int E, int R, int per,
                                           int id, int lane, int& expert, int& row0, int& row1) {
  int base = 0;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, hi = 0;
    if (e < E) {
      lo = min(max(offsets[e], 0), R);
      hi = min(max(offsets[e + 1], 0), R);
    }
    const int n = hi > lo ? (hi - lo + per - 1) / per : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    const bool here = id < base + sum && id >= base + sum - n;
    const unsigned m = __ballot_sync(0xffffffffu, here);
    if (m) {
      const int src = __ffs(m) - 1;
      expert = e0 + src;
      const int first = __shfl_sync(0xffffffffu, lo + (id - (base + sum - n)) * per, src);
      const int end = __shfl_sync(0xffffffffu, hi, src);
      row0 = first;
      row1 = min(first + per, end);
      return true;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// MT token tiles of 8; GATED: MMA rows 0-7 are gate rows, 8-15 the up rows of the same outputs
template <typename T, int MT, bool GATED>
__global__ void __launch_bounds__(kWarps * 32)
    matmul_rows_kernel(const MatmulArgs a, int wk_count, int tiles) {
  __shared__ float red[kWarps][MT * 4][32];
  __shared__ int seg[3];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  constexpr int PER = 8 * MT;

  int expert = 0, row0, row1;
  if (a.offsets) {
    if (warp == 0) {
      int e = 0, r0 = 0, r1 = -1;
      find_chunk(a.offsets, a.E, a.R, PER, blockIdx.y, lane, e, r0, r1);
      if (lane == 0) {
        seg[0] = e;
        seg[1] = r0;
        seg[2] = r1;
      }
    }
    __syncthreads();
    expert = seg[0];
    row0 = seg[1];
    row1 = seg[2];
    if (row1 < 0) return;
  } else {
    row0 = blockIdx.y * PER;
    row1 = min(row0 + PER, a.R);
  }

  const int wk = warp % wk_count, wn = warp / wk_count;
  const int tile = blockIdx.x * (kWarps / wk_count) + wn;
  const int n_out = GATED ? a.N / 2 : a.N;
  const int G = a.K / 64, chunks = (a.K + kChunk - 1) / kChunk;
  // weight rows of this lane (clamped into the matrix; what is past it is not stored)
  const int nA = GATED ? tile * 8 + g : tile * 16 + g;
  const int nB = GATED ? nA : nA + 8;
  const int last = n_out - 1;
  const long long rA = (long long)expert * a.N + min(nA, last);
  const long long rB = (long long)expert * a.N + min(nB, last) + (GATED ? n_out : 0);
  const char* wA = (const char*)a.w + rA * (a.K / 2) + t * 8;
  const char* wB = (const char*)a.w + rB * (a.K / 2) + t * 8;
  const uint16_t* sA = (const uint16_t*)a.scales + rA * G;
  const uint16_t* sB = (const uint16_t*)a.scales + rB * G;
  const uint16_t* bA = (const uint16_t*)a.biases + rA * G;
  const uint16_t* bB = (const uint16_t*)a.biases + rB * G;

  // rows of x: token g of each tile
  const char* xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = row0 + m * 8 + g;
    int src = -1;
    if (r < row1) src = a.rows ? a.rows[r] : r;
    xp[m] = src >= 0 && src < a.x_rows
                ? (const char*)a.x + ((long long)src * a.ldx + t * 16) * 2
                : nullptr;
  }

  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[m][i] = 0.f;

  uint2 pa[4], pb[4];          // packed codes of the chunk: rows g and g + 8
  uint32_t ps = 0, pbias = 0;  // (row g | row g+8 << 16) scale and bias of group t
  auto load_w = [&](int c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = c < chunks && c * 4 + j < G;
      pa[j] = in ? ld_stream(wA + (long long)c * 128 + j * 32) : make_uint2(0, 0);
      pb[j] = in ? ld_stream(wB + (long long)c * 128 + j * 32) : make_uint2(0, 0);
    }
    ps = pbias = 0;
    if (c < chunks && c * 4 + t < G) {
      ps = sA[c * 4 + t] | (uint32_t)sB[c * 4 + t] << 16;
      pbias = bA[c * 4 + t] | (uint32_t)bB[c * 4 + t] << 16;
    }
  };
  auto load_x = [&](int gi, uint4 (&v)[MT][2]) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const bool in = xp[m] && gi < G;
      v[m][0] = in ? ld_x(xp[m] + (long long)gi * 128) : make_uint4(0, 0, 0, 0);
      v[m][1] = in ? ld_x(xp[m] + (long long)gi * 128 + 16) : make_uint4(0, 0, 0, 0);
    }
  };

  if (tile < tiles) {
    uint4 xn[MT][2];
    load_w(wk);
    load_x(wk * 4, xn);
    for (int c = wk; c < chunks; c += wk_count) {
      uint2 ca[4], cb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ca[j] = pa[j];
        cb[j] = pb[j];
      }
      const uint32_t cs = ps, cbias = pbias;
      load_w(c + wk_count);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t xr[MT][8];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint4 v = xn[m][i];
            xr[m][i * 4 + 0] = prmt(v.x, v.z, 0x5410);
            xr[m][i * 4 + 1] = prmt(v.x, v.z, 0x7632);
            xr[m][i * 4 + 2] = prmt(v.y, v.w, 0x5410);
            xr[m][i * 4 + 3] = prmt(v.y, v.w, 0x7632);
          }
        load_x(j < 3 ? c * 4 + j + 1 : (c + wk_count) * 4, xn);
        if (c * 4 + j < G) {
          float d[MT][4], sx[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][i] = sx[m][i] = 0.f;
          const uint32_t ones[4] = {Codes<T>::kOnes, Codes<T>::kOnes, Codes<T>::kOnes,
                                    Codes<T>::kOnes};
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t u = i ? ca[j].y : ca[j].x, v = i ? cb[j].y : cb[j].x;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t f[4] = {and_or(u >> (8 * h), 0x000f000fu, Codes<T>::kMagic),
                                     and_or(v >> (8 * h), 0x000f000fu, Codes<T>::kMagic),
                                     and_or(u >> (8 * h + 4), 0x000f000fu, Codes<T>::kMagic),
                                     and_or(v >> (8 * h + 4), 0x000f000fu, Codes<T>::kMagic)};
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                Codes<T>::mma(d[m], f, xr[m][i * 4 + h * 2], xr[m][i * 4 + h * 2 + 1]);
                Codes<T>::mma(sx[m], ones, xr[m][i * 4 + h * 2], xr[m][i * 4 + h * 2 + 1]);
              }
            }
          }
          // scale and bias of group j live in lane j of the quad
          const uint32_t s2 = __shfl_sync(0xffffffffu, cs, (lane & ~3) | j);
          const uint32_t b2 = __shfl_sync(0xffffffffu, cbias, (lane & ~3) | j);
          const float s0 = Elem<T>::bits_to_f32((uint16_t)s2), s1 = Elem<T>::bits_to_f32((uint16_t)(s2 >> 16));
          const float b0 = Codes<T>::bias(s0, Elem<T>::bits_to_f32((uint16_t)b2));
          const float b1 = Codes<T>::bias(s1, Elem<T>::bits_to_f32((uint16_t)(b2 >> 16)));
          const float q0 = Codes<T>::scale(s0), q1 = Codes<T>::scale(s1);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            acc[m][0] = fmaf(q0, d[m][0], fmaf(b0, sx[m][0], acc[m][0]));
            acc[m][1] = fmaf(q0, d[m][1], fmaf(b0, sx[m][1], acc[m][1]));
            acc[m][2] = fmaf(q1, d[m][2], fmaf(b1, sx[m][0], acc[m][2]));
            acc[m][3] = fmaf(q1, d[m][3], fmaf(b1, sx[m][1], acc[m][3]));
          }
        }
      }
    }
  }

  if (wk_count > 1) {
    if (wk) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][m * 4 + i][lane] = acc[m][i];
    }
    __syncthreads();
    if (wk) return;
    for (int o = 1; o < wk_count; ++o)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][i] += red[warp + o][m * 4 + i][lane];
  }
  if (tile >= tiles) return;

  T* out = (T*)a.out;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + m * 8 + t * 2 + i;
      if (r >= row1) continue;
      T* o = out + (long long)r * n_out;
      if (GATED) {
        const float gate = acc[m][i], up = acc[m][i + 2];
        if (nA < n_out) o[nA] = Elem<T>::from_f32(gate / (1.f + expf(-gate)) * up);
      } else {
        if (nA < n_out) o[nA] = Elem<T>::from_f32(acc[m][i]);
        if (nB < n_out) o[nB] = Elem<T>::from_f32(acc[m][i + 2]);
      }
    }
}

template <typename T, int MT>
int launch_rows(const MatmulArgs& a, cudaStream_t st) {
  const bool gated = a.act == QKV_ACT_SWIGLU;
  const int n_out = gated ? a.N / 2 : a.N;
  const int tiles = gated ? (n_out + 7) / 8 : (n_out + 15) / 16;
  const int per = 8 * MT;
  long long segs = (a.R + per - 1) / per;
  if (a.offsets) segs = std::min<long long>(a.R, (long long)std::min(a.E, a.R) + segs);
  if (segs > 65535) return QKV_EUNSUPPORTED;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  // warps share K until the machine holds enough of them to keep HBM busy
  int wk = 1;
  while (wk < kWarps && wk * 2 <= chunks && (long long)tiles * segs * wk < 16ll * num_sms()) wk *= 2;
  const int wn = kWarps / wk;
  const dim3 grid((unsigned)((tiles + wn - 1) / wn), (unsigned)segs);
  if (gated)
    matmul_rows_kernel<T, MT, true><<<grid, kWarps * 32, 0, st>>>(a, wk, tiles);
  else
    matmul_rows_kernel<T, MT, false><<<grid, kWarps * 32, 0, st>>>(a, wk, tiles);
  return QKV_OK;
}

}  // namespace

int launch_matmul_rows(const MatmulArgs& a, cudaStream_t st) {
  if (a.dtype == QKV_BF16) return launch_rows<__nv_bfloat16, 1>(a, st);
  return launch_rows<__half, 1>(a, st);
}

// By rows per weight matrix (experts without rows unknown): at 22 rows per expert the tcgen05
// kernel took 44 us where the one above took 122.
bool matmul_takes_tc(int R, int E, int N) {
  return matmul_tc_fits(E, N) && R >= 16ll * std::min(E, R);
}

int launch_matmul(const MatmulArgs& a, cudaStream_t st) {
  if (matmul_takes_tc(a.R, a.E, a.N)) return launch_matmul_tc(a, st);
  return launch_matmul_rows(a, st);
}

}  // namespace qkv
