// Routing of tokens to experts, and the weighted sum of the experts' rows (sm_100a).
//
// Route: the k largest of E logits per token (ties to the lowest expert, NaN counts as the
// largest), softmax weights over all logits or over the chosen ones, and the stable counting
// sort of the T*k pairs by expert: rows (token of each sorted pair), slots (sorted position
// of each pair) and offsets (first sorted pair of each expert).
//
// One warp per token holds its logits in registers as order-preserving unsigned keys; a
// selection is one redux.max over the keys and one redux.min over the indices that have it.
// A token takes an expert at most once, so a pair's rank within its expert is the number of
// earlier tokens that took it: a popcount over a per-expert bit mask of tokens. Counts and
// masks are integers, so the order of their atomics does not show.
//
// What bounds it: a decode batch is one block's latency; a long chunk reads the logits once
// (HBM) and then the counts of the earlier blocks (L2).
#include <algorithm>

#include "matmul_internal.h"
#include "qkv_common.cuh"
#include "qkv_internal.h"

namespace qkv {

namespace {

constexpr int kRouteThreads = 1024;
constexpr int kMaxBlockTokens = 1024;

__device__ __forceinline__ float load_logit(const void* p, long long i, int dtype) {
  if (dtype == QKV_F32) return ((const float*)p)[i];
  const uint16_t b = ((const uint16_t*)p)[i];
  return dtype == QKV_BF16 ? Elem<__nv_bfloat16>::bits_to_f32(b) : Elem<__half>::bits_to_f32(b);
}

// order-preserving key: a < b as floats <=> key(a) < key(b); -0 = +0, NaN above all
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One warp, one token: experts[0..k), weights[0..k). PER = logits per lane.
template <int PER>
__device__ __forceinline__ void route_token(const RouteArgs& a, int token, int lane) {
  float v[PER];
  uint32_t key[PER];
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < a.E ? load_logit(a.logits, (long long)token * a.E + e, a.dtype) : -INFINITY;
    key[i] = e < a.E ? order_key(v[i]) : 0u;  // 0: below every logit's key (-inf maps to 0x7fffff)
    mx = fmaxf(mx, v[i]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) total += v[i] == -INFINITY ? 0.f : expf(v[i] - mx);
#pragma unroll
  for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);

  int mine = 0;        // lane j < k keeps the j-th choice
  float p_mine = 0.f;
  for (int j = 0; j < a.k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = max(best, key[i]);
    best = __reduce_max_sync(0xffffffffu, best);
    unsigned at = 0xffffffffu;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i)
      if (key[i] == best) at = i * 32 + lane;
    at = __reduce_min_sync(0xffffffffu, at);
    float p = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if ((unsigned)(i * 32 + lane) == at) {
        p = v[i] == -INFINITY ? 0.f : expf(v[i] - mx);
        key[i] = 0u;
      }
    p = __shfl_sync(0xffffffffu, p, at & 31);
    if (lane == j) {
      mine = (int)at;
      p_mine = p;
    }
  }
  if (a.normalize) {
    total = lane < a.k ? p_mine : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane < a.k) {
    // total is 0 only for a row of -inf, whose weights are 0
    a.experts[(long long)token * a.k + lane] = mine;
    a.weights[(long long)token * a.k + lane] = total == 0.f ? 0.f : p_mine / total;
  }
}

__device__ __forceinline__ void route_block(const RouteArgs& a, int t0, int t1) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (a.E + 31) / 32;
  for (int t = t0 + warp; t < t1; t += kRouteThreads / 32) {
    if (per <= 1) route_token<1>(a, t, lane);
    else if (per <= 2) route_token<2>(a, t, lane);
    else if (per <= 4) route_token<4>(a, t, lane);
    else if (per <= 8) route_token<8>(a, t, lane);
    else route_token<16>(a, t, lane);
  }
}

// Exclusive prefix sum over E counts in shared memory, in place; returns nothing, total in
// count[E]. All threads of the block call it.
__device__ __forceinline__ void scan_counts(int* count, int E) {
  __shared__ int warp_sum[32];
  __shared__ int carry;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) carry = 0;
  __syncthreads();
  for (int e0 = 0; e0 < E; e0 += kRouteThreads) {
    const int e = e0 + threadIdx.x;
    const int n = e < E ? count[e] : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    if (lane == 31) warp_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      int s = warp_sum[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
      }
      warp_sum[lane] = s;
    }
    __syncthreads();
    if (e < E) count[e] = carry + sum - n + (warp ? warp_sum[warp - 1] : 0);
    __syncthreads();
    if (threadIdx.x == 0) carry += warp_sum[31];
    __syncthreads();
  }
  if (threadIdx.x == 0) count[E] = carry;
  __syncthreads();
}

// Choices of one block of tokens and its count per expert (several blocks: the first launch)
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs a, int bt) {
  extern __shared__ int smem[];
  const int t0 = blockIdx.x * bt, t1 = min(t0 + bt, a.T);
  for (int e = threadIdx.x; e < a.E; e += kRouteThreads) smem[e] = 0;
  route_block(a, t0, t1);
  __syncthreads();
  for (int i = threadIdx.x; i < (t1 - t0) * a.k; i += kRouteThreads)
    atomicAdd(&smem[a.experts[(long long)t0 * a.k + i]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kRouteThreads)
    a.hist[(long long)blockIdx.x * a.E + e] = smem[e];
}

// Sorted positions of one block's pairs. ONE: a single block that also chooses (a decode
// batch); otherwise the base of every expert is summed over the earlier blocks' counts.
template <bool ONE>
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a, int bt) {
  extern __shared__ int smem[];
  const int words = (bt + 31) / 32;
  int* base = smem;                                  // E + 1
  int* before = smem + a.E + 1;                      // E: pairs of earlier blocks
  uint32_t* mask = (uint32_t*)(smem + 2 * a.E + 1);  // words x E
  const int t0 = ONE ? 0 : blockIdx.x * bt, t1 = min(t0 + bt, a.T);
  for (int i = threadIdx.x; i < words * a.E; i += kRouteThreads) mask[i] = 0;
  if (ONE) {
    route_block(a, t0, t1);
  } else {
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) {
      int all = 0, prior = 0;
#pragma unroll 8
      for (int b = 0; b < gridDim.x; ++b) {
        const int n = a.hist[(long long)b * a.E + e];
        all += n;
        prior += b < blockIdx.x ? n : 0;
      }
      base[e] = all;
      before[e] = prior;
    }
  }
  __syncthreads();
  const int pairs = (t1 - t0) * a.k;
  const long long p0 = (long long)t0 * a.k;
  for (int i = threadIdx.x; i < pairs; i += kRouteThreads) {
    const int t = i / a.k;
    atomicOr(&mask[(t >> 5) * a.E + a.experts[p0 + i]], 1u << (t & 31));
  }
  __syncthreads();
  if (ONE) {
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) {
      int n = 0;
      for (int w = 0; w < words; ++w) n += __popc(mask[w * a.E + e]);
      base[e] = n;
      before[e] = 0;
    }
    __syncthreads();
  }
  scan_counts(base, a.E);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= a.E; e += kRouteThreads) a.offsets[e] = base[e];
  for (int i = threadIdx.x; i < pairs; i += kRouteThreads) {
    const int t = i / a.k, e = a.experts[p0 + i];
    int rank = before[e];
    for (int w = 0; w < (t >> 5); ++w) rank += __popc(mask[w * a.E + e]);
    rank += __popc(mask[(t >> 5) * a.E + e] & ((1u << (t & 31)) - 1));
    const int pos = base[e] + rank;
    a.slots[p0 + i] = pos;
    a.rows[pos] = t0 + t;
  }
}

// Tokens of a block: 64, growing past 256 blocks so that the sums over earlier blocks'
// counts stay short (they are read by every block).
int route_block_tokens(int T) {
  int bt = 64;
  while (bt < kMaxBlockTokens && (T + bt - 1) / bt > 256) bt *= 2;
  return bt;
}
// One block chooses and places a batch of up to this many tokens in one launch.
constexpr int kOneBlock = 64;

size_t place_smem(int E, int bt) { return (size_t)(2 * E + 1 + (bt + 31) / 32 * E) * sizeof(int); }

// out[t] = residual[t] + sum_j weights[t][j] * y[slots[t][j]], in fp32, j in order; a slot
// outside [0, R) adds nothing. VEC values per thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    expert_combine_kernel(const T* __restrict__ y, int R, const int* __restrict__ slots,
                          const float* __restrict__ weights, const T* __restrict__ residual,
                          T* __restrict__ out, long long n_vec, int per_row, int k, int N) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n_vec) return;
  const long long t = i / per_row;
  const int c = (int)(i - t * per_row) * VEC;
  float acc[VEC];
  auto add = [&](const T* p, float w) {
    if constexpr (VEC == 8) {
      const uint4 v = __ldg((const uint4*)p);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        acc[2 * q] = fmaf(w, Elem<T>::bits_to_f32((uint16_t)u[q]), acc[2 * q]);
        acc[2 * q + 1] = fmaf(w, Elem<T>::bits_to_f32((uint16_t)(u[q] >> 16)), acc[2 * q + 1]);
      }
    } else {
      acc[0] = fmaf(w, Elem<T>::to_f32(*p), acc[0]);
    }
  };
#pragma unroll
  for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
  for (int j = 0; j < k; ++j) {
    const int s = slots[t * k + j];
    if (s >= 0 && s < R) add(y + (long long)s * N + c, weights[t * k + j]);
  }
  if (residual) add(residual + t * N + c, 1.f);
  T* o = out + t * N + c;
#pragma unroll
  for (int q = 0; q < VEC; ++q) o[q] = Elem<T>::from_f32(acc[q]);
}

template <typename T>
int launch_combine_t(const void* y, int R, const int* slots, const float* weights,
                     const void* residual, void* out, int tokens, int k, int N, cudaStream_t st) {
  const bool vec = N % 8 == 0;
  const int per_row = vec ? N / 8 : N;
  const long long n = (long long)tokens * per_row;
  const long long blocks = (n + 255) / 256;
  if (blocks > 0x7fffffffll) return QKV_EUNSUPPORTED;
  if (vec)
    expert_combine_kernel<T, 8><<<(unsigned)blocks, 256, 0, st>>>(
        (const T*)y, R, slots, weights, (const T*)residual, (T*)out, n, per_row, k, N);
  else
    expert_combine_kernel<T, 1><<<(unsigned)blocks, 256, 0, st>>>(
        (const T*)y, R, slots, weights, (const T*)residual, (T*)out, n, per_row, k, N);
  return QKV_OK;
}

}  // namespace

size_t route_workspace_bytes(int T, int E) {
  if (T <= kOneBlock) return 0;
  const int bt = route_block_tokens(T);
  return (size_t)((T + bt - 1) / bt) * E * sizeof(int);
}

int launch_route(const RouteArgs& a, cudaStream_t st) {
  if (a.T <= kOneBlock) {
    route_place_kernel<true><<<1, kRouteThreads, place_smem(a.E, kOneBlock), st>>>(a, kOneBlock);
    return QKV_OK;
  }
  const int bt = route_block_tokens(a.T);
  const size_t smem = place_smem(a.E, bt);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(route_place_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)smem) != cudaSuccess)
    return QKV_ECUDA;
  const unsigned blocks = (unsigned)((a.T + bt - 1) / bt);
  route_choose_kernel<<<blocks, kRouteThreads, a.E * sizeof(int), st>>>(a, bt);
  route_place_kernel<false><<<blocks, kRouteThreads, smem, st>>>(a, bt);
  return QKV_OK;
}

int launch_expert_combine(const void* y, int R, const int* slots, const float* weights,
                          const void* residual, void* out, int T, int k, int N, int dtype,
                          cudaStream_t st) {
  if (dtype == QKV_BF16)
    return launch_combine_t<__nv_bfloat16>(y, R, slots, weights, residual, out, T, k, N, st);
  return launch_combine_t<__half>(y, R, slots, weights, residual, out, T, k, N, st);
}

}  // namespace qkv
