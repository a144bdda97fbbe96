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

constexpr int kRouteThreads = 1024;   // of a block that places
constexpr int kChooseThreads = 512;   // of a block that chooses: two fit an SM
constexpr int kPlaceBlocks = 4;       // choosing blocks whose pairs one block places
constexpr int kMaxBlockTokens = 512;

template <int DTYPE>
__device__ __forceinline__ float load_logit(const void* p, long long i) {
  if (DTYPE == QKV_F32) return __ldg((const float*)p + i);
  const uint16_t b = __ldg((const uint16_t*)p + i);
  return DTYPE == QKV_BF16 ? Elem<__nv_bfloat16>::bits_to_f32(b) : Elem<__half>::bits_to_f32(b);
}

// order-preserving key: a < b as floats <=> key(a) < key(b); -0 = +0, NaN above all
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The value of a key (NaN for the NaN key).
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

// One warp, one token: experts[0..k), weights[0..k). PER = logits per lane. Every lane keeps the
// best of its own logits; a choice is a redux.max over the lanes' best keys, a redux.min over
// the indices that have it, and a new best for the lane it came from. The first choice is the
// softmax's maximum.
template <int DTYPE, int PER>
__device__ __forceinline__ void route_token(const RouteArgs& a, int token, int lane) {
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    // 0 is below every logit's key (-inf has 0x7fffff)
    key[i] = e < a.E ? order_key(load_logit<DTYPE>(a.logits, (long long)token * a.E + e)) : 0u;
  }
  uint32_t best;
  int best_i;
  auto find_best = [&]() {
    best = key[0];
    best_i = 0;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        best_i = i;
      }
  };
  find_best();
  const uint32_t top = __reduce_max_sync(0xffffffffu, best);
  const float mx = key_value(top);
  float total = 0.f;
  if (!a.normalize) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float v = key_value(key[i]);
      if (key[i] != 0u && v != -INFINITY) total += expf(v - mx);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  uint32_t at = 0, chosen = 0;  // lane j < k keeps the j-th choice
#pragma unroll 1
  for (int j = 0; j < a.k; ++j) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, best);
    const uint32_t mine = best == high ? best_i * 32u + lane : ~0u;
    const uint32_t e = __reduce_min_sync(0xffffffffu, mine);
    if (lane == j) {
      at = e;
      chosen = high;
    }
    // without a branch: the lane of the choice drops it and finds its next best
    const int drop = e == mine ? best_i : -1;
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = i == drop ? 0u : key[i];
    find_best();
  }
  const float v = key_value(chosen);
  const float p = lane >= a.k || v == -INFINITY ? 0.f : expf(v - mx);
  if (a.normalize) {
    total = p;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (lane < a.k) {
    // total is 0 only for a row of -inf, whose weights are 0
    a.experts[(long long)token * a.k + lane] = (int)at;
    a.weights[(long long)token * a.k + lane] = total == 0.f ? 0.f : p / total;
  }
}

template <int DTYPE, int THREADS>
__device__ __forceinline__ void route_block(const RouteArgs& a, int t0, int t1) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (a.E + 31) / 32;
  for (int t = t0 + warp; t < t1; t += THREADS / 32) {
    if (per <= 1) route_token<DTYPE, 1>(a, t, lane);
    else if (per <= 2) route_token<DTYPE, 2>(a, t, lane);
    else if (per <= 4) route_token<DTYPE, 4>(a, t, lane);
    else if (per <= 8) route_token<DTYPE, 8>(a, t, lane);
    else route_token<DTYPE, 16>(a, t, lane);
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
template <int DTYPE>
__global__ void __launch_bounds__(kChooseThreads, 2) route_choose_kernel(const RouteArgs a, int bt) {
  extern __shared__ int smem[];
  const int t0 = blockIdx.x * bt, t1 = min(t0 + bt, a.T);
  wait_for_previous();
  for (int e = threadIdx.x; e < a.E; e += kChooseThreads) smem[e] = 0;
  route_block<DTYPE, kChooseThreads>(a, t0, t1);
  __syncthreads();
  for (int i = threadIdx.x; i < (t1 - t0) * a.k; i += kChooseThreads)
    atomicAdd(&smem[a.experts[(long long)t0 * a.k + i]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kChooseThreads)
    a.hist[(long long)blockIdx.x * a.E + e] = smem[e];
}

// Sorted positions of one block's pairs. ONE: a single block that also chooses (a decode
// batch); otherwise the base of every expert is summed over the earlier blocks' counts.
template <bool ONE, int DTYPE>
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a, int bt,
                                                                      int counted) {
  extern __shared__ int smem[];
  const int words = (bt + 31) / 32;
  int* base = smem;                                  // E + 1
  int* before = smem + a.E + 1;                      // E: pairs of earlier blocks
  uint32_t* mask = (uint32_t*)(smem + 2 * a.E + 1);  // words x E
  const int t0 = ONE ? 0 : blockIdx.x * bt, t1 = min(t0 + bt, a.T);
  for (int i = threadIdx.x; i < words * a.E; i += kRouteThreads) mask[i] = 0;
  wait_for_previous();
  if (ONE) {
    route_block<DTYPE, kRouteThreads>(a, t0, t1);
  } else {
    // the block's threads share the rows of counts of every expert
    for (int e = threadIdx.x; e < a.E; e += kRouteThreads) base[e] = before[e] = 0;
    __syncthreads();
    const int lanes = (a.E + 31) / 32 * 32, share = kRouteThreads / lanes;
    const int e = threadIdx.x % lanes, part = threadIdx.x / lanes;
    if (part < share && e < a.E) {
      int all = 0, prior = 0;
      const int mine = blockIdx.x * kPlaceBlocks;
      for (int b0 = part; b0 < counted; b0 += 16 * share) {
        int n[16];  // sixteen loads in flight
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int b = b0 + i * share;
          n[i] = b < counted ? __ldg(a.hist + (long long)b * a.E + e) : 0;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          all += n[i];
          prior += b0 + i * share < mine ? n[i] : 0;
        }
      }
      atomicAdd(&base[e], all);
      atomicAdd(&before[e], prior);
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

// Tokens of a choosing block: 32, growing past 256 blocks so that the sums over earlier blocks'
// counts stay short (they are read by every block).
int route_block_tokens(int T) {
  int bt = 32;
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
  wait_for_previous();
  if (i >= n_vec) return;
  const long long t = i / per_row;
  const int c = (int)(i - t * per_row) * VEC;
  float acc[VEC];
  auto add = [&](const uint4& v, float w) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    if constexpr (VEC == 8) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        acc[2 * q] = fmaf(w, Elem<T>::bits_to_f32((uint16_t)u[q]), acc[2 * q]);
        acc[2 * q + 1] = fmaf(w, Elem<T>::bits_to_f32((uint16_t)(u[q] >> 16)), acc[2 * q + 1]);
      }
    } else {
      acc[0] = fmaf(w, Elem<T>::bits_to_f32((uint16_t)u[0]), acc[0]);
    }
  };
  auto get = [&](const T* p) -> uint4 {
    if constexpr (VEC == 8) return __ldg((const uint4*)p);
    return make_uint4(__ldg((const uint16_t*)p), 0, 0, 0);
  };
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const uint4 res = residual ? get(residual + t * N + c) : zero;
#pragma unroll
  for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
  // eight rows in flight at a time
  for (int j0 = 0; j0 < k; j0 += 8) {
    float w[8];
    uint4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool in = j0 + j < k;
      const int s = in ? __ldg(slots + t * k + j0 + j) : -1;
      const bool held = s >= 0 && s < R;  // (a dropped pair's weight may be anything)
      w[j] = held ? __ldg(weights + t * k + j0 + j) : 0.f;
      v[j] = held ? get(y + (long long)s * N + c) : zero;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) add(v[j], w[j]);
  }
  add(res, residual ? 1.f : 0.f);
  T* o = out + t * N + c;
  if constexpr (VEC == 8) {
    alignas(16) T r[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) r[q] = Elem<T>::from_f32(acc[q]);
    *(uint4*)o = *(const uint4*)r;
  } else {
    o[0] = Elem<T>::from_f32(acc[0]);
  }
}

template <typename T>
int launch_combine_t(const void* y, int R, const int* slots, const float* weights,
                     const void* residual, void* out, int tokens, int k, int N, cudaStream_t st) {
  const bool vec = N % 8 == 0;
  const int per_row = vec ? N / 8 : N;
  const long long n = (long long)tokens * per_row;
  const long long blocks = (n + 255) / 256;
  if (blocks > 0x7fffffffll) return QKV_EUNSUPPORTED;
  return launch(true, vec ? expert_combine_kernel<T, 8> : expert_combine_kernel<T, 1>,
                          dim3((unsigned)blocks), 256, 0, st, y, R, slots, weights, residual, out, n,
                          per_row, k, N);
}

}  // namespace

size_t route_workspace_bytes(int T, int E) {
  if (T <= kOneBlock) return 0;
  const int bt = route_block_tokens(T);
  return (size_t)((T + bt - 1) / bt) * E * sizeof(int);
}

template <int DTYPE>
static int launch_route_t(const RouteArgs& a, cudaStream_t st) {
  if (a.T <= kOneBlock) {
    return launch(true, route_place_kernel<true, DTYPE>, dim3(1), kRouteThreads,
                            place_smem(a.E, kOneBlock), st, a, kOneBlock, 0);
  }
  const int bt = route_block_tokens(a.T), place = bt * kPlaceBlocks;
  const unsigned blocks = (unsigned)((a.T + bt - 1) / bt);
  const size_t smem = place_smem(a.E, place);
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(route_place_kernel<false, QKV_F32>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return QKV_ECUDA;
  const int rc = launch(true, route_choose_kernel<DTYPE>, dim3(blocks), kChooseThreads,
                                  a.E * sizeof(int), st, a, bt);
  if (rc) return rc;
  return launch(false, route_place_kernel<false, QKV_F32>,
                          dim3((blocks + kPlaceBlocks - 1) / kPlaceBlocks), kRouteThreads, smem, st,
                          a, place, (int)blocks);
}

int launch_route(const RouteArgs& a, cudaStream_t st) {
  if (a.dtype == QKV_BF16) return launch_route_t<QKV_BF16>(a, st);
  if (a.dtype == QKV_F16) return launch_route_t<QKV_F16>(a, st);
  return launch_route_t<QKV_F32>(a, st);
}

int launch_expert_combine(const void* y, int R, const int* slots, const float* weights,
                          const void* residual, void* out, int T, int k, int N, int dtype,
                          cudaStream_t st) {
  if (dtype == QKV_BF16)
    return launch_combine_t<__nv_bfloat16>(y, R, slots, weights, residual, out, T, k, N, st);
  return launch_combine_t<__half>(y, R, slots, weights, residual, out, T, k, N, st);
}

}  // namespace qkv
