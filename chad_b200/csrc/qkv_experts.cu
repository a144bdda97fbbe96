// Routing of tokens to experts, and the weighted sum of the experts' rows (sm_100a).
//
// Route: the k largest of E logits per token (ties to the lowest expert, NaN counts as the
// largest), softmax weights over all logits or over the chosen ones, and the stable counting
// sort of the T*k pairs by expert: rows (token of each sorted pair), slots (sorted position
// of each pair) and offsets (first sorted pair of each expert).
//
// One warp per token holds its logits in registers as order-preserving unsigned keys.
// A token takes an expert at most once, so a pair's rank within its expert is the number of
// earlier tokens that took it: a popcount over a per-expert bit mask of tokens. Counts and
// masks are integers, so the order of their atomics does not show.
//
// What bounds it: a decode batch is one block's latency (16 tokens of 128 experts 4.5 us); a
// long chunk reads the logits once (HBM) and then the counts of the earlier blocks (L2), and is
// bound by the chains of warp reductions of a token's choice (8192 tokens of 256 experts in fp32
// 18.5 us, two thirds of it the choices; the 8.4 MB of logits take 1.3).
#include <algorithm>
#include <atomic>

#include "matmul_internal.h"
#include "qkv_common.cuh"
#include "qkv_internal.h"

namespace qkv {

namespace {

constexpr int kRouteThreads = 1024;   // of a block that places
constexpr int kChooseThreads = 512;   // of a block that chooses: two fit an SM
constexpr int kPlaceBlocks = 4;       // choosing blocks whose pairs one block places
constexpr int kMaxBlockTokens = 512;
constexpr int kMaxRouteExperts = 512;

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

// One warp, one token: experts[0..k), weights[0..k). PER = logits per lane.
//
// The k-th largest of the lanes' best keys is a lower bound of the k-th largest key, found by
// redux.max over one key per lane. What reaches it, a few more than k keys, goes to shared
// memory in the experts' order, one to a lane, where its rank is the number of those before it:
// compares that do not wait for one another. (Choosing one after the other among all keys, each
// time with a new best for the lane it came from, took 17.5 us for 8192 tokens of 256 experts.)
// Keys in such numbers that 32 lanes do not hold them are chosen one after the other.
template <int DTYPE, int PER>
__device__ __forceinline__ void route_token(const RouteArgs& a, int token, int lane, uint2* held) {
  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    // 0 is below every logit's key (-inf has 0x7fffff)
    key[i] = e < a.E ? order_key(load_logit<DTYPE>(a.logits, (long long)token * a.E + e)) : 0u;
  }
  uint32_t best = key[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) best = max(best, key[i]);
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
  // (at least min(E, 32) >= k lanes have a key, so the bound is a key)
  uint32_t bound = top;
  for (int n = 0;;) {
    n += __popc(__ballot_sync(0xffffffffu, best == bound));
    if (n >= a.k) break;
    best = best == bound ? 0u : best;
    bound = __reduce_max_sync(0xffffffffu, best);
  }
  int count = 0;
  __syncwarp();  // (the token before has been read)
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const bool in = key[i] >= bound;
    const uint32_t m = __ballot_sync(0xffffffffu, in);
    const int at = count + __popc(m & ((1u << lane) - 1));
    if (in && at < 32) held[at] = make_uint2(key[i], i * 32 + lane);
    count += __popc(m);
  }
  __syncwarp();
  uint32_t chosen = 0, at = 0;  // key and expert of this lane, and where it stands
  int rank = 32;
  if (count <= 32) {
    if (lane < count) {
      const uint2 c = held[lane];
      chosen = c.x;
      at = c.y;
      rank = 0;
    }
#pragma unroll 4
    for (int c = 0; c < count; ++c) {
      const uint32_t other = __shfl_sync(0xffffffffu, chosen, c);
      rank += other > chosen || (other == chosen && c < lane);
    }
  } else {
#pragma unroll 1
    for (int j = 0; j < a.k; ++j) {
      uint32_t b = 0;
      int b_i = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] > b) {
          b = key[i];
          b_i = i;
        }
      const uint32_t high = __reduce_max_sync(0xffffffffu, b);
      const uint32_t mine = b == high ? b_i * 32u + lane : ~0u;
      const uint32_t e = __reduce_min_sync(0xffffffffu, mine);
      if (lane == j) {
        at = e;
        chosen = high;
        rank = j;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = e == mine && i == b_i ? 0u : key[i];
    }
  }
  const float v = key_value(chosen);
  const float p = rank >= a.k || v == -INFINITY ? 0.f : expf(v - mx);
  if (a.normalize) {
    total = p;
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  if (rank < a.k) {
    // total is 0 only for a row of -inf, whose weights are 0
    a.experts[(long long)token * a.k + rank] = (int)at;
    a.weights[(long long)token * a.k + rank] = total == 0.f ? 0.f : p / total;
  }
}

template <int DTYPE, int THREADS>
__device__ __forceinline__ void route_block(const RouteArgs& a, int t0, int t1) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (a.E + 31) / 32;
  __shared__ uint2 held_of[THREADS / 32][32];
  uint2* held = held_of[warp];
  for (int t = t0 + warp; t < t1; t += THREADS / 32) {
    if (per <= 1) route_token<DTYPE, 1>(a, t, lane, held);
    else if (per <= 2) route_token<DTYPE, 2>(a, t, lane, held);
    else if (per <= 4) route_token<DTYPE, 4>(a, t, lane, held);
    else if (per <= 8) route_token<DTYPE, 8>(a, t, lane, held);
    else route_token<DTYPE, 16>(a, t, lane, held);
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
  // (a block's count fits 16 bits: every placing block reads all of them)
  const int words = (a.E + 1) / 2;
  for (int i = threadIdx.x; i < words; i += kChooseThreads)
    a.hist[(long long)blockIdx.x * words + i] =
        smem[2 * i] | (2 * i + 1 < a.E ? smem[2 * i + 1] << 16 : 0);
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
    // (words of two counts)
    const int width = (a.E + 1) / 2, lanes = (width + 31) / 32 * 32, share = kRouteThreads / lanes;
    const int w = threadIdx.x % lanes, part = threadIdx.x / lanes;
    if (part < share && w < width) {
      int all[2] = {0, 0}, prior[2] = {0, 0};
      const int mine = blockIdx.x * kPlaceBlocks;
      for (int b0 = part; b0 < counted; b0 += 16 * share) {
        uint32_t n[16];  // sixteen loads in flight
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int b = b0 + i * share;
          n[i] = b < counted ? __ldg((const uint32_t*)a.hist + (long long)b * width + w) : 0;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int lo = n[i] & 0xffff, hi = n[i] >> 16;
          const bool before_mine = b0 + i * share < mine;
          all[0] += lo;
          all[1] += hi;
          prior[0] += before_mine ? lo : 0;
          prior[1] += before_mine ? hi : 0;
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (2 * w + q < a.E) {
          atomicAdd(&base[2 * w + q], all[q]);
          atomicAdd(&before[2 * w + q], prior[q]);
        }
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

// Bound by HBM: 2048 tokens of 8 rows of 2048 with a residual 19.5 us, 4.3 of 6.6 TB/s; the rows
// come in the order of the experts, 4 KB at a time.
//
// out[t] = residual[t] + sum_j weights[t][j] * y[slots[t][j]], in fp32, j in order; a slot
// outside [0, R) adds nothing. VEC values per thread. The result may be the residual: a thread
// reads its own values before it writes them, and nothing promises that the two are apart.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    expert_combine_kernel(const T* __restrict__ y, int R, const int* __restrict__ slots,
                          const float* __restrict__ weights, const T* residual, T* out,
                          long long n_vec, int per_row, int k, int N) {
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
  // (an ordinary load: the residual may be the result, which other threads are writing)
  uint4 res = zero;
  if (residual) {
    if constexpr (VEC == 8) res = *(const uint4*)(residual + t * N + c);
    else res.x = *(const uint16_t*)(residual + t * N + c);
  }
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
  const bool vec = N % 8 == 0;  // (y, residual and out are then 16-byte aligned)
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
  return (size_t)((T + bt - 1) / bt) * ((E + 1) / 2) * sizeof(int);
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
  // Set on a device's first call, whatever its sizes: the bound that holds without it counts the
  // kernel's static bytes as well.
  static std::atomic<unsigned long long> ready{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return QKV_ECUDA;
  if (dev < 0 || dev >= kMaxDevices || !(ready.load() >> dev & 1)) {
    if (cudaFuncSetAttribute(route_place_kernel<false, QKV_F32>,
                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)place_smem(kMaxRouteExperts, kMaxBlockTokens * kPlaceBlocks)) !=
        cudaSuccess)
      return QKV_ECUDA;
    if (dev >= 0 && dev < kMaxDevices) ready.fetch_or(1ull << dev);
  }
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
