// Launch interface of the 4-bit weight products (qkv_matmul.cu, qkv_matmul_tc.cu) and of the
// expert routing around them (qkv_experts.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

namespace qkv {

// One product y[r] = act(x[rows[r]] W_e^T) over the rows r of every expert e
// (offsets[e] <= r < offsets[e+1]); without offsets one weight matrix and all R rows.
struct MatmulArgs {
  const void* x;       // (x_rows, K) in dtype, ldx elements between rows
  long long ldx;
  int x_rows;          // rows of x; an entry of `rows` outside [0, x_rows) reads as zeros
  const int* rows;     // device int32[R] or nullptr (row r of y comes from row r of x)
  const int* offsets;  // device int32[E + 1] or nullptr
  const void* w;       // codes (E, N, K/8) uint32
  const void* scales;  // (E, N, K/64) in dtype
  const void* biases;
  void* out;           // (R, N) in dtype, (R, N/2) with the gated activation
  int R, E, N, K;
  int dtype;           // QKV_BF16 / QKV_F16
  int act;             // QKV_ACT_NONE / QKV_ACT_SWIGLU
  void* workspace;
  size_t ws_bytes;
  int* status;         // device status word for bounded-wait failures
};

int launch_matmul_rows(const MatmulArgs& a, cudaStream_t st);  // few rows per weight matrix
int launch_matmul_tc(const MatmulArgs& a, cudaStream_t st);    // many (tcgen05)
bool matmul_tc_fits(int E, int N);  // whether the tcgen05 kernel takes the stacked weights
size_t matmul_tc_workspace(int R, int K);  // when it gathers rows of x
int launch_matmul(const MatmulArgs& a, cudaStream_t st);       // whichever is faster
bool matmul_takes_tc(int R, int E, int N, int K);

struct RouteArgs {
  const void* logits;  // (T, E) in dtype
  int dtype, T, E, k, normalize;
  int* experts;        // (T, k)
  float* weights;      // (T, k)
  int* rows;           // (T * k) token of each sorted pair
  int* slots;          // (T, k) sorted position of each pair
  int* offsets;        // (E + 1)
  int* hist;           // workspace: (blocks, (E + 1) / 2) pairs of 16-bit counts
};

size_t route_workspace_bytes(int T, int E);
int launch_route(const RouteArgs& a, cudaStream_t st);
int launch_expert_combine(const void* y, int R, const int* slots, const float* weights,
                          const void* residual, void* out, int T, int k, int N, int dtype,
                          cudaStream_t st);

// Launch a kernel that waits for the one before it by itself. early: it may be set up while the one
// before it in the stream still runs. Not after a kernel of many small blocks: blocks set up
// early take their places (gather and product of 16384 expert rows 159 us with, 148 without;
// choosing and placing of 8192 tokens 29.0 with, 22.9 without).
template <typename... P, typename... A>
int launch(bool early, void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem,
           cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess ? 0 : -3;  // QKV_ECUDA
}

#ifdef __CUDACC__
// Waits for the kernel before, and only then lets the next one be set up: the
// attention kernel reads older cache positions ahead of its own wait, counting on the kernel
// just before it alone to be unfinished.
__device__ __forceinline__ void wait_for_kernel_before() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void allow_next_kernel() {
  asm volatile("griddepcontrol.launch_dependents;");
}
__device__ __forceinline__ void wait_for_previous() {
  wait_for_kernel_before();
  allow_next_kernel();
}
#endif

}  // namespace qkv
