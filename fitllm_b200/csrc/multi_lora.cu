// Low-rank adapters of many requests beside a shared projection:
//   y[n] = y_add[n] + s_l (x[n].A_l^T).B_l^T,   l = adapter of token n's sequence.
// Two kernels: T = x.A_l^T in fp32 (a CTA per token), then y (a thread per output).
#include "kernels.cuh"
#include "kv4.cuh"

namespace fitq {
namespace {

constexpr int kThreads = 128;

struct MultiLoraParams {
  const void *x, *a, *b, *y_add;
  void* y;
  const float* scale;
  const int32_t* adapter;
  const int32_t* q_start;
  int64_t tokens, x_stride, y_add_stride;
  int batch, adapters, k, n, rank, t_new;
  float* t;
  int* status;
};

// Adapter of token n, -1 for none, -2 for a token of no sequence.
__device__ __forceinline__ int adapter_of(const MultiLoraParams& p, int64_t n, bool* bad) {
  Kv4Seq s{};
  s.q_start = p.q_start;
  s.batch = p.batch;
  s.t_new = p.t_new;
  const int b = kv4_sequence(s, n);
  if (b < 0) return -2;
  const int l = p.adapter[b];
  if (l >= -1 && l < p.adapters) return l;
  *bad = true;
  return -1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) multi_lora_shrink_kernel(const MultiLoraParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t n = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool bad = false;
  const int l = adapter_of(p, n, &bad);
  if (bad && threadIdx.x == 0) report_device_error(p.status, FITQ_ERR_ARG);
  if (l < 0) return;
  const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + n * p.x_stride);
  for (int r = warp; r < p.rank; r += kThreads / 32) {
    const uint4* a = reinterpret_cast<const uint4*>(static_cast<const T*>(p.a) + (static_cast<int64_t>(l) * p.rank + r) * p.k);
    float s = 0.f;
    for (int c = lane; c < p.k / 8; c += 32) {
      float f[8], g[8];
      unpack8<T>(x[c], f);
      unpack8<T>(a[c], g);
      for (int i = 0; i < 8; ++i) s = fmaf(f[i], g[i], s);
    }
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) p.t[n * p.rank + r] = s;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) multi_lora_expand_kernel(const MultiLoraParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t n = blockIdx.x;
  const int col = blockIdx.y * kThreads + threadIdx.x;
  if (col >= p.n) return;
  bool bad = false;
  const int l = adapter_of(p, n, &bad);
  if (l == -2) return;
  const T y = static_cast<const T*>(p.y_add)[n * p.y_add_stride + col];
  T* dst = static_cast<T*>(p.y) + n * p.n + col;
  if (l < 0) {
    *dst = y;
    return;
  }
  const T* b = static_cast<const T*>(p.b) + (static_cast<int64_t>(l) * p.n + col) * p.rank;
  float s = 0.f;
  for (int r = 0; r < p.rank; ++r) s = fmaf(p.t[n * p.rank + r], static_cast<float>(b[r]), s);
  *dst = static_cast<T>(fmaf(p.scale[l], s, static_cast<float>(y)));
}

}  // namespace

size_t multi_lora_workspace(int64_t tokens, int64_t, int64_t, int rank, int, int) {
  return static_cast<size_t>(tokens) * rank * sizeof(float);
}

int launch_multi_lora(const void* x, int64_t x_stride, int64_t tokens, int64_t k, int64_t n, const void* a,
                      const void* b, int rank, int adapters, const float* scale, const int32_t* adapter,
                      const int32_t* q_start, int batch, const void* y_add, int64_t y_add_stride, void* y, int dtype,
                      void* workspace, int* status, cudaStream_t st, int) {
  const MultiLoraParams p{x, a, b, y_add, y, scale, adapter, q_start, tokens, x_stride, y_add_stride, batch, adapters,
                          static_cast<int>(k), static_cast<int>(n), rank,
                          q_start ? 0 : static_cast<int>(tokens / batch), static_cast<float*>(workspace), status};
  const bool bf = dtype == FITQ_DTYPE_BF16;
  cudaError_t e = launch_pdl(bf ? multi_lora_shrink_kernel<__nv_bfloat16> : multi_lora_shrink_kernel<__half>,
                             dim3(static_cast<unsigned>(tokens)), dim3(kThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  e = launch_pdl(bf ? multi_lora_expand_kernel<__nv_bfloat16> : multi_lora_expand_kernel<__half>,
                 dim3(static_cast<unsigned>(tokens), static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace fitq
