// Attention of a tree of drafted tokens over a 16-bit key/value cache.
//
// For token i of sequence b and head h on KV head h / group, with s_j = q.k_j / sqrt(D)
// over the cached positions and the ancestors of i (and i):
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max s_j.
// One pass with a running maximum; a CTA per (token, head), 128 positions at a time.
#include "kernels.cuh"
#include "tree.cuh"

namespace fitq {
namespace {

constexpr int kThreads = 128;

struct TreeAttnParams {
  TreeView tree;
  const void *q, *k_cache, *v_cache;
  void* out;
  int64_t q_stride;
  int heads, group;
  float scale;
  int* status;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads) tree_attn_kernel(const TreeAttnParams p) {
  __shared__ int up[kTreeTokens];
  __shared__ float sq[D], sw[kThreads], red[kThreads];
  pdl_launch_dependents();
  pdl_wait();
  const TreeView& t = p.tree;
  const int b = blockIdx.x / t.tokens, i = blockIdx.x % t.tokens, h = blockIdx.y, tid = threadIdx.x;
  if (tid <= i) {
    bool bad = false;
    up[tid] = tree_parent(t, b, tid, &bad);
    if (bad && tid == i && h == 0) report_device_error(p.status, FITQ_ERR_ARG);
  }
  const int64_t n = static_cast<int64_t>(b) * t.tokens + i;
  if (tid < D / 8) {
    float f[8];
    unpack8<T>(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + n * p.q_stride + h * D)[tid], f);
    for (int x = 0; x < 8; ++x) sq[8 * tid + x] = f[x];
  }
  __syncthreads();
  const int64_t pre = t.prefix[b];
  uint64_t seen;
  int depth;
  bool here = tree_walk(up, i, &seen, &depth);
  if (here && (pre < 0 || pre + i >= t.capacity)) {
    if (tid == 0 && h == 0) report_device_error(p.status, FITQ_ERR_ARG);
    here = false;
  }
  const int64_t len = here ? pre + i + 1 : 0;
  const int64_t base = b * t.stride_b + (h / p.group) * t.stride_h;
  const T* kc = static_cast<const T*>(p.k_cache) + base;
  const T* vc = static_cast<const T*>(p.v_cache) + base;
  float m = -INFINITY, l = 0.f, acc = 0.f;  // acc: element tid of the output
  for (int64_t at = 0; at < len; at += kThreads) {
    const int64_t pos = at + tid;
    const bool vis = pos < pre || (pos < len && ((seen >> (pos - pre)) & 1ull));
    float s = -INFINITY;
    if (vis) {
      s = 0.f;
      for (int c = 0; c < D / 8; ++c) {
        float f[8];
        unpack8<T>(reinterpret_cast<const uint4*>(kc + pos * t.stride_p)[c], f);
        for (int x = 0; x < 8; ++x) s = fmaf(f[x], sq[8 * c + x], s);
      }
      s *= p.scale;
    }
    red[tid] = s;
    __syncthreads();
    float top = m;
    for (int x = 0; x < kThreads; ++x) top = fmaxf(top, red[x]);
    const float w = vis ? __expf(s - top) : 0.f;
    sw[tid] = w;
    __syncthreads();
    const float keep = m == -INFINITY ? 0.f : __expf(m - top);
    float sum = 0.f;
    acc *= keep;
    for (int x = 0; x < kThreads && at + x < len; ++x) {
      const float wx = sw[x];
      const bool vx = at + x < pre || ((seen >> (at + x - pre)) & 1ull);
      if (!vx) continue;
      sum += wx;
      if (tid < D) acc = fmaf(wx, static_cast<float>(vc[(at + x) * t.stride_p + tid]), acc);
    }
    l = l * keep + sum;
    m = top;
    __syncthreads();
  }
  if (tid < D) static_cast<T*>(p.out)[(n * p.heads + h) * D + tid] = static_cast<T>(l == 0.f ? 0.f : acc / l);
}

}  // namespace

size_t tree_attention_workspace(const TreeView&, int, int, int) { return 16; }

int launch_tree_attention(const TreeView& tree, const void* q, int64_t q_stride, const void* k_cache,
                          const void* v_cache, void* out, int heads, int dim, int dtype, void*, int* status,
                          cudaStream_t st, int) {
  const TreeAttnParams p{tree, q, k_cache, v_cache, out, q_stride, heads, heads / tree.kv_heads,
                         1.f / sqrtf(static_cast<float>(dim)), status};
  auto* kernel = dtype == FITQ_DTYPE_BF16
                     ? (dim == 128 ? tree_attn_kernel<__nv_bfloat16, 128> : tree_attn_kernel<__nv_bfloat16, 64>)
                     : (dim == 128 ? tree_attn_kernel<__half, 128> : tree_attn_kernel<__half, 64>);
  const cudaError_t e = launch_pdl(kernel, dim3(static_cast<unsigned>(tree.batch) * tree.tokens, heads), dim3(kThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace fitq
