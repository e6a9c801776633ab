// A tree of drafted tokens enters the key/value cache, and the accepted path stays.
//
// tree_append_kernel: queries and keys of token i rotated at position prefix + depth(i)
// (rotate-half: a' = a c - b s, b' = b c + a s, in fp32, rounded once), keys and values
// written to slot prefix + i.  A CTA takes one token: its position is one walk to the root,
// by one thread, and its threads take 16-byte pieces of the heads.
// Bound: latency for few tokens (a launch and the chain parents, walk, tables: 2.5 us), HBM for many (2 B in
// and out per element): 64 trees of up to 16 tokens of 40 + 2 x 8 heads of 128, 6.5 us, 2.7 TB/s.
//
// tree_keep_kernel: slot prefix + path[i] moves to prefix + i for the accepted tokens, in
// every layer.  path ascends and path[i] >= i, so a thread that owns an element column and
// copies in order of i never overwrites what it still has to read.  The lengths follow in a launch of
// their own (1 us), as they may be written over the old ones.
#include "kernels.cuh"
#include "tree.cuh"

namespace fitq {
namespace {

constexpr int kAppendThreads = 256;

struct TreeAppendParams {
  TreeView tree;
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  void *q_out, *k_cache, *v_cache;
  const float *cs, *sn;
  int rope_len, heads, dim;
  int* status;
};

template <typename T>
__global__ void __launch_bounds__(kAppendThreads) tree_append_kernel(const TreeAppendParams p) {
  __shared__ int up[kTreeTokens];
  __shared__ int sh_pos;   // rotary position, -1: no token
  pdl_launch_dependents();
  pdl_wait();
  const TreeView& t = p.tree;
  const int b = blockIdx.x / t.tokens, i = blockIdx.x % t.tokens;
  if (threadIdx.x <= i) {
    bool bad = false;
    up[threadIdx.x] = tree_parent(t, b, threadIdx.x, &bad);
    if (bad && threadIdx.x == i) report_device_error(p.status, FITQ_ERR_ARG);
  }
  __syncthreads();
  const int64_t pre = t.prefix[b];
  if (threadIdx.x == 0) {
    uint64_t seen;
    int depth;
    sh_pos = -1;
    if (tree_walk(up, i, &seen, &depth)) {
      if (pre < 0 || pre + i >= t.capacity || pre + depth >= p.rope_len)
        report_device_error(p.status, FITQ_ERR_ARG);
      else
        sh_pos = static_cast<int>(pre) + depth;
    }
  }
  __syncthreads();
  const int pos = sh_pos;
  const int half = p.dim / 2, per = half / 8;  // 16-byte pieces of half a head
  const int64_t n = static_cast<int64_t>(b) * t.tokens + i;
  const T* q = static_cast<const T*>(p.q) + n * p.q_stride;
  const T* k = static_cast<const T*>(p.k) + n * p.k_stride;
  const T* v = static_cast<const T*>(p.v) + n * p.v_stride;
  T* q_out = static_cast<T*>(p.q_out) + n * p.heads * p.dim;
  if (pos < 0) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int e = threadIdx.x; e < p.heads * p.dim / 8; e += kAppendThreads) reinterpret_cast<uint4*>(q_out)[e] = zero;
    return;
  }
  const int64_t slot = b * t.stride_b + (pre + i) * t.stride_p;
  T* kc = static_cast<T*>(p.k_cache) + slot;
  T* vc = static_cast<T*>(p.v_cache) + slot;
  const float* cs = p.cs + static_cast<int64_t>(pos) * half;
  const float* sn = p.sn + static_cast<int64_t>(pos) * half;
  const int turns = (p.heads + t.kv_heads) * per;
  for (int e = threadIdx.x; e < turns + t.kv_heads * 2 * per; e += kAppendThreads) {
    if (e >= turns) {  // values
      const int c = e - turns, h = c / (2 * per), o = (c % (2 * per)) * 8;
      *reinterpret_cast<uint4*>(vc + h * t.stride_h + o) = *reinterpret_cast<const uint4*>(v + h * p.dim + o);
      continue;
    }
    const int h = e / per, o = (e % per) * 8;
    const bool is_q = h < p.heads;
    const T* src = is_q ? q + h * p.dim + o : k + (h - p.heads) * p.dim + o;
    T* dst = is_q ? q_out + h * p.dim + o : kc + (h - p.heads) * t.stride_h + o;
    float x[8], y[8], c[8], s[8], r0[8], r1[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(src), x);
    unpack8<T>(*reinterpret_cast<const uint4*>(src + half), y);
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      *reinterpret_cast<float4*>(c + j) = __ldg(reinterpret_cast<const float4*>(cs + o + j));
      *reinterpret_cast<float4*>(s + j) = __ldg(reinterpret_cast<const float4*>(sn + o + j));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r0[j] = __fsub_rn(__fmul_rn(x[j], c[j]), __fmul_rn(y[j], s[j]));
      r1[j] = __fadd_rn(__fmul_rn(y[j], c[j]), __fmul_rn(x[j], s[j]));
    }
    *reinterpret_cast<uint4*>(dst) = pack8<T>(r0);
    *reinterpret_cast<uint4*>(dst + half) = pack8<T>(r1);
  }
}

constexpr int kKeepLayers = 64;  // layers of a launch: their pointers are kernel arguments
constexpr int kKeepThreads = 256;

struct TreeKeepParams {
  TreeView tree;
  uint4* caches[2 * kKeepLayers];  // keys and values of a layer in turn
  const int32_t* path;      // [batch, tokens]
  const int64_t* accepted;  // [batch]
  int32_t* lengths;         // [batch]
  int64_t vec_b, vec_h, vec_p;  // strides in 16-byte pieces
  int per_head;                 // 16-byte pieces of a head
  int* status;
};

// How many tokens of sequence b stay: the whole CTA asks, thread i holding path[i]; -1 for a path
// that does not ascend within the tree and the capacity.
__device__ __forceinline__ int kept_tokens(const TreeKeepParams& p, int b, int64_t pre, int* src) {
  const TreeView& t = p.tree;
  const int64_t acc = p.accepted[b];
  const int count = static_cast<int>(acc < 0 ? 0 : acc + 1 > t.tokens ? t.tokens : acc + 1);
  bool bad = acc >= t.tokens || acc < -1 || (count > 0 && pre < 0);
  if (static_cast<int>(threadIdx.x) < count) {
    const int32_t* path = p.path + static_cast<int64_t>(b) * t.tokens + threadIdx.x;
    const int before = threadIdx.x ? path[-1] : -1;
    src[threadIdx.x] = path[0];
    bad = bad || path[0] <= before || path[0] >= t.tokens || pre + path[0] >= t.capacity;
  }
  return __syncthreads_or(bad) ? -1 : count;
}

// Grid (caches, batch): a CTA moves one sequence's path in one cache.
__global__ void __launch_bounds__(kKeepThreads) tree_keep_kernel(const TreeKeepParams p) {
  __shared__ int src[kTreeTokens];
  pdl_launch_dependents();
  pdl_wait();
  const TreeView& t = p.tree;
  const int b = blockIdx.y;
  const int64_t pre = t.prefix[b];
  const int count = kept_tokens(p, b, pre, src);
  uint4* base = p.caches[blockIdx.x] + b * p.vec_b + pre * p.vec_p;
  for (int e = threadIdx.x; e < t.kv_heads * p.per_head; e += kKeepThreads) {
    uint4* col = base + (e / p.per_head) * p.vec_h + e % p.per_head;
    for (int i = 0; i < count; ++i)
      if (src[i] != i) col[i * p.vec_p] = col[src[i] * p.vec_p];
  }
}

// The new lengths, behind all moves: they may be written over the old ones, which every CTA of a
// move reads.
__global__ void __launch_bounds__(kTreeTokens) tree_lengths_kernel(const TreeKeepParams p) {
  __shared__ int src[kTreeTokens];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x;
  const int64_t pre = p.tree.prefix[b];
  const int count = kept_tokens(p, b, pre, src);
  if (threadIdx.x != 0) return;
  if (count < 0) report_device_error(p.status, FITQ_ERR_ARG);
  p.lengths[b] = static_cast<int32_t>(pre) + (count < 0 ? 0 : count);
}

}  // namespace

int launch_tree_append(const TreeView& tree, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                       const void* v, int64_t v_stride, void* q_out, void* k_cache, void* v_cache, const float* cs,
                       const float* sn, int rope_len, int heads, int dim, int dtype, int* status, cudaStream_t st) {
  const TreeAppendParams p{tree, q, k, v, q_stride, k_stride, v_stride, q_out, k_cache, v_cache, cs, sn, rope_len, heads,
                           dim, status};
  const dim3 grid(static_cast<unsigned>(tree.batch) * tree.tokens);
  const cudaError_t e =
      dtype == FITQ_DTYPE_BF16
          ? launch_pdl(tree_append_kernel<__nv_bfloat16>, grid, dim3(kAppendThreads), 0, st, p)
          : launch_pdl(tree_append_kernel<__half>, grid, dim3(kAppendThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

int launch_tree_keep(const TreeView& tree, void* const* k_caches, void* const* v_caches, int layers, int dim,
                     const int32_t* path, const int64_t* accepted, int32_t* lengths, int* status, cudaStream_t st) {
  TreeKeepParams p{};
  p.tree = tree;
  p.path = path;
  p.accepted = accepted;
  p.lengths = lengths;
  p.vec_b = tree.stride_b / 8;
  p.vec_h = tree.stride_h / 8;
  p.vec_p = tree.stride_p / 8;
  p.per_head = dim / 8;
  p.status = status;
  for (int at = 0; at < layers; at += kKeepLayers) {
    const int n = layers - at < kKeepLayers ? layers - at : kKeepLayers;
    for (int i = 0; i < n; ++i) {
      p.caches[2 * i] = static_cast<uint4*>(k_caches[at + i]);
      p.caches[2 * i + 1] = static_cast<uint4*>(v_caches[at + i]);
    }
    const cudaError_t e = launch_pdl(tree_keep_kernel, dim3(2 * n, tree.batch), dim3(kKeepThreads), 0, st, p);
    note_launch();
    if (e != cudaSuccess) return FITQ_ERR_CUDA;
  }
  const cudaError_t e = launch_pdl(tree_lengths_kernel, dim3(tree.batch), dim3(kTreeTokens), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace fitq
