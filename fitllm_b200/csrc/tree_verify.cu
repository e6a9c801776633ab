// Drafted tokens against the model's probabilities, from given random numbers.
//
// A sequence's walk starts at token 0 with p = softmax(logits / temperature) (temperature
// 0: all of it on the largest logit, the lowest index where two are equal).  The token's
// children are tried in order of their index: child c with id x is accepted where
// u_c q(x) < p(x) (q: the distribution the children were drawn from; without one, where
// u_c < p(x)), and the walk goes on from it.  Where it is refused p becomes
// max(p - q, 0) (without q: p with p(x) = 0), normalised, which makes the accepted tokens
// and the one drawn behind them a sample of the model's own distribution.  Behind the
// last child the next token is the first whose cumulated p exceeds u_0.
//
// Everything is computed in fp64 from the logits: a border between two tokens moves by
// some 1e-15 with the order of a sum, by 1e-8 in fp32, and a random number falls into
// that gap once in 10^3 rows of 152,064 tokens.
//
// A cluster of up to eight CTAs walks with a sequence; every warp owns a run of the
// vocabulary, so that the cumulated sum is found by its parts: ranks, warps, lanes.
#include <type_traits>

#include "kernels.cuh"
#include "tree.cuh"

namespace fitq {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCtas = 8;

struct TreeVerifyParams {
  const void* logits;
  int64_t stride_b, stride_t;  // elements between sequences and between their rows
  const int64_t* tokens;       // [batch, T]
  const int32_t* parents;
  int64_t parents_stride;
  const float* uniforms;       // [batch, T]
  const float* probs;          // [batch, T - 1, V] rows of q, or null
  int64_t probs_stride_b, probs_stride_t;
  const float* temperatures;   // [batch], or null: `temperature` for all
  float temperature;
  int T, V;
  int32_t* path;       // [batch, T]
  int64_t* accepted;   // [batch]
  int64_t* next_token; // [batch]
  int* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint64_t remote_u64(const void* p, uint32_t rank) {
  uint32_t a;
  uint64_t v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
}

// Floats in an order that unsigned comparison follows (-0 as 0), every NaN the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) tree_verify_kernel(const TreeVerifyParams p) {
  __shared__ int up[kTreeTokens];
  __shared__ uint64_t sh_warp[kWarps], sh_mine[2];
  __shared__ double sh_inv[kTreeTokens];   // 1 / sum of the weights before refusal k
  __shared__ int64_t sh_gone[kTreeTokens]; // ids refused at this token (without q)
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int64_t b = blockIdx.x / ranks;
  if (tid < p.T) {
    const int pr = p.parents[b * p.parents_stride + tid];
    const bool fine = pr >= -2 && pr < tid;
    if (!fine && rank == 0) report_device_error(p.status, FITQ_ERR_ARG);
    up[tid] = fine ? pr : -2;
    if (rank == 0) p.path[b * p.T + tid] = -1;
  }
  __syncthreads();
  const float temp = p.temperatures ? p.temperatures[b] : p.temperature;
  if (up[0] != -1 || !(temp >= 0.f) || temp == INFINITY) {  // no token to start from: the whole cluster
    if (tid == 0 && rank == 0) {
      if (up[0] != -2) report_device_error(p.status, FITQ_ERR_ARG);
      p.accepted[b] = -1;
      p.next_token[b] = -1;
    }
    return;
  }
  const bool greedy = temp == 0.f;
  const double inv_t = greedy ? 0.0 : 1.0 / static_cast<double>(temp);
  // this warp's run of the vocabulary
  const int per = (p.V + static_cast<int>(ranks) * kWarps - 1) / (static_cast<int>(ranks) * kWarps);
  const int lo = min(p.V, (static_cast<int>(rank) * kWarps + warp) * per), hi = min(p.V, lo + per);
  int slot = 0;

  // The cluster's words in the order of its warps; every thread gets all ranks' totals.
  auto gather = [&](uint64_t mine, auto join, uint64_t (&all)[kMaxCtas]) {
    if (lane == 0) sh_warp[warp] = mine;
    __syncthreads();
    if (tid == 0) {
      uint64_t x = sh_warp[0];
      for (int w = 1; w < kWarps; ++w) x = join(x, sh_warp[w]);
      sh_mine[slot] = x;
    }
    cluster_barrier();
    for (uint32_t r = 0; r < ranks; ++r) all[r] = remote_u64(&sh_mine[slot], r);
    slot ^= 1;
  };
  auto add = [](uint64_t x, uint64_t y) {
    return static_cast<uint64_t>(__double_as_longlong(__longlong_as_double(x) + __longlong_as_double(y)));
  };
  auto larger = [](uint64_t x, uint64_t y) { return x > y ? x : y; };

  int cur = 0, taken = 0, refused = 0;
  bool usable = true;
  double total = 0.0;
  float top = 0.f;
  int best = 0;
  const T* z = nullptr;
  const float* q = nullptr;
  // the weight of token v at this point of the walk
  auto weight = [&](int v) -> double {
    double w;
    if (greedy) {
      w = v == best ? 1.0 : 0.0;
    } else {
      const float x = static_cast<float>(z[v]);
      w = exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
      if (p.probs) {
        for (int k = 0; k < refused; ++k) w = fmax(w * sh_inv[k] - static_cast<double>(q[v]), 0.0);
      } else {
        for (int k = 0; k < refused; ++k)
          if (sh_gone[k] == v) w = 0.0;
      }
    }
    return w;
  };
  auto warp_sum = [&](double s) {
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  };
  uint64_t all[kMaxCtas];
  double run = 0.0;  // this warp's sum
  auto sum_up = [&]() {
    double s = 0.0;
    for (int v = lo + lane; v < hi; v += 32) s += weight(v);
    run = warp_sum(s);
    gather(static_cast<uint64_t>(__double_as_longlong(run)), add, all);
    total = 0.0;
    for (uint32_t r = 0; r < ranks; ++r) total += __longlong_as_double(all[r]);
  };
  auto enter = [&]() {  // the row of token cur
    z = static_cast<const T*>(p.logits) + b * p.stride_b + cur * p.stride_t;
    q = p.probs ? p.probs + b * p.probs_stride_b + min(cur, p.T - 2) * p.probs_stride_t : nullptr;
    refused = 0;
    uint64_t key = 0;
    for (int v = lo + lane; v < hi; v += 32) {
      const uint64_t k = (static_cast<uint64_t>(order_of(static_cast<float>(z[v]))) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
      key = key > k ? key : k;
    }
    for (int o = 16; o; o >>= 1) key = larger(key, __shfl_xor_sync(0xffffffffu, key, o));
    gather(key, larger, all);
    for (uint32_t r = 0; r < ranks; ++r) key = larger(key, all[r]);
    top = value_of(static_cast<uint32_t>(key >> 32));
    best = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    usable = static_cast<uint32_t>(key >> 32) != 0xffffffffu && top != -INFINITY && (greedy || top != INFINITY);
    if (usable) sum_up();
  };

  enter();
  if (tid == 0 && rank == 0) p.path[b * p.T] = 0;
  for (int i = 1; i < p.T && usable; ++i) {
    if (up[i] != cur) continue;
    const int64_t x = p.tokens[b * p.T + i];
    const bool known = x >= 0 && x < p.V;
    const double u = p.uniforms[b * p.T + i];
    const double w = known ? weight(static_cast<int>(x)) : 0.0;
    const bool take = known && total > 0.0 && (greedy ? w > 0.0 : u * (q ? static_cast<double>(q[x]) : 1.0) * total < w);
    if (take) {
      cur = i;
      ++taken;
      if (tid == 0 && rank == 0) p.path[b * p.T + taken] = i;
      __syncthreads();
      enter();
    } else if (!greedy && total > 0.0) {
      __syncthreads();  // weights read the refusals so far
      if (tid == 0) {
        sh_inv[refused] = 1.0 / total;
        sh_gone[refused] = x;
      }
      __syncthreads();
      ++refused;
      sum_up();
    }
  }
  int64_t next = -1;
  if (usable && (greedy || !(total > 0.0))) {
    next = best;
  } else if (usable) {
    // the first token whose cumulated weight exceeds u_0 of the total
    const double goal = static_cast<double>(p.uniforms[b * p.T]) * total;
    double before = 0.0;
    int at = -1, last = 0;
    for (int r = 0; r < static_cast<int>(ranks); ++r) {
      const double s = __longlong_as_double(all[r]);
      if (s > 0.0) last = r;
      if (at < 0 && before + s > goal) at = r;
      if (at < 0) before += s;
    }
    const bool past = at < 0;  // a random number of one or more: the last token that has weight
    if (past) at = last;
    if (static_cast<int>(rank) == at) {
      // sh_warp still holds the sums of this CTA's warps
      int w_at = -1, w_last = 0;
      double base = past ? 0.0 : before;
      for (int w = 0; w < kWarps; ++w) {
        const double s = __longlong_as_double(sh_warp[w]);
        if (s > 0.0) w_last = w;
        if (!past && w_at < 0 && base + s > goal) w_at = w;
        if (w_at < 0 && !past) base += s;
      }
      if (w_at < 0) w_at = w_last;
      if (warp == w_at) {
        int found = -1, heavy = lo;
        for (int v0 = lo; v0 < hi && found < 0; v0 += 32) {
          const int v = v0 + lane;
          const double w = v < hi ? weight(v) : 0.0;
          double c = w;
          for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += y;
          }
          const uint32_t have = __ballot_sync(0xffffffffu, w > 0.0);
          const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && base + c > goal);
          if (have) heavy = v0 + 31 - __clz(have);
          if (!past && hit) found = v0 + __ffs(hit) - 1;
          base += __shfl_sync(0xffffffffu, c, 31);
        }
        if (lane == 0) p.next_token[b] = found >= 0 ? found : heavy;
      }
    }
    if (tid == 0 && rank == 0) p.accepted[b] = taken;
    cluster_barrier();  // no CTA leaves while its words are read
    return;
  }
  if (tid == 0 && rank == 0) {
    p.accepted[b] = taken;
    p.next_token[b] = next;
  }
  cluster_barrier();
}

template <typename T>
int verify_t(const TreeVerifyParams& p, int64_t batch, cudaStream_t st, int num_sms) {
  int ctas = 1;
  while (ctas < kMaxCtas && batch * ctas * 2 <= 2ll * num_sms && p.V > kThreads * ctas * 2) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, tree_verify_kernel<T>, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace

int launch_tree_verify(const void* logits, int dtype, int64_t stride_b, int64_t stride_t, int64_t batch, int tokens,
                       int64_t vocab, const int64_t* ids, const int32_t* parents, int64_t parents_stride,
                       const float* uniforms, const float* probs, int64_t probs_stride_b, int64_t probs_stride_t,
                       const float* temperatures, float temperature, int32_t* path, int64_t* accepted,
                       int64_t* next_token, int* status, cudaStream_t st, int num_sms) {
  const TreeVerifyParams p{logits, stride_b, stride_t, ids, parents, parents_stride, uniforms, tokens > 1 ? probs : nullptr,
                           probs_stride_b, probs_stride_t, temperatures, temperature, tokens, static_cast<int>(vocab),
                           path, accepted, next_token, status};
  if (dtype == FITQ_DTYPE_BF16) return verify_t<__nv_bfloat16>(p, batch, st, num_sms);
  if (dtype == FITQ_DTYPE_F16) return verify_t<__half>(p, batch, st, num_sms);
  return verify_t<float>(p, batch, st, num_sms);
}

}  // namespace fitq
