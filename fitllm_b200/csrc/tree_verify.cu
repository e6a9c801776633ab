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
// some 1e-14 with the order of a sum and the exponentials' last digits, by 1e-8 in fp32, and a
// random number falls into that gap once in 10^3 rows of 152,064 tokens (once in 10^6 with
// what is left here).  An exponential is 2^(n / 1024) from a table times a polynomial of degree
// two (its Taylor series: 7e-12 of it at |x| <= ln 2 / 2048): with its place in the sum eight fp64
// operations and some ten others per element, which the issue of instructions bounds.
//
// A cluster of up to sixteen CTAs walks with a sequence; every warp owns a run of the
// vocabulary, so that the cumulated sum is found by its parts: ranks, warps, lanes.  A CTA sums
// by its own largest logit, and one exchange over the cluster joins largest logits and
// sums.  A refused child costs another read of the row (from L1 and L2) with its q, and without a q a
// subtraction.
// Bound: the chain of a visited row (largest 1.1, sum 2.8, exchange 0.8, joining 0.8, a child's test 0.7 us
// on eight CTAs), and a batch's deepest path.  A chain of 5 rows of 152,064 tokens on sixteen CTAs: 28 us where all
// drafts are accepted, 15 where the first is refused (a row and the row again with its q), 8.9 for a row alone: 4.9 for
// each further one.  64 such chains: 95 to 99; at temperature 0, which reads a row for its largest logit and again for
// its index, 56; 16 trees of 32 tokens over 32,001: 19.5; one row of each of 64 sequences: 21.
#include <mutex>
#include <type_traits>

#include "kernels.cuh"
#include "tree.cuh"

namespace fitq {
namespace {

constexpr int kMaxCtas = 16;
constexpr int kAlone = 120 * 1024;  // shared memory that leaves an SM to one CTA
constexpr int kTable = 1024;
constexpr int kAhead = 2;  // a lane's granules on their way

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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_barrier() {
  cluster_arrive();
  cluster_wait();
}
__device__ __forceinline__ void store_remote(const void* p, uint32_t rank, uint64_t v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

__device__ __forceinline__ void store_remote_f32(const void* p, uint32_t rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

// The larger, a NaN before all.
__device__ __forceinline__ float max_nan(float x, float y) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
template <typename T>
__device__ __forceinline__ float max_vec(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    auto pair = [](uint32_t x, uint32_t y) {
      uint32_t r;
      if constexpr (std::is_same<T, __half>::value)
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
      else
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
      return r;
    };
    const float2 f = Half16<T>::unpack(pair(pair(u.x, u.y), pair(u.z, u.w)));
    return max_nan(f.x, f.y);
  }
}

// A float as a double by integer operations (the conversion instruction kept its pipe 64% busy).
// Zeros and subnormals read as some 2^-127, infinities as 2^128, none of which a weight shows.  16-bit
// types leave the low word empty.
template <bool kLow>
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double((static_cast<int>(u) >> 3 & 0x8fffffff) + (896 << 20), kLow ? static_cast<int>(u << 29) : 0);
}

template <typename T>
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void unpack_vec<__nv_bfloat16>(const uint4& u, float (&f)[8]) { unpack8<__nv_bfloat16>(u, f); }
template <>
__device__ __forceinline__ void unpack_vec<__half>(const uint4& u, float (&f)[8]) { unpack8<__half>(u, f); }
template <>
__device__ __forceinline__ void unpack_vec<float>(const uint4& u, float (&f)[4]) {
  f[0] = __uint_as_float(u.x);
  f[1] = __uint_as_float(u.y);
  f[2] = __uint_as_float(u.z);
  f[3] = __uint_as_float(u.w);
}

// 2^(j / 1024) in [1, 2), its high word less by j << 10: adding n << 10 for any n with n & 1023 = j
// then makes it 2^(n / 1024).  By all threads of a CTA.
__device__ __forceinline__ void make_table(double* table, double* roots) {
  if (threadIdx.x < 64) roots[threadIdx.x] = exp2(static_cast<double>(threadIdx.x < 32 ? threadIdx.x : (threadIdx.x - 32) * 32) / kTable);
  __syncthreads();
  for (int j = threadIdx.x; j < kTable; j += blockDim.x) {
    const double e = roots[j & 31] * roots[32 + (j >> 5)];
    table[j] = __hiloint2double(__double2hiint(e) - (j << 10), __double2loint(e));
  }
}

// Weights exp((x - top) / temperature) of logits.
struct Scale {
  double scale, start;  // exponent in 1024ths: scale x + start
  float low;            // what lies below weighs nothing: some 2^-1020 of the largest
  // Where the largest is so far from 0 that its weight would have no digits left, the exponents are as
  // much smaller as leaves all other logits nothing still.
  __device__ __forceinline__ void set(float top, float temp) {
    const double per = kTable * 1.4426950408889634074 / static_cast<double>(temp), far = per * static_cast<double>(fabsf(top));
    scale = far <= 1.4e17 ? per : per * (1.4e17 / far);
    start = -scale * static_cast<double>(top);
    low = __double2float_ru(static_cast<double>(top) - 707.0 * static_cast<double>(temp));
  }
  template <bool kLow>
  __device__ __forceinline__ double weigh(const double* table, float x) const {  // for x >= low
    const double v = fma(widen<kLow>(x), scale, start);
    const double t = v + 6755399441055744.0;  // 1.5 * 2^52: the whole part in the low bits
    const double r = v - (t - 6755399441055744.0);
    constexpr double kL = 0.69314718055994531 / kTable;
    const int n = __double2loint(t);
    const double e = table[n & (kTable - 1)];
    return __hiloint2double(__double2hiint(e) + (n << 10), __double2loint(e)) * fma(r, fma(r, kL * kL / 2.0, kL), 1.0);
  }
  __device__ __forceinline__ double point(const double* table, float x) const { return x >= low ? weigh<true>(table, x) : 0.0; }
};

// A row of logits as 16-byte granules, the first and the last perhaps shared with other rows.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const uint4* frame;
  int lead, V, granules;
  __device__ __forceinline__ Row(const T* z, int v) : V(v) {
    frame = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(z) & ~static_cast<uintptr_t>(15));
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15u) / sizeof(T));
    granules = (lead + V + kVec - 1) / kVec;
  }
  __device__ __forceinline__ int first(int i) const { return i * kVec - lead; }  // index of granule i's element 0
  __device__ __forceinline__ bool inside(int i) const { return first(i) >= 0 && first(i) + kVec <= V; }
  // calls f(granule, its 16 bytes) for granules lo + lane, lo + lane + 32 .. below hi, kAhead on their way
  template <typename F>
  __device__ __forceinline__ void each(int lo, int hi, F f) const {
    for (int i0 = lo + static_cast<int>(threadIdx.x & 31); i0 < hi; i0 += 32 * kAhead) {
      uint4 u[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) u[k] = i0 + 32 * k < hi ? __ldg(frame + i0 + 32 * k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i0 + 32 * k < hi) f(i0 + 32 * k, u[k]);
    }
  }
  // the largest of a warp's granules, a NaN before all
  __device__ __forceinline__ float largest(int lo, int hi) const {
    float m = -INFINITY;
    each(lo, hi, [&](int i, const uint4& u) {
      if (inside(i)) {
        m = max_nan(m, max_vec<T>(u));
      } else {
        float x[kVec];
        unpack_vec<T>(u, x);
#pragma unroll
        for (int y = 0; y < kVec; ++y)
          if (first(i) + y >= 0 && first(i) + y < V) m = max_nan(m, x[y]);
      }
    });
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
  }
  // the first index of a warp's granules with logit x, or 2^31 - 1
  __device__ __forceinline__ int first_of(int lo, int hi, float x) const {
    int at = 0x7fffffff;
    each(lo, hi, [&](int i, const uint4& u) {
      float f[kVec];
      unpack_vec<T>(u, f);
#pragma unroll
      for (int y = kVec - 1; y >= 0; --y) {
        const int v = first(i) + y;
        if (f[y] == x && v >= 0 && v < V && v < at) at = v;
      }
    });
    return __reduce_min_sync(0xffffffffu, at);
  }
  // the weights of a granule, side by side (one after the other, each with its refusals, they took five
  // times as long)
  __device__ __forceinline__ void weights(const double* table, const Scale& s, int i, const uint4& u, double (&w)[kVec]) const {
    float x[kVec];
    unpack_vec<T>(u, x);
#pragma unroll
    for (int y = 0; y < kVec; ++y) w[y] = s.weigh<sizeof(T) == 4>(table, x[y]);
#pragma unroll
    for (int y = 0; y < kVec; ++y) w[y] = x[y] >= s.low ? w[y] : 0.0;
    if (!inside(i)) {
#pragma unroll
      for (int y = 0; y < kVec; ++y)
        if (first(i) + y < 0 || first(i) + y >= V) w[y] = 0.0;
    }
  }
  static __device__ __forceinline__ double total_of(const double (&w)[kVec]) {
    double s[kVec / 2];
#pragma unroll
    for (int y = 0; y < kVec / 2; ++y) s[y] = w[2 * y] + w[2 * y + 1];
    if constexpr (kVec == 8) return (s[0] + s[1]) + (s[2] + s[3]);
    return s[0] + s[1];
  }
};

__device__ __forceinline__ double warp_sum(double s) {
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 2) tree_verify_kernel(const TreeVerifyParams p) {
  constexpr int kWarps = kThreads / 32;
  constexpr int kVec = 16 / sizeof(T);
  __shared__ int up[kTreeTokens];
  __shared__ double sh_table[kTable], sh_roots[64];
  __shared__ float sh_top[kWarps], sh_tops[2][kMaxCtas];   // largest logits; double-buffered by exchange
  __shared__ double sh_run[kWarps], sh_sums[2][kMaxCtas];
  __shared__ double sh_inv[kTreeTokens];   // 1 / sum of the weights before refusal k
  __shared__ int64_t sh_gone[kTreeTokens]; // ids refused at this token (without q)
  __shared__ int sh_hit[kWarps], sh_have[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  make_table(sh_table, sh_roots);
  pdl_launch_dependents();
  pdl_wait();
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
  if (up[0] != -1 || !(temp == 0.f || temp >= 1e-30f) || temp == INFINITY) {  // no token to start from: the whole cluster
    if (tid == 0 && rank == 0) {
      if (up[0] != -2) report_device_error(p.status, FITQ_ERR_ARG);
      p.accepted[b] = -1;
      p.next_token[b] = -1;
    }
    return;
  }
  cluster_arrive();  // waited for before the first store into another CTA's shared memory
  const bool greedy = temp == 0.f;
  int slot = 0;
  bool fresh = true;

  int cur = 0, taken = 0, refused = 0;
  bool usable = true;
  double total = 0.0;       // of the weights as refusals have left them
  double entered = 0.0;     // the total before any refusal
  uint64_t kids = 0;        // children of token cur
  bool exact = false;       // total, the parts and sh_run are sums of the weights as they are drawn from
  float top = 0.f;          // the row's largest logit
  int best = 0;
  Scale by{};
  const T* z = nullptr;
  const float* q = nullptr;
  Row<T> row(static_cast<const T*>(p.logits), p.V);
  int lo = 0, hi = 0;       // this warp's granules
  double rescale = 0.0;     // what makes sh_run this CTA's part of the total
  double its_sum = 0.0;     // lane r: rank r's part
  float its_top = 0.f;      // lane r: the logit that it was summed by

  // what makes weights by logit x weights by the row's largest
  auto part_of = [&](float x) -> double { return x == top ? 1.0 : by.point(sh_table, x); };
  // what refusals have left of weight w of token v
  auto left = [&](double w, int v, float qv) -> double {
    if (q) {
      for (int k = 0; k < refused; ++k) w = fmax(fma(w, sh_inv[k], -widen<true>(qv)), 0.0);
    } else {
      for (int k = 0; k < refused; ++k)
        if (sh_gone[k] == v) w = 0.0;
    }
    return w;
  };
  // the same of granule i's weights
  auto refuse = [&](int i, double (&w)[kVec]) {
    if (refused == 0) return;
    const int v0 = row.first(i);
    if (q) {
      float qv[kVec];
      const float* src = q + v0;
      if (row.inside(i) && (reinterpret_cast<uintptr_t>(src) & 15u) == 0) {
#pragma unroll
        for (int y = 0; y < kVec; y += 4) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(src + y));
          qv[y] = f.x;
          qv[y + 1] = f.y;
          qv[y + 2] = f.z;
          qv[y + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int y = 0; y < kVec; ++y) qv[y] = v0 + y >= 0 && v0 + y < p.V ? __ldg(src + y) : 0.f;
      }
      for (int k = 0; k < refused; ++k) {
        const double inv = sh_inv[k];
#pragma unroll
        for (int y = 0; y < kVec; ++y) {
          w[y] = fma(w[y], inv, -widen<true>(qv[y]));
          w[y] = w[y] > 0.0 ? w[y] : 0.0;
        }
      }
    } else {
      for (int k = 0; k < refused; ++k) {
        const int64_t at = sh_gone[k] - v0;
#pragma unroll
        for (int y = 0; y < kVec; ++y)
          if (at == y) w[y] = 0.0;
      }
    }
  };
  // sh_run's sum (and this CTA's largest logit) to all CTAs; on return sh_sums[slot ^ 1] and
  // sh_tops[slot ^ 1] hold the ranks'
  auto exchange = [&](bool tops, float mine) {
    __syncthreads();
    if (fresh) cluster_wait();  // every CTA of the cluster runs
    fresh = false;
    if (warp == 0) {
      double s = lane < kWarps ? sh_run[lane] : 0.0;
      s = warp_sum(s);
      if (lane < static_cast<int>(ranks)) {
        store_remote(&sh_sums[slot][rank], lane, static_cast<uint64_t>(__double_as_longlong(s)));
        if (tops) store_remote_f32(&sh_tops[slot][rank], lane, mine);
      }
    }
    cluster_barrier();
    slot ^= 1;
  };
  auto sum_runs = [&](float mine, const Scale& s) {  // this warp's weights, as refusals have left them
    double sum = 0.0;
    if (fabsf(mine) < INFINITY)
      row.each(lo, hi, [&](int i, const uint4& u) {
        double w[kVec];
        row.weights(sh_table, s, i, u, w);
        refuse(i, w);
        sum += Row<T>::total_of(w);
      });
    sum = warp_sum(sum);
    if (lane == 0) sh_run[warp] = sum;
  };
  auto sum_up = [&]() {  // by the row's largest logit, which is known
    __syncthreads();
    sum_runs(top, by);
    exchange(false, 0.f);
    its_top = top;
    its_sum = lane < static_cast<int>(ranks) ? sh_sums[slot ^ 1][lane] : 0.0;
    total = warp_sum(its_sum);
    rescale = 1.0;
    exact = true;
  };
  // the row's first token with its largest logit, by the whole cluster
  auto find_best = [&]() {
    const int at = row.first_of(lo, hi, top);
    __syncthreads();
    if (lane == 0) sh_run[warp] = static_cast<double>(at);
    __syncthreads();
    double low = sh_run[0];
    for (int w = 1; w < kWarps; ++w) low = fmin(low, sh_run[w]);
    __syncthreads();
    if (lane == 0) sh_run[warp] = warp == 0 ? low : 0.0;  // the exchange adds the warps' up
    exchange(false, 0.f);
    low = sh_sums[slot ^ 1][0];
    for (uint32_t r = 1; r < ranks; ++r) low = fmin(low, sh_sums[slot ^ 1][r]);
    best = static_cast<int>(low);
  };
  auto enter = [&]() {  // the row of token cur
    z = static_cast<const T*>(p.logits) + b * p.stride_b + cur * p.stride_t;
    q = p.probs ? p.probs + b * p.probs_stride_b + min(cur, p.T - 2) * p.probs_stride_t : nullptr;
    refused = 0;
    exact = false;
    row = Row<T>(z, p.V);
    const int warps = static_cast<int>(ranks) * kWarps, per = (row.granules + warps - 1) / warps;
    lo = min(row.granules, (static_cast<int>(rank) * kWarps + warp) * per);
    hi = min(row.granules, lo + per);
    kids = __ballot_sync(0xffffffffu, lane < p.T && lane > cur && up[lane] == cur) |
           static_cast<uint64_t>(__ballot_sync(0xffffffffu, lane + 32 < p.T && lane + 32 > cur && up[lane + 32] == cur)) << 32;
    // ---- the CTA's largest logit, its weights' sum by it, and the cluster's
    float mine = row.largest(lo, hi);
    if (lane == 0) sh_top[warp] = mine;
    __syncthreads();
    mine = sh_top[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mine = max_nan(mine, sh_top[w]);
    if (greedy) {  // and the first index with it, in the sum's place
      const int at = row.first_of(lo, hi, mine);
      if (lane == 0) sh_run[warp] = static_cast<double>(at);
      __syncthreads();
      double low = sh_run[0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) low = fmin(low, sh_run[w]);
      __syncthreads();
      if (lane == 0) sh_run[warp] = warp == 0 ? low : 0.0;
    } else {
      Scale own{};
      own.set(mine, temp);
      sum_runs(mine, own);
    }
    exchange(true, mine);
    top = -INFINITY;
    for (uint32_t r = 0; r < ranks; ++r) top = max_nan(top, sh_tops[slot ^ 1][r]);
    usable = top == top && top != -INFINITY && (greedy || top != INFINITY);
    if (!usable) return;
    if (greedy) {
      double low = 0x7fffffff;
      for (uint32_t r = 0; r < ranks; ++r)
        if (sh_tops[slot ^ 1][r] == top) low = fmin(low, sh_sums[slot ^ 1][r]);
      best = static_cast<int>(low);
      return;
    }
    by.set(top, temp);
    // the ranks' sums, by the row's largest logit: a lane each
    its_top = lane < static_cast<int>(ranks) ? sh_tops[slot ^ 1][lane] : -INFINITY;
    its_sum = lane < static_cast<int>(ranks) ? sh_sums[slot ^ 1][lane] * part_of(its_top) : 0.0;
    total = warp_sum(its_sum);
    rescale = part_of(mine);
    entered = total;
  };

  enter();
  if (tid == 0 && rank == 0) p.path[b * p.T] = 0;
  while (usable && kids) {
    const int i = __ffsll(static_cast<long long>(kids)) - 1;
    kids &= kids - 1;
    const int64_t x = p.tokens[b * p.T + i];
    const bool known = x >= 0 && x < p.V;
    bool take = false;
    double w = 0.0;
    if (greedy) {
      take = known && x == best;
    } else if (known && total > 0.0) {
      const double u = p.uniforms[b * p.T + i];
      const float qx = q ? q[x] : 1.f;
      w = left(by.point(sh_table, static_cast<float>(z[x])), static_cast<int>(x), qx);
      take = u * static_cast<double>(qx) * total < w;
    }
    if (take) {
      cur = i;
      ++taken;
      if (tid == 0 && rank == 0) p.path[b * p.T + taken] = i;
      enter();
    } else if (!greedy && total > 0.0) {
      __syncthreads();  // weights read the refusals so far
      if (tid == 0) {
        sh_inv[refused] = 1.0 / total;
        sh_gone[refused] = x;
      }
      __syncthreads();
      ++refused;
      // Without q a refusal takes one weight away, by the logit that its part was summed by: what is subtracted
      // is the number that was added (by another logit it differs by some 1e-11 of itself, which is then all that
      // is left of a part without tokens).  As long as a thousandth of the row's weight is left, the sums'
      // roundings, some 100 x 2^-53 of it, are 1e-11 of the difference; behind that, and with q, the sum is taken anew.
      if (q || !(total - w >= entered * 0x1p-10)) {
        sum_up();
      } else if (w > 0.0) {
        exact = false;
        const int warps = static_cast<int>(ranks) * kWarps, per = (row.granules + warps - 1) / warps;
        const int owner = static_cast<int>((x + row.lead) / kVec) / per;
        Scale own{};
        own.set(__shfl_sync(0xffffffffu, its_top, owner / kWarps), temp);
        const double gone = own.point(sh_table, static_cast<float>(z[x]));
        if (lane == owner / kWarps) its_sum -= gone * part_of(its_top);
        total = warp_sum(its_sum);
        if (static_cast<int>(rank) == owner / kWarps && tid == 0) sh_run[owner % kWarps] -= gone;
      }
    }
  }
  if (tid == 0 && rank == 0) p.accepted[b] = taken;
  if (!usable || greedy || !(total > 0.0)) {
    if (usable && !greedy) find_best();  // refusals have left no weight
    if (tid == 0 && rank == 0) p.next_token[b] = usable ? best : -1;
  } else {
    // The first token whose cumulated weight exceeds u_0 of the total.  A difference may leave some last digits
    // (1e-11 of the total) to a part in which no weight is left, and a sum by another largest logit moves its
    // borders as far: where the random number falls within 1e-9 of a border the parts are summed anew, and a
    // part then has a sum where it has a token to name.
    const double u0 = fmax(static_cast<double>(p.uniforms[b * p.T]), 0.0);
    double goal, before;
    int at;
    bool past;  // a random number of one or more: the last token that has weight
    for (;;) {
      __syncthreads();  // sh_run is complete
      goal = u0 * total;
      before = 0.0;
      at = -1;
      int last = 0;
      double here = 0.0;
      for (int r = 0; r < static_cast<int>(ranks); ++r) {
        const double s = __shfl_sync(0xffffffffu, its_sum, r);
        if (s > 0.0) last = r;
        if (at < 0 && before + s > goal) {
          at = r;
          here = s;
        }
        if (at < 0) before += s;
      }
      past = at < 0;
      if (past) at = last;
      if (exact || (!past && goal - before > total * 1e-9 && before + here - goal > total * 1e-9)) break;
      sum_up();
    }
    if (static_cast<int>(rank) == at) {
      int w_at;
      double base;
      for (;;) {
        int w_last = 0;
        double here = 0.0;
        w_at = -1;
        base = past ? 0.0 : before;
        for (int w = 0; w < kWarps; ++w) {
          const double s = sh_run[w] * rescale;
          if (s > 0.0) w_last = w;
          if (!past && w_at < 0 && base + s > goal) {
            w_at = w;
            here = s;
          }
          if (w_at < 0 && !past) base += s;
        }
        const bool clear = w_at >= 0 && goal - base > total * 1e-9 && base + here - goal > total * 1e-9;
        if (w_at < 0) w_at = w_last;
        if (exact || clear) break;
        __syncthreads();  // sh_run has been read
        sum_runs(top, by);
        rescale = 1.0;
        exact = true;
        __syncthreads();
      }
      // that run again, 32 granules a warp, then the warp in whose granules it lies
      const int warps = static_cast<int>(ranks) * kWarps, per = (row.granules + warps - 1) / warps;
      const int first = min(row.granules, (static_cast<int>(rank) * kWarps + w_at) * per), end = min(row.granules, first + per);
      int found = -1, heavy = -1;
      for (int i0 = first; i0 < end && found < 0; i0 += 32 * kWarps) {
        const int i = i0 + 32 * warp + lane;
        double w[kVec], mine = 0.0;
#pragma unroll
        for (int y = 0; y < kVec; ++y) w[y] = 0.0;
        if (i < end) {
          row.weights(sh_table, by, i, __ldg(row.frame + i), w);
          refuse(i, w);
        }
#pragma unroll
        for (int y = 0; y < kVec; ++y) mine += w[y];
        double c = mine;
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += y;
        }
        __syncthreads();  // sh_run has been read
        if (lane == 31) sh_run[warp] = c;
        __syncthreads();
        double at_warp = base;  // what lies before this warp's granules
        for (int k = 0; k < warp; ++k) at_warp += sh_run[k];
        for (int k = 0; k < kWarps; ++k) base += sh_run[k];
        // within the lane's elements
        int hit = -1, have = -1;
        double sum = at_warp + (c - mine);
#pragma unroll
        for (int y = 0; y < kVec; ++y) {
          sum += w[y];
          if (w[y] > 0.0) {
            have = row.first(i) + y;
            if (hit < 0 && !past && sum > goal) hit = have;
          }
        }
        const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0), haves = __ballot_sync(0xffffffffu, have >= 0);
        if (lane == 0) {
          sh_hit[warp] = -1;
          sh_have[warp] = -1;
        }
        __syncwarp();
        if (hits && lane == __ffs(hits) - 1) sh_hit[warp] = hit;
        if (haves && lane == 31 - __clz(haves)) sh_have[warp] = have;
        __syncthreads();
        for (int k = 0; k < kWarps; ++k) {
          if (found < 0) found = sh_hit[k];
          if (sh_have[k] >= 0) heavy = sh_have[k];
        }
      }
      if (tid == 0) p.next_token[b] = found >= 0 ? found : heavy;
    }
  }
  cluster_barrier();  // no CTA leaves while its words are written
}

template <typename T, int kThreads>
int verify_t(const TreeVerifyParams& p, int64_t batch, int ctas, cudaStream_t st, int num_sms) {
  auto* kernel = tree_verify_kernel<T, kThreads>;
  // sixteen CTAs where they fill a third of the card at most, on cards whose GPCs have room for such a cluster
  if (ctas == 8 && batch * 48 <= num_sms && p.V > 8192) {
    static std::mutex mu;
    static int room[64] = {0};  // by device: 0 not asked yet, else clusters + 1
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FITQ_ERR_CUDA;
    if (!set_smem_limit(kernel, kAlone)) return FITQ_ERR_CUDA;
    std::lock_guard<std::mutex> lk(mu);
    if (room[dev] == 0) {
      cudaLaunchConfig_t ask = {};
      cudaLaunchAttribute shape[1];
      shape[0].id = cudaLaunchAttributeClusterDimension;
      shape[0].val.clusterDim.x = 16;
      shape[0].val.clusterDim.y = shape[0].val.clusterDim.z = 1;
      ask.gridDim = dim3(16);
      ask.blockDim = dim3(kThreads);
      ask.dynamicSmemBytes = kAlone;
      ask.attrs = shape;
      ask.numAttrs = 1;
      int clusters = 0;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
          cudaOccupancyMaxActiveClusters(&clusters, kernel, &ask) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
      }
      room[dev] = clusters + 1;
    }
    if (room[dev] > 1) ctas = 16;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(batch * ctas));
  cfg.blockDim = dim3(kThreads);
  // few CTAs spread over the SMs instead of meeting on some of them
  if (batch * ctas <= num_sms / 2) {
    if (!set_smem_limit(kernel, kAlone)) return FITQ_ERR_CUDA;
    cfg.dynamicSmemBytes = kAlone;
  }
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T>
int verify_sized(const TreeVerifyParams& p, int64_t batch, cudaStream_t st, int num_sms) {
  // CTAs of a sequence: as many as find room at once, two on an SM, and have work for their lanes.
  // Where eight do, of 256 threads, which have registers for a granule's weights side by side; else of
  // 384, of which more run at once: one chain 22 us instead of 25, 64 chains 106 instead of 96 (with
  // 512 of 64 registers 103).
  int ctas = 1;
  while (ctas < 8 && batch * ctas * 2 <= 2ll * num_sms && p.V > 1024 * ctas) ctas *= 2;
  return ctas == 8 ? verify_t<T, 256>(p, batch, ctas, st, num_sms) : verify_t<T, 384>(p, batch, ctas, st, num_sms);
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
  if (dtype == FITQ_DTYPE_BF16) return verify_sized<__nv_bfloat16>(p, batch, st, num_sms);
  if (dtype == FITQ_DTYPE_F16) return verify_sized<__half>(p, batch, st, num_sms);
  return verify_sized<float>(p, batch, st, num_sms);
}

}  // namespace fitq
