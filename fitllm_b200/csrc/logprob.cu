// Log probabilities of given tokens with the row's entropy and top alternatives,
// and the gradient.
//
// For a row z of V logits with M = max z, S = sum exp(z - M) = 1 + S' (S': all elements but
// one that is M), E' = sum exp(z - M) (z - M):
//   logp = z[id] - M - log1p(S'),   H = log1p(S') - E' / (1 + S'),
// and the k largest logits in order, the lower index first where two are equal
// (a NaN counts as the largest).  Upstream gradients a (logp), h (entropy) and
// t_j (alternatives) give, with p_v = exp(z_v - M - log S),
//   dz_v = [v = id] a + sum_j [v = top_j] t_j
//          - p_v (a + sum_j t_j) - h p_v (z_v - M - log S + H).
// M and log S are kept apart for the backward: their sum would lose the digits
// that log S carries behind M.
//
// logprob_fwd_kernel: up to eight CTAs (a cluster) share a row.  Sums are kept
// relative to a thread's own running maximum, which stays out of them (a likely token's 1
// would take the digits of what the others add up to: entropies of 0.04 were off by 5e-4 of
// themselves, now by 2e-6), and joined over warps, the CTA and the cluster.  Few rows: a thread's share stays in registers, every load issued
// before the first use.  Many rows: a CTA streams its row, eight 16-byte loads
// in flight per thread.  Alternatives: the k-th largest of 128 thread-group maxima
// bounds the k-th largest logit of the CTA's share from below; the few elements at
// or above it are ranked by (value, index), then the CTAs' lists are ranked together.
// Where more elements tie than the list holds, k rounds of a maximum search take over.
// A streamed row's bound comes from its first granules, behind which a granule whose
// maximum reaches it is noted and read again at the end; only a list that overflows
// reads the whole row again.
// Bound: HBM (one read) for many rows, latency for few: 2,048 rows of 152,064 bf16
// logits 123 us, 5.1 TB/s; 40 of fp32 with 5 alternatives 14 us; one of bf16 with 20
// alternatives 8.6 us.
//
// logprob_bwd_kernel: one read and one write of the row; the up to k + 1 marked
// elements are rewritten behind a CTA barrier.  Bound: HBM; 2,048 rows as above 233 us,
// 5.3 TB/s.
#include <type_traits>

#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 64;
constexpr int kLpGroups = 128;  // thread groups whose maxima bound the k-th largest
constexpr int kLpList = 1024;   // candidates a CTA ranks

constexpr float kLog2e = 1.4426950408889634f;
// Exponents below this weigh exactly 0; the bound keeps a weight of 0 from
// meeting an exponent of -inf.
constexpr float kLowest = -1000.f;
constexpr float kFarBelow = -3.402823466e38f;  // a base that stands for -inf: no finite value is smaller
// How far a streamed element may exceed the sums' base, by which what lies between loses digits
// and for which a warp's granules wait: 4 / 6 / 8 / 20 took 125.7 / 123.3 / 122.0 / 121.8 us for
// 2,048 rows of 152,064, 127.8 / 127.2 / 126.3 / 122.1 of logits spread by 6.
constexpr float kMove = 6.f;

// max(d, kLowest) that keeps a NaN.
__device__ __forceinline__ float bounded(float d) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(d), "f"(kLowest));
  return r;
}

// Floats in an order that unsigned comparison follows; equal floats get equal
// values (-0 as 0), every NaN the largest.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The float of an order value (0 for -0).
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t key_of(float x, int64_t idx) {
  return (static_cast<uint64_t>(order_of(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(idx));
}

// A row as 16-byte granules at 16-byte boundaries: the first and the last may hold
// elements of other rows.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const T* z;          // first element
  const uint4* frame;  // granule 0
  int lead;            // elements of granule 0 that lie before the row
  int vectors;         // granules that hold the row
  int in_lo, in_hi;    // granules [in_lo, in_hi) lie inside it
  int V;
  __device__ __forceinline__ Row(const T* base, int64_t v) : z(base), V(static_cast<int>(v)) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15u) / sizeof(T));
    frame = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(base) & ~static_cast<uintptr_t>(15));
    vectors = (lead + V + kVec - 1) / kVec;
    in_lo = lead ? 1 : 0;
    in_hi = (lead + V) / kVec;
  }
  // index of element 0 of granule i (may be negative for i = 0)
  __device__ __forceinline__ int first(int i) const { return i * kVec - lead; }
  __device__ __forceinline__ bool inside(int i) const { return i >= in_lo && i < in_hi; }
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// The elements of a granule as floats.
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
template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ uint4 pack_vec<__nv_bfloat16>(const float (&f)[8]) { return pack8<__nv_bfloat16>(f); }
template <>
__device__ __forceinline__ uint4 pack_vec<__half>(const float (&f)[8]) { return pack8<__half>(f); }
template <>
__device__ __forceinline__ uint4 pack_vec<float>(const float (&f)[4]) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// Granule i of a row; elements outside the row read as -inf.
template <typename T>
__device__ __forceinline__ uint4 load_vec(const Row<T>& r, int i) {
  if (r.inside(i)) return r.frame[i];
  float f[Row<T>::kVec];
#pragma unroll
  for (int j = 0; j < Row<T>::kVec; ++j) {
    const int e = r.first(i) + j;
    f[j] = (e >= 0 && e < r.V) ? to_f32<T>(r.z[e]) : -INFINITY;
  }
  return pack_vec<T>(f);
}

struct LogprobFwdParams {
  const void* logits;
  const int64_t* ids;
  int64_t V, stride;
  int top;
  float* logp;     // [rows]
  float* entropy;  // [rows]
  float* stats;    // [rows, 2]: M, log S; may be null
  float* top_logp; // [rows, top]
  int64_t* top_ids;
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
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// (m, s, t): the maximum m, and sum exp(d) and sum exp(d) d, d = z - m, over all elements
// but one that is m; of two parts joined.
__device__ __forceinline__ void join(float& m, float& s, float& t, float m2, float s2, float t2) {
  if (m2 > m) {
    const float a = m, b = s, c = t;
    m = m2, s = s2, t = t2;
    m2 = a, s2 = b, t2 = c;
  }
  if (m2 == -INFINITY) return;  // no element
  const float d = fmaxf(m2 - m, kLowest), k = exp2_approx(d * kLog2e), all = s2 + 1.f;
  s = fmaf(k, all, s);
  t = fmaf(k, fmaf(d, all, t2), t);
}

// Largest element of a granule; a NaN is passed over.
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& u);
template <>
__device__ __forceinline__ float vec_max<float>(const uint4& u) {
  return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
}
template <>
__device__ __forceinline__ float vec_max<__nv_bfloat16>(const uint4& u) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}
template <>
__device__ __forceinline__ float vec_max<__half>(const uint4& u) {
  const __half2* h = reinterpret_cast<const __half2*>(&u);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

constexpr int kLpUnroll = 8;  // granules in flight per thread of a streamed row
// From four rows per SM on, without alternatives, CTAs of 256 threads, four on an SM, cover
// each other's starts and ends better than two of 512: 2,048 / 1,200 / 600 rows of 152,064
// bf16 logits 123 / 84 / 53 us against 140 / 91 / 53, 5,000 rows of 32,001 86 against 117; 400
// rows lost (37 against 33).  With alternatives, whose bound and ranking are work of a whole
// CTA, they lose too (2,048 rows with 20: 248 against 217 us).
constexpr int kLpSmall = 256, kLpUnrollSmall = 6, kLpSmallRows = 4;

// kNV > 0: a thread's granules stay in registers; kNV = 0: they are streamed.
template <typename T, int kNV, bool kTop, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprob_fwd_kernel(const LogprobFwdParams p) {
  static_assert(!kTop || kThreads == 4 * kLpGroups, "four threads a group");
  constexpr int kVec = Row<T>::kVec;
  constexpr int kLpWarps = kThreads / 32;
  constexpr int kHeld = kNV > 0 ? kNV : (kThreads == kLpThreads ? kLpUnroll : kLpUnrollSmall);
  __shared__ float sh_m[kLpWarps], sh_s[kLpWarps], sh_t[kLpWarps];
  __shared__ float sh_part[8][3];  // the cluster's parts, in its first CTA
  __shared__ __align__(16) uint32_t sh_group[kTop ? kLpGroups : 4];
  __shared__ uint32_t sh_bound;
  __shared__ int sh_count, sh_granules;
  __shared__ int sh_granule[kTop && kNV == 0 ? kLpList : 1];  // a streamed row's granules that reach the bound
  __shared__ uint64_t sh_list[kTop ? kLpList : 1];
  __shared__ uint64_t sh_best[kTop ? kLpMaxTop : 1];      // this CTA's top, in order
  __shared__ uint64_t sh_all[kTop ? 8 * kLpMaxTop : 1];   // every CTA's, in the first CTA
  __shared__ uint64_t sh_red[kLpWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t cta = cluster_rank(), ctas = cluster_size();
  const int64_t row = blockIdx.x / ctas;
  cluster_arrive();  // waited for before the first store into another CTA's shared memory
  pdl_launch_dependents();
  pdl_wait();  // the logits come from the previous kernel
  const Row<T> r(static_cast<const T*>(p.logits) + row * p.stride, p.V);
  const int share = (r.vectors + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
  const int v_lo = share * static_cast<int>(cta), v_hi = min(v_lo + share, r.vectors);

  uint4 held[kHeld];
  constexpr int kStep = kThreads;  // granules between a thread's own
  // the given token's logit, fetched early
  int64_t id = -1;
  float z_id = 0.f;
  if (cta == 0 && tid == 0) {
    id = p.ids[row];
    if (id >= 0 && id < p.V) z_id = to_f32<T>(r.z[id]);
  }
  // f(granule) over those of `held` from..to that the thread has, `held` being its granules from
  // v0 on; a mask of those for which it is true.  refill: each is replaced by the one kHeld
  // behind it at once.
  auto for_held = [&](auto from, auto to, auto refill, int v0, auto f) -> uint32_t {
    uint32_t mask = 0;
#pragma unroll
    for (int i = from.value; i < to.value; ++i) {
      const int v = v0 + i * kStep;
      if (v < v_hi && f(held[i])) mask |= 1u << i;
      if (refill.value && v + kHeld * kStep < v_hi) held[i] = load_vec(r, v + kHeld * kStep);
    }
    return mask;
  };
  constexpr std::integral_constant<int, 0> k0{};
  constexpr std::integral_constant<int, kHeld> kAll{};
  constexpr std::false_type kKeep{};
  constexpr std::true_type kRefill{};
  {
    const int v0 = v_lo + tid;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (v0 + i * kStep < v_hi) held[i] = load_vec(r, v0 + i * kStep);
  }

  // ---- the elements of a granule that are not below a bound go to the CTA's list
  auto collect = [&](int v, float bound_f) {
    float x[kVec];
    unpack_vec<T>(load_vec(r, v), x);
    uint32_t hits = 0;
    const int e0 = r.first(v);
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (!(x[j] < bound_f) && static_cast<uint32_t>(e0 + j) < static_cast<uint32_t>(r.V)) hits |= 1u << j;
    int at = atomicAdd(&sh_count, __popc(hits));
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if ((hits >> j) & 1u) {
        if (at < kLpList) sh_list[at] = key_of(x[j], e0 + j);
        ++at;
      }
  };
  // the same for the granules of a mask (few: they are read again)
  auto collect_mask = [&](uint32_t mask, int v0, float bound_f) {
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      collect(v0 + i * kStep, bound_f);
    }
  };
  // The top-th largest of the thread groups' maxima (equal ones ranked by group), or
  // -inf where fewer groups have elements: at least `top` elements are not smaller.
  // Four threads rank a group.
  auto find_bound = [&](float thread_max) -> float {
    uint32_t g = (v_lo + tid < v_hi) ? order_of(thread_max) : 0u;  // 0: no element
    g = max(g, __shfl_xor_sync(0xffffffffu, g, 1));
    g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
    if ((tid & 3) == 0) sh_group[tid >> 2] = g;
    if (tid == 0) sh_count = sh_granules = 0;
    __syncthreads();
    const uint4* all = reinterpret_cast<const uint4*>(sh_group);
    const int own = tid >> 2;
    int rank = 0;
#pragma unroll
    for (int i = 0; i < kLpGroups / 16; ++i) {
      const int at = 4 * (4 * i + (tid & 3));
      const uint4 o = all[4 * i + (tid & 3)];
      rank += (o.x > g || (o.x == g && at < own)) + (o.y > g || (o.y == g && at + 1 < own)) +
              (o.z > g || (o.z == g && at + 2 < own)) + (o.w > g || (o.w == g && at + 3 < own));
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (rank == p.top - 1) sh_bound = g;
    __syncthreads();
    const uint32_t b = sh_bound;
    return b <= 0x007fffffu ? -INFINITY : value_of(b);
  };

  // ---- maximum and sums of the thread's share
  float m = -INFINITY, base = 0.f;
  uint64_t s2 = 0, t2 = 0;  // the sums of the even and the odd elements
  auto add = [&](const uint4& u) {
    float x[kVec];
    unpack_vec<T>(u, x);
#pragma unroll
    for (int j = 0; j < kVec; j += 2) {
      // the difference first: it is exact near the maximum, and the type's lowest
      // value times log2 e would overflow
      float d0, d1, x0, x1;
      unpack2(add2(pack2(x[j], x[j + 1]), pack2(-base, -base)), d0, d1);
      const uint64_t d = pack2(bounded(d0), bounded(d1));
      unpack2(mul2(d, pack2(kLog2e, kLog2e)), x0, x1);
      const uint64_t e = pack2(exp2_approx(x0), exp2_approx(x1));
      s2 = add2(s2, e);
      t2 = fma2(e, d, t2);
    }
  };
  // sums without one of the elements that are the base: a 1 in the larger half
  auto less_one = [](uint64_t x) {
    float a, b;
    unpack2(x, a, b);
    return a >= b ? pack2(a - 1.f, b) : pack2(a, b - 1.f);
  };
  float bound_f = INFINITY;  // what the alternatives are not smaller than
  auto reaches = [&](const uint4& u) { return vec_max<T>(u) >= bound_f; };
  if (kNV > 0) {
    for_held(k0, kAll, kKeep, v_lo + tid, [&](const uint4& u) {
      m = fmaxf(m, vec_max<T>(u));
      return false;
    });
    base = m == -INFINITY ? 0.f : m;
    for_held(k0, kAll, kKeep, v_lo + tid, [&](const uint4& u) {
      add(u);
      return false;
    });
    if (m != -INFINITY) s2 = less_one(s2);
    if (kTop) {
      bound_f = find_bound(m);
      collect_mask(for_held(k0, kAll, kKeep, v_lo + tid, reaches), v_lo + tid, bound_f);
    }
  } else {
    // The sums' base, an element that stays out of them, only moves when a granule exceeds it
    // by kMove: moving it for every new maximum would cost a warp most of its granules.  The
    // first granules give a bound already.
    // Behind a batch in which it moved, it is taken off the sums, and the one before it comes in:
    // an element far above the others takes the digits of its batch's sums only.
    float was = kFarBelow;
    auto settle = [&] {
      if (base == was) return;
      const float d = fmaxf(was - base, kLowest), k = exp2_approx(d * kLog2e);
      s2 = add2(less_one(s2), pack2(k, 0.f));
      t2 = add2(t2, pack2(k * d, 0.f));
      was = base;
    };
    auto stream = [&](const uint4& u) -> bool {
      const float mx = vec_max<T>(u);
      m = fmaxf(m, mx);
      if (mx > base + kMove) {
        const float d = fmaxf(base - mx, kLowest), k = exp2_approx(d * kLog2e);
        t2 = mul2(pack2(k, k), fma2(pack2(d, d), s2, t2));
        s2 = mul2(pack2(k, k), s2);
        base = mx;
      }
      add(u);
      return kTop && mx >= bound_f;
    };
    int v0 = v_lo + tid;
    base = kFarBelow;
    if (v0 < v_hi) {
      const float first = vec_max<T>(held[0]);
      base = first == -INFINITY ? kFarBelow : first;
    }
    if (base == kFarBelow) s2 = pack2(-1.f, 0.f);
    // granules that reach the bound are noted, for the CTA to take together behind the row: at
    // once a warp would wait for each (2,048 rows of 152,064 with 20 alternatives: 249 -> 217 us,
    // 222 with what follows for the digits of likely tokens)
    auto note = [&](uint32_t mask) {
      if (mask == 0) return;
      for (int at = atomicAdd(&sh_granules, __popc(mask)); mask; mask &= mask - 1, ++at)
        if (at < kLpList) sh_granule[at] = v0 + (__ffs(mask) - 1) * kStep;
    };
    if (kTop) {
      for_held(k0, kAll, kKeep, v0, stream);
      settle();
      bound_f = find_bound(m);
      note(for_held(k0, kAll, kRefill, v0, reaches));
      v0 += kHeld * kStep;
    }
    for (; v0 < v_hi; v0 += kHeld * kStep) {
      const uint32_t mask = for_held(k0, kAll, kRefill, v0, stream);
      settle();
      if (kTop) note(mask);
    }
  }
  float s, t, s_odd, t_odd;
  unpack2(s2, s, s_odd);
  unpack2(t2, t, t_odd);
  s += s_odd;
  t += t_odd;
  const bool nan_here = s != s;
  const float thread_max = m;
  if (kNV == 0 && m > base) {
    // from here on relative to the maximum itself, which stays out instead of the base
    const float d = m - base, e = exp2_approx(d * kLog2e), k = exp2_approx(-d * kLog2e);
    s = s + 1.f - e;
    t = k * fmaf(-d, s, fmaf(-e, d, t));
    s *= k;
  }
  {
    float wm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    // one lane's maximum stays out, the others' come in
    const bool out = lane == __ffs(__ballot_sync(0xffffffffu, m == wm)) - 1 || m == -INFINITY;
    const float d = fmaxf(m - (wm == -INFINITY ? 0.f : wm), kLowest), k = exp2_approx(d * kLog2e);
    s += out ? 0.f : 1.f;
    t = k * fmaf(d, s, t);
    s *= k;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0) {
      sh_m[warp] = wm;
      sh_s[warp] = s;
      sh_t[warp] = t;
    }
  }
  if (kTop && tid < kLpMaxTop) sh_best[tid] = 0;
  // a granule's maximum passes NaNs over: a share that has one is searched again
  const int nan_seen = kTop ? __syncthreads_or(nan_here) : (__syncthreads(), 0);
  cluster_wait();  // every CTA of the cluster runs
  if (warp == 0) {
    float cm = lane < kLpWarps ? sh_m[lane] : -INFINITY;
    float cs = lane < kLpWarps ? sh_s[lane] : 0.f, ct = lane < kLpWarps ? sh_t[lane] : 0.f;
#pragma unroll
    for (int o = kLpWarps / 2; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, cm, o), s2 = __shfl_xor_sync(0xffffffffu, cs, o),
                  t2 = __shfl_xor_sync(0xffffffffu, ct, o);
      join(cm, cs, ct, m2, s2, t2);
    }
    if (lane == 0) {
      const uint32_t dst = map_rank(smem_u32(&sh_part[cta][0]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(cm) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(cs) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(ct) : "memory");
    }
  }
  if (kTop) {
    if (kNV == 0) {
      const int granules = sh_granules;
      for (int i = tid; i < granules && granules <= kLpList; i += kThreads) collect(sh_granule[i], bound_f);
      if (granules > kLpList && tid == 0) sh_count = kLpList + 1;
      __syncthreads();
    }
    int count = sh_count;
    if ((kNV == 0 && count > kLpList) || nan_seen) {  // uniform: once more, with the whole share's bound
      __syncthreads();
      bound_f = find_bound(thread_max);
      for (int v = v_lo + tid; v < v_hi; v += kStep) collect(v, bound_f);
      __syncthreads();
      count = sh_count;
    }
    if (count <= kLpList) {
      // the list's order varies, the keys' ranks do not: every key is unique; eight
      // threads rank a key
      for (int i0 = 0; i0 < count; i0 += kThreads / 8) {
        const int i = i0 + (tid >> 3);
        const uint64_t k = i < count ? sh_list[i] : 0;
        int rank = 0;
#pragma unroll 4
        for (int j = tid & 7; j < count; j += 8) rank += sh_list[j] > k ? 1 : 0;
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        rank += __shfl_xor_sync(0xffffffffu, rank, 4);
        if (i < count && rank < p.top && (tid & 7) == 0) sh_best[rank] = k;
      }
      __syncthreads();
    } else {
      uint64_t last = ~0ull;
      for (int n = 0; n < p.top; ++n) {
        uint64_t best = 0;
        for (int v = v_lo + tid; v < v_hi; v += kStep) {
          float x[kVec];
          unpack_vec<T>(load_vec(r, v), x);
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const int e = r.first(v) + j;
            if (e < 0 || e >= r.V) continue;
            const uint64_t k = key_of(x[j], e);
            if (k < last && k > best) best = k;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
          if (k > best) best = k;
        }
        if (lane == 0) sh_red[warp] = best;
        __syncthreads();
        best = 0;
        for (int w = 0; w < kLpWarps; ++w)
          if (sh_red[w] > best) best = sh_red[w];
        __syncthreads();
        last = best;
        if (tid == 0) sh_best[n] = best;
        if (best == 0) break;  // uniform: fewer elements than asked for in this share
      }
      __syncthreads();
    }
    if (tid < p.top) {
      const uint32_t dst = map_rank(smem_u32(&sh_all[cta * kLpMaxTop + tid]), 0);
      asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(dst), "l"(sh_best[tid]) : "memory");
    }
  }
  cluster_arrive();
  cluster_wait();  // the parts have arrived; the other CTAs' shared memory is read by nobody
  if (cta != 0) return;
  float M = sh_part[0][0], S = sh_part[0][1], E = sh_part[0][2];
  for (uint32_t c = 1; c < ctas; ++c) join(M, S, E, sh_part[c][0], sh_part[c][1], sh_part[c][2]);
  // S: of all elements but one that is M.  Nothing but -inf, or an infinity: no distribution
  const float log_s = fabsf(M) <= 3.402823466e38f ? log1pf(S) : NAN;
  if (tid == 0) {
    const bool valid = id >= 0 && id < p.V;
    p.logp[row] = valid ? (z_id - M) - log_s : 0.f;
    p.entropy[row] = log_s - E / (1.f + S);
    if (p.stats) {
      p.stats[2 * row] = M;
      p.stats[2 * row + 1] = log_s;
    }
  }
  if (kTop) {
    // every list is in order: a key's rank is its place in its own list and the
    // number of larger keys in each other one
    for (int i = tid; i < static_cast<int>(ctas) * kLpMaxTop; i += kThreads) {
      const int own = i / kLpMaxTop, place = i % kLpMaxTop;
      if (place >= p.top) continue;
      const uint64_t k = sh_all[i];
      if (k == 0) continue;  // no element
      int rank = place;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c >= static_cast<int>(ctas) || c == own) continue;
        int lo = 0, hi = p.top;  // how many keys of list c are larger
#pragma unroll
        for (int step = 0; step < 7; ++step) {
          if (lo >= hi) continue;
          const int mid = (lo + hi) >> 1;
          if (sh_all[c * kLpMaxTop + mid] > k)
            lo = mid + 1;
          else
            hi = mid;
        }
        rank += lo;
      }
      if (rank < p.top) {
        const uint32_t o = static_cast<uint32_t>(k >> 32);
        p.top_ids[row * p.top + rank] = 0xffffffffu - static_cast<uint32_t>(k);
        p.top_logp[row * p.top + rank] = ((o == 0xffffffffu ? NAN : value_of(o)) - M) - log_s;
      }
    }
  }
}

struct LogprobBwdParams {
  const void* logits;
  const int64_t* ids;
  int64_t V, stride;
  int top;
  const float *stats, *entropy;
  const int64_t* top_ids;
  const float *g_logp, *g_entropy, *g_top;  // each may be null
  void* d;  // [rows, V]
};

constexpr int kLbThreads = 256;
constexpr int kLbVectors = 8;  // granules per thread

template <typename T>
__global__ void __launch_bounds__(kLbThreads) logprob_bwd_kernel(const LogprobBwdParams p, int parts) {
  constexpr int kVec = Row<T>::kVec;
  __shared__ int64_t sh_id[kLpMaxTop + 1];
  __shared__ float sh_g[kLpMaxTop + 1];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  T* drow = static_cast<T*>(p.d) + row * p.V;
  const T* zrow = static_cast<const T*>(p.logits) + row * p.stride;
  const Row<T> out(drow, p.V);  // granules follow the gradient's alignment
  const bool aligned = ((reinterpret_cast<uintptr_t>(zrow) ^ reinterpret_cast<uintptr_t>(drow)) & 15u) == 0;
  const float M = p.stats[2 * row], log_s = p.stats[2 * row + 1];
  const float H = p.entropy[row];
  const int64_t id = p.ids[row];
  const int marks = (p.g_top ? p.top : 0) + 1;
  if (tid < marks) {
    const bool given = tid == 0;
    sh_id[tid] = given ? id : p.top_ids[row * p.top + tid - 1];
    sh_g[tid] = given ? ((p.g_logp && id >= 0 && id < p.V) ? p.g_logp[row] : 0.f) : p.g_top[row * p.top + tid - 1];
  }
  __syncthreads();
  float a = 0.f;
  for (int i = 0; i < marks; ++i) a += sh_g[i];
  const float h = p.g_entropy ? p.g_entropy[row] : 0.f;
  auto grad = [&](float z) {
    const float lp = (z - M) - log_s;
    const float pr = exp2_approx(lp * kLog2e);
    return -pr * fmaf(h, fmaxf(lp + H, kLowest), a);  // a probability of 0 takes no -inf with it
  };
  const int v0 = part * (kLbThreads * kLbVectors) + tid;
  uint4 z[kLbVectors];
#pragma unroll
  for (int i = 0; i < kLbVectors; ++i) {
    const int v = v0 + i * kLbThreads;
    if (aligned && v < out.vectors && out.inside(v)) z[i] = *reinterpret_cast<const uint4*>(zrow + out.first(v));
  }
#pragma unroll
  for (int i = 0; i < kLbVectors; ++i) {
    const int v = v0 + i * kLbThreads;
    if (v >= out.vectors) continue;
    if (aligned && out.inside(v)) {
      float x[kVec];
      unpack_vec<T>(z[i], x);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[j] = grad(x[j]);
      *reinterpret_cast<uint4*>(drow + out.first(v)) = pack_vec<T>(x);
    } else {
      for (int j = 0; j < kVec; ++j) {
        const int64_t e = out.first(v) + j;
        if (e >= 0 && e < p.V) drow[e] = from_f32<T>(grad(to_f32<T>(zrow[e])));
      }
    }
  }
  // ---- the marked elements of this part, every mark on the same element summed in order
  const int64_t e_lo = static_cast<int64_t>(part) * (kLbThreads * kLbVectors) * kVec - out.lead;
  const int64_t e_hi = e_lo + static_cast<int64_t>(kLbThreads) * kLbVectors * kVec;
  __syncthreads();
  if (tid < marks) {
    const int64_t e = sh_id[tid];
    if (e >= 0 && e < p.V && e >= e_lo && e < e_hi) {
      float g = 0.f;
      for (int i = 0; i < marks; ++i)
        if (sh_id[i] == e) g += sh_g[i];
      drow[e] = from_f32<T>(g + grad(to_f32<T>(zrow[e])));
    }
  }
}

template <typename T, int kNV>
int fwd_t(const LogprobFwdParams& p, int64_t rows, int ctas, cudaStream_t st, bool small = false) {
  auto* kernel = p.top > 0 ? logprob_fwd_kernel<T, kNV, true, kLpThreads>
                 : small   ? logprob_fwd_kernel<T, 0, false, kLpSmall>
                           : logprob_fwd_kernel<T, kNV, false, kLpThreads>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * ctas));
  cfg.blockDim = dim3(p.top == 0 && small ? kLpSmall : kLpThreads);
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
int fwd_sized(const LogprobFwdParams& p, int64_t rows, cudaStream_t st, int num_sms) {
  const int64_t vectors = (p.V * static_cast<int64_t>(sizeof(T)) + 15) / 16 + 1;
  // As many CTAs per row (one, two, four or eight) as find room at once, two on an SM, and
  // work for every thread: of 152,064 bf16 logits, on 148 SMs, up to 37 rows take eight each,
  // up to 74 four, up to 148 two, more rows one.
  int ctas = 1;
  while (ctas < 8 && rows * ctas * 2 <= 2ll * num_sms && vectors > kLpThreads * ctas) ctas *= 2;
  const int64_t per = (vectors + ctas - 1) / ctas;
  if (per <= 2 * kLpThreads) return fwd_t<T, 2>(p, rows, ctas, st);
  if (per <= 5 * kLpThreads) return fwd_t<T, 5>(p, rows, ctas, st);
  return fwd_t<T, 0>(p, rows, ctas, st, ctas == 1 && rows >= kLpSmallRows * num_sms);
}

template <typename T>
int bwd_t(const LogprobBwdParams& p, int64_t rows, cudaStream_t st) {
  const int64_t vectors = (p.V * static_cast<int64_t>(sizeof(T)) + 15) / 16 + 1;
  const int parts = static_cast<int>((vectors + kLbThreads * kLbVectors - 1) / (kLbThreads * kLbVectors));
  const cudaError_t e = launch_pdl(logprob_bwd_kernel<T>, dim3(static_cast<unsigned>(rows * parts)), dim3(kLbThreads), 0,
                                   st, p, parts);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace

int launch_token_logprobs(const void* logits, int dtype, const int64_t* ids, int64_t rows, int64_t V, int64_t stride,
                          int top, float* logp, float* entropy, float* stats, float* top_logp, int64_t* top_ids,
                          cudaStream_t st, int num_sms) {
  const LogprobFwdParams p{logits, ids, V, stride, top, logp, entropy, stats, top_logp, top_ids};
  if (dtype == FITQ_DTYPE_F32) return fwd_sized<float>(p, rows, st, num_sms);
  if (dtype == FITQ_DTYPE_F16) return fwd_sized<__half>(p, rows, st, num_sms);
  return fwd_sized<__nv_bfloat16>(p, rows, st, num_sms);
}

int launch_token_logprobs_bwd(const void* logits, int dtype, const int64_t* ids, int64_t rows, int64_t V,
                              int64_t stride, int top, const float* stats, const float* entropy,
                              const int64_t* top_ids, const float* g_logp, const float* g_entropy,
                              const float* g_top, void* d, cudaStream_t st) {
  const LogprobBwdParams p{logits, ids, V, stride, top, stats, entropy, top_ids, g_logp, g_entropy, g_top, d};
  if (dtype == FITQ_DTYPE_F32) return bwd_t<float>(p, rows, st);
  if (dtype == FITQ_DTYPE_F16) return bwd_t<__half>(p, rows, st);
  return bwd_t<__nv_bfloat16>(p, rows, st);
}

}  // namespace fitq
