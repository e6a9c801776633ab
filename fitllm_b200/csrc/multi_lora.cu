// Low-rank adapters of many requests beside a shared projection:
//   y[n] = y_add[n] + s_l (x[n].A_l^T).B_l^T,   l = adapter of token n's sequence.
//
// Both products run on mma.sync m16n8k16: an adapter's R columns or rows give it a few
// operations per byte, so that the bytes of x, A, B and y are what costs.
//
// Tokens are taken in slots of up to kSlot of one sequence.  Slot numbers need no counting:
// sequence b, whose tokens begin at q_start[b], owns the numbers from q_start[b] / kSlot + b
// on, which leaves room for its slots whatever the lengths, so that the host launches
// tokens / kSlot + batch of them without knowing any.
//
// multi_lora_shrink_kernel, T = x.A_l^T: a cluster of up to eight CTAs shares a slot, each a part of
// K; a CTA's eight warps are dealt to its tokens (32 each) and the parts of K that are left over,
// so that a single token is summed by 64 warps.  A lane reads 16 bytes of a row of x and of A at
// a time and feeds them to two MMAs: the contraction index is permuted alike in both.  Parts
// join in shared memory, then over the cluster, in order (deterministic); T stays in fp32.
//
// multi_lora_expand_kernel, y = y_add + s T.B_l^T: T enters as two 16-bit numbers, hi + lo (a
// relative error of eps^2; one alone would cost the delta half its digits), scaled by a power of
// two per token for fp16's range.  The columns of four MMAs are dealt so that a lane's are eight in a
// row: y and y_add move in 16-byte pieces.  One rounding, of y.
#include <type_traits>

#include "kernels.cuh"
#include "kv4.cuh"

namespace fitq {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSlot = 256;       // tokens of a slot: 32 for each warp of the first kernel
constexpr int kTile = 128;       // of one of the second: 16 for each warp
constexpr int kCols = 512;       // columns of a CTA of the second
constexpr int kMaxParts = 8;     // CTAs of a cluster

struct MultiLoraParams {
  const void *x, *a, *b, *y_add;
  void* y;
  const float* scale;
  const int32_t* adapter;
  const int32_t* q_start;
  int64_t tokens, x_stride, y_add_stride;
  int batch, adapters, k, n, t_new;
  int parts;       // of K
  int part_cols;   // columns of a part, a multiple of 32
  int chunks;      // parts of N
  float* t;        // [tokens][rank]
  int* status;
};

// Tokens [first, first + count) of slot number s (slots of kSize), and their adapter (-1: none).
template <int kSize>
__device__ __forceinline__ bool slot_of(const MultiLoraParams& p, int64_t s, int lane, int64_t& first, int& count, int& l,
                                        bool report) {
  int64_t b, begin, end;
  if (p.q_start == nullptr) {
    const int per = (p.t_new + kSize - 1) / kSize;
    b = s / per;
    if (b >= p.batch) return false;
    begin = b * p.t_new;
    end = begin + p.t_new;
    first = begin + (s - b * per) * kSize;
  } else {
    // the last sequence whose numbers begin at or before s: 32 candidates at a time
    int64_t lo = 0, hi = p.batch;  // answer + 1 in [lo, hi]; every lane holds the same
    while (lo < hi) {
      const int64_t span = hi - lo, step = (span + 31) / 32;
      const int64_t at = lo + (lane + 1) * step - 1;  // asks whether the answer lies behind
      bool before = false;
      if (at < hi) {
        int64_t q = p.q_start[at];
        q = q < 0 ? 0 : q > p.tokens ? p.tokens : q;
        before = q / kSize + at <= s;
      }
      const uint32_t yes = __ballot_sync(0xffffffffu, before);
      const int n = __ffs(~yes) ? __ffs(~yes) - 1 : 32;  // leading candidates that say so
      const int64_t up = lo + (n + 1) * step - 1;
      lo += n * step;
      if (n < 32 && up < hi) hi = up;
      if (lo > hi) lo = hi;
    }
    b = lo - 1;
    if (b < 0) return false;
    begin = p.q_start[b];
    end = p.q_start[b + 1];
    begin = begin < 0 ? 0 : begin;
    end = end > p.tokens ? p.tokens : end;
    if (begin > p.tokens) return false;
    first = begin + (s - (begin / kSize + b)) * kSize;
  }
  if (first < begin || first >= end) return false;
  count = static_cast<int>(end - first < kSize ? end - first : kSize);
  l = p.adapter[b];
  if (l < -1 || l >= p.adapters) {
    if (report && lane == 0) report_device_error(p.status, FITQ_ERR_ARG);
    l = -1;
  }
  return true;
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 remote_float4(const float* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
  return v;
}

extern __shared__ float4 g_lora_smem[];

template <typename T, int R>
__global__ void __launch_bounds__(kThreads) multi_lora_shrink_kernel(const MultiLoraParams p) {
  constexpr int NT = R / 8;
  constexpr int kUnroll = R == 16 ? 4 : R == 32 ? 2 : 1;  // what the registers hold beside the sums
  float* red = reinterpret_cast<float*>(g_lora_smem);     // [warps][32][R]
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int part = blockIdx.x % p.parts;
  int64_t first;
  int count, l;
  if (!slot_of<kSlot>(p, blockIdx.x / p.parts, lane, first, count, l, part == 0 && warp == 0) || l < 0) return;  // the whole cluster
  // warps over tokens and, what is left, over K
  const int mw = count <= 32 ? 1 : count <= 64 ? 2 : count <= 128 ? 4 : 8, kw = kWarps / mw;
  const int wm = warp / kw, wk = warp % kw;
  const int m0 = wm * 32;
  const bool second = count - m0 > 16;  // the warp's other sixteen tokens
  const int k0 = part * p.part_cols, k1 = min(p.k, k0 + p.part_cols);
  float acc[2][NT][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[h][t][i] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const T* x = static_cast<const T*>(p.x);
  const T* rows[4];
  bool has[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    has[i] = m0 + 8 * i + g < count;
    rows[i] = x + (first + (has[i] ? m0 + 8 * i + g : 0)) * p.x_stride;
  }
  const T* a = static_cast<const T*>(p.a) + (static_cast<int64_t>(l) * R + g) * p.k;
  if (m0 < count) {
    for (int c0 = k0 + wk * 32; c0 < k1; c0 += kw * 32 * kUnroll) {
      uint4 xv[kUnroll][4], av[kUnroll][NT];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int col = c0 + u * kw * 32 + 8 * q;
        const bool in = col < k1;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          av[u][t] = in ? __ldg(reinterpret_cast<const uint4*>(a + static_cast<int64_t>(8 * t) * p.k + col)) : zero;
#pragma unroll
        for (int i = 0; i < 2; ++i) xv[u][i] = in && has[i] ? __ldg(reinterpret_cast<const uint4*>(rows[i] + col)) : zero;
        if (second) {
#pragma unroll
          for (int i = 2; i < 4; ++i) xv[u][i] = in && has[i] ? __ldg(reinterpret_cast<const uint4*>(rows[i] + col)) : zero;
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_16816<T>(acc[0][t], xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y, av[u][t].x, av[u][t].y);
          mma_16816<T>(acc[0][t], xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w, av[u][t].z, av[u][t].w);
        }
        if (second) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_16816<T>(acc[1][t], xv[u][2].x, xv[u][3].x, xv[u][2].y, xv[u][3].y, av[u][t].x, av[u][t].y);
            mma_16816<T>(acc[1][t], xv[u][2].z, xv[u][3].z, xv[u][2].w, xv[u][3].w, av[u][t].z, av[u][t].w);
          }
        }
      }
    }
  }
  float* mine = red + warp * 32 * R;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1 && !second) break;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      *reinterpret_cast<float2*>(mine + (16 * h + g) * R + 8 * t + 2 * q) = make_float2(acc[h][t][0], acc[h][t][1]);
      *reinterpret_cast<float2*>(mine + (16 * h + g + 8) * R + 8 * t + 2 * q) = make_float2(acc[h][t][2], acc[h][t][3]);
    }
  }
  __syncthreads();
  // the parts of K of a CTA, in the warps' order, into the first warp's place
  const int cells = count * (R / 4);
  float4* red4 = reinterpret_cast<float4*>(red);
  auto place = [&](int e) { return (e / (32 * (R / 4))) * kw * (32 * (R / 4)) + e % (32 * (R / 4)); };
  if (kw > 1) {
    for (int e = threadIdx.x; e < cells; e += kThreads) {
      float4* at = red4 + place(e);
      float4 s = *at;
      for (int w = 1; w < kw; ++w) {
        const float4 v = at[w * 32 * (R / 4)];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      *at = s;
    }
  }
  float4* out = reinterpret_cast<float4*>(p.t + first * R);
  if (p.parts == 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < cells; e += kThreads) out[e] = red4[place(e)];
    return;
  }
  cluster_barrier();
  for (int e = threadIdx.x * p.parts + part; e < cells; e += kThreads * p.parts) {
    const float* at = reinterpret_cast<const float*>(red4 + place(e));
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r < p.parts; ++r) {
      const float4 v = remote_float4(at, r);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    out[e] = s;
  }
  cluster_barrier();  // no CTA leaves while its sums are read
}

template <typename T, int R>
__global__ void __launch_bounds__(kThreads) multi_lora_expand_kernel(const MultiLoraParams p) {
  constexpr int KS = R / 16;   // steps of the contraction
  constexpr int kPer = R / 4;  // its elements that a lane holds: [q kPer, (q + 1) kPer), four to a step
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  int64_t first;
  int count, l;
  if (!slot_of<kTile>(p, blockIdx.x / p.chunks, lane, first, count, l, false)) return;
  const int c_lo = blockIdx.x % p.chunks * kCols, c_hi = min(p.n, c_lo + kCols);
  const int mw = count <= 16 ? 1 : count <= 32 ? 2 : count <= 64 ? 4 : 8, nw = kWarps / mw;
  const int m0 = warp / nw * 16, wn = warp % nw;
  if (m0 >= count) return;
  const bool has0 = m0 + g < count, has1 = m0 + g + 8 < count;
  const int64_t n0 = first + m0 + g, n1 = n0 + 8;
  const T* add0 = static_cast<const T*>(p.y_add) + n0 * p.y_add_stride;
  const T* add1 = static_cast<const T*>(p.y_add) + n1 * p.y_add_stride;
  T* y0 = static_cast<T*>(p.y) + n0 * p.n;
  T* y1 = static_cast<T*>(p.y) + n1 * p.n;
  if (l < 0) {  // no adapter: y_add as it is
    if (p.y == p.y_add) return;
    for (int c = c_lo + wn * 32 + 8 * q; c < c_hi; c += nw * 32) {
      if (has0) *reinterpret_cast<uint4*>(y0 + c) = *reinterpret_cast<const uint4*>(add0 + c);
      if (has1) *reinterpret_cast<uint4*>(y1 + c) = *reinterpret_cast<const uint4*>(add1 + c);
    }
    return;
  }
  // T of rows g and g + 8 as hi + lo
  uint32_t hi[KS][4], lo[KS][4];  // registers 0 and 2 row g, 1 and 3 row g + 8
  float f0 = p.scale[l], f1 = f0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool has = r ? has1 : has0;
    float t[kPer];
    const float4* src = reinterpret_cast<const float4*>(p.t + (r ? n1 : n0) * R + q * kPer);
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) {
      const float4 v = has ? src[i] : make_float4(0.f, 0.f, 0.f, 0.f);
      t[4 * i] = v.x;
      t[4 * i + 1] = v.y;
      t[4 * i + 2] = v.z;
      t[4 * i + 3] = v.w;
    }
    float up = 1.f;
    if (std::is_same<T, __half>::value) {  // the row's largest at 2^8 or below it
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) mx = fmaxf(mx, fabsf(t[i]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = (__float_as_int(mx) >> 23) - 127;
      e = mx == 0.f || e > 127 ? 8 : e < -100 ? -100 : e > 100 ? 100 : e;
      up = pow2(8 - e);
      (r ? f1 : f0) *= pow2(e - 8);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float u = t[4 * s + 2 * i] * up, v = t[4 * s + 2 * i + 1] * up;
        const uint32_t h = Half16<T>::pack(u, v);
        const float2 back = Half16<T>::unpack(h);
        // what is not finite has no rest
        hi[s][2 * i + r] = h;
        lo[s][2 * i + r] = Half16<T>::pack(fabsf(back.x) < INFINITY ? u - back.x : 0.f, fabsf(back.y) < INFINITY ? v - back.y : 0.f);
      }
  }
  const T* b = static_cast<const T*>(p.b) + static_cast<int64_t>(l) * p.n * R + q * kPer;
  for (int c0 = c_lo + wn * 32; c0 < c_hi; c0 += nw * 32) {
    // column 2 q' + e of MMA j is column 8 q' + 2 j + e of the thirty-two
    uint2 bv[4][KS];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int col = c0 + 8 * (g >> 1) + 2 * j + (g & 1);
      const uint2* src = reinterpret_cast<const uint2*>(b + static_cast<int64_t>(col < p.n ? col : 0) * R);
      if constexpr (KS % 2 == 0) {
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + s));
          bv[j][s] = make_uint2(v.x, v.y);
          bv[j][s + 1] = make_uint2(v.z, v.w);
        }
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) bv[j][s] = __ldg(src + s);
      }
    }
    const int c = c0 + 8 * q;
    const bool in = c < c_hi;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint4 v0 = in && has0 ? *reinterpret_cast<const uint4*>(add0 + c) : zero;
    const uint4 v1 = in && has1 ? *reinterpret_cast<const uint4*>(add1 + c) : zero;
    float o0[8], o1[8];
    unpack8<T>(v0, o0);
    unpack8<T>(v1, o1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) mma_16816<T>(d, lo[s][0], lo[s][1], lo[s][2], lo[s][3], bv[j][s].x, bv[j][s].y);
#pragma unroll
      for (int s = 0; s < KS; ++s) mma_16816<T>(d, hi[s][0], hi[s][1], hi[s][2], hi[s][3], bv[j][s].x, bv[j][s].y);
      o0[2 * j] = fmaf(f0, d[0], o0[2 * j]);
      o0[2 * j + 1] = fmaf(f0, d[1], o0[2 * j + 1]);
      o1[2 * j] = fmaf(f1, d[2], o1[2 * j]);
      o1[2 * j + 1] = fmaf(f1, d[3], o1[2 * j + 1]);
    }
    if (in && has0) *reinterpret_cast<uint4*>(y0 + c) = pack8<T>(o0);
    if (in && has1) *reinterpret_cast<uint4*>(y1 + c) = pack8<T>(o1);
  }
}

int64_t slots_of(int64_t tokens, int batch, bool ragged, int size) {
  if (ragged) return tokens / size + batch;
  const int64_t t_new = tokens / batch;
  return (t_new + size - 1) / size * batch;
}

template <typename T, int R>
int multi_lora_t(MultiLoraParams p, cudaStream_t st, int num_sms) {
  const int64_t slots = slots_of(p.tokens, p.batch, p.q_start != nullptr, kSlot);
  // parts of K: as many as give every SM some eight CTAs, of 256 columns at least
  int parts = 1;
  while (parts < kMaxParts && slots * parts * 2 <= 8ll * num_sms && p.k > 256 * parts) parts *= 2;
  p.parts = parts;
  p.part_cols = ((p.k + parts - 1) / parts + 31) / 32 * 32;
  constexpr int smem = kWarps * 32 * R * 4;
  auto* shrink = multi_lora_shrink_kernel<T, R>;
  if (smem > 48 * 1024 && !set_smem_limit(shrink, smem)) return FITQ_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(slots * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(parts);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, shrink, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  const int64_t tiles = slots_of(p.tokens, p.batch, p.q_start != nullptr, kTile);
  p.chunks = (p.n + kCols - 1) / kCols;
  e = launch_pdl(multi_lora_expand_kernel<T, R>, dim3(static_cast<unsigned>(tiles * p.chunks)), dim3(kThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T>
int multi_lora_sized(const MultiLoraParams& p, int rank, cudaStream_t st, int num_sms) {
  if (rank == 16) return multi_lora_t<T, 16>(p, st, num_sms);
  if (rank == 32) return multi_lora_t<T, 32>(p, st, num_sms);
  if (rank == 48) return multi_lora_t<T, 48>(p, st, num_sms);
  return multi_lora_t<T, 64>(p, st, num_sms);
}

}  // namespace

size_t multi_lora_workspace(int64_t tokens, int64_t, int64_t, int rank, int, int) {
  return static_cast<size_t>(tokens > 0 ? tokens : 1) * rank * sizeof(float);
}

int launch_multi_lora(const void* x, int64_t x_stride, int64_t tokens, int64_t k, int64_t n, const void* a,
                      const void* b, int rank, int adapters, const float* scale, const int32_t* adapter,
                      const int32_t* q_start, int batch, const void* y_add, int64_t y_add_stride, void* y, int dtype,
                      void* workspace, int* status, cudaStream_t st, int num_sms) {
  const MultiLoraParams p{x, a, b, y_add, y, scale, adapter, q_start, tokens, x_stride, y_add_stride, batch, adapters,
                          static_cast<int>(k), static_cast<int>(n), q_start ? 0 : static_cast<int>(tokens / batch), 0, 0, 0,
                          static_cast<float*>(workspace), status};
  return dtype == FITQ_DTYPE_BF16 ? multi_lora_sized<__nv_bfloat16>(p, rank, st, num_sms)
                                  : multi_lora_sized<__half>(p, rank, st, num_sms);
}

}  // namespace fitq
