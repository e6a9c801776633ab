// Low-rank adapters of many requests beside a shared projection:
//   y[n] = y_add[n] + s_l (x[n].A_l^T).B_l^T,   l = adapter of token n's sequence.
//
// An adapter's R columns or rows give it a few operations per byte: the bytes of x, A, B and y are
// what costs.  Few tokens, and the second product, whose contraction is R long, run on mma.sync m16n8k16.
//
// Tokens are taken in slots of up to kSlot of one sequence.  Slot numbers need no counting:
// sequence b, whose tokens begin at q_start[b], owns the numbers from q_start[b] / kSlot + b
// on, which leaves room for its slots whatever the lengths, so that the host launches
// tokens / kSlot + batch of them without knowing any.
//
// multi_lora_shrink_kernel, T = x.A_l^T: a cluster of up to eight CTAs shares a slot, each a part of
// K.  Up to sixteen tokens: the eight warps split the part again, and a lane reads 16 bytes of a
// row of x and of A at a time and feeds them to two MMAs (the contraction index is permuted
// alike in both), so that a single token is summed by 64 warps with every load in flight at
// once.  More: tcgen05, M = 128 tokens by N = R, x and A through a ring of TMA tiles of 64 columns (a
// full slot's x is one copy, as four from one lane are issued too slowly).  Parts join in shared memory, then over
// the cluster, in order (deterministic); T stays in fp32.  The accumulation in tensor memory rounds towards zero:
// where one CTA sums all of K = 27,648 the result's error is 1.2% above its own rounding's in fp16, 0.02% in bf16.
//
// multi_lora_expand_kernel, y = y_add + s T.B_l^T: T enters as two 16-bit numbers, hi + lo (a
// relative error of eps^2; one alone would cost the delta half its digits), scaled by a power of
// two per token for fp16's range.  The columns of four MMAs are dealt so that a lane's are eight in a
// row: y and y_add move in 16-byte pieces.  One rounding, of y.
//
// Bound: one token, two launches (5.3 us at K = N = 5,120, rank 16); 64 tokens of as many adapters on 5,120 x
// 27,648: 23 us, B at 2.9 TB/s, as a CTA waits for its adapter, T and B in turn; one token at K = 27,648, rank 64:
// 12.4 us, as a slot has eight CTAs at most and they read 3.5 MB of A; six prompts of 4,180
// tokens on 27,648 x 5,120 at rank 64: 88 us, 50 of them the first kernel's (x at 4.3 TB/s, with A 7 TB/s into
// the SMs), 33 the second's, whose loads and mma.sync (36% busy) wait for each other.
#include <type_traits>

#include "kernels.cuh"
#include "kv4.cuh"
#include "umma_warp.cuh"

namespace fitq {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kSlot = 128;       // tokens of a slot: 16 for each warp
constexpr int kCols = 256;       // columns of a CTA of the second kernel for more than sixteen tokens
constexpr int kAhead = 4;        // of their groups of 32, those whose y_add is on its way
constexpr int kMaxParts = 8;     // CTAs of a cluster
constexpr int kBox = 32;         // tokens of a copy where a slot is not full: few behind its last one are read

struct MultiLoraParams {
  const void *x, *a, *b, *y_add;
  void* y;
  const float* scale;
  const int32_t* adapter;
  const int32_t* q_start;
  int64_t tokens, x_stride, y_add_stride;
  int batch, adapters, k, n, t_new;
  int parts;       // of K
  int part_cols;   // columns of a part, a multiple of 64
  int chunks;      // parts of N
  float* t;        // [tokens][rank]
  int* status;
};

__device__ __forceinline__ int start_of(const MultiLoraParams& p, int64_t b) {
  const int q = p.q_start[b];
  return q < 0 ? 0 : q > p.tokens ? static_cast<int>(p.tokens) : q;
}
// The last sequence b < p.batch for which before(q_start[b], b) holds, or -1: 32 candidates at a time, every lane the
// same answer.  Starts are clamped to the tokens; `mine` is the lane's.
template <typename F>
__device__ __forceinline__ int64_t last_sequence(const MultiLoraParams& p, int lane, int mine, F before) {
  if (p.batch <= 32) {
    const uint32_t no = ~__ballot_sync(0xffffffffu, lane < p.batch && before(mine, lane));
    return no ? __ffs(no) - 2 : 31;
  }
  int64_t lo = 0, hi = p.batch;  // answer + 1 in [lo, hi]
  while (lo < hi) {
    const int64_t span = hi - lo, step = (span + 31) / 32;
    const int64_t at = lo + (lane + 1) * step - 1;  // asks whether the answer lies behind
    const uint32_t no = ~__ballot_sync(0xffffffffu, at < hi && before(start_of(p, at), static_cast<int>(at)));
    const int n = no ? __ffs(no) - 1 : 32;  // leading candidates that say yes
    const int64_t up = lo + (n + 1) * step - 1;
    lo += n * step;
    if (n < 32 && up < hi) hi = up;
    if (lo > hi) lo = hi;
  }
  return lo - 1;
}

// Tokens [first, first + count) of slot number s (slots of kSize), and their adapter (-1: none).  Where starts fall
// sequences may share tokens: each then belongs to the last sequence that begins at or before it, as the search
// finds it.  That sequence does not fall as the token rises (a candidate's yes stays one), so that a slot whose first
// and last tokens are its sequence's own meets no other slot; a slot that has others' is left out.
template <int kSize>
__device__ __forceinline__ bool slot_of(const MultiLoraParams& p, int64_t s, int lane, int64_t& first, int& count, int& l,
                                        bool report) {
  int64_t b;
  bool own = true;
  if (p.q_start == nullptr) {
    const int per = (p.t_new + kSize - 1) / kSize;
    b = s / per;
    if (b >= p.batch) return false;
    first = b * p.t_new + (s - b * per) * kSize;
    const int64_t left = (b + 1) * p.t_new - first;
    count = static_cast<int>(left < kSize ? left : kSize);
    l = p.adapter[b];
  } else {
    const int mine = lane < p.batch ? start_of(p, lane) : 0;
    b = last_sequence(p, lane, mine, [&](int q, int at) { return q / kSize + at <= s; });
    if (b < 0) return false;
    int64_t begin = p.q_start[b], end = p.q_start[b + 1];
    begin = begin < 0 ? 0 : begin;
    end = end > p.tokens ? p.tokens : end;
    if (begin > p.tokens) return false;
    first = begin + (s - (begin / kSize + b)) * kSize;
    if (first < begin || first >= end) return false;
    count = static_cast<int>(end - first < kSize ? end - first : kSize);
    l = p.adapter[b];
    own = last_sequence(p, lane, mine, [&](int q, int) { return q <= first; }) == b &&
          last_sequence(p, lane, mine, [&](int q, int) { return q < first + count; }) == b;
  }
  if (l < -1 || l >= p.adapters) {
    if (report && lane == 0) report_device_error(p.status, FITQ_ERR_ARG);
    l = -1;
  }
  return own;
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

__device__ __forceinline__ void cp16_zfill(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Stages of the first kernel's copies: 64 columns of a slot's tokens and of A, as many as leave an SM
// room for two CTAs (twice as many for one CTA: no faster where the SMs have equal shares, and slower where
// clusters then find no place).
template <int R>
struct ShrinkSmem {
  static constexpr int kX = kSlot * 128, kA = R * 128, kStage = kX + kA;
  static constexpr int kStages = R <= 32 ? 5 : 4;
  static constexpr int kPitch = R + 4;              // floats of a token's sums: 16-byte stores of eight rows meet no bank twice
  static constexpr int kRed = kWarps * 16 * R * 4;  // up to sixteen tokens: the warps' sums
  static constexpr int kMany = kStages * kStage + 1024;
  static constexpr uint32_t kTmem = R <= 32 ? 32 : 64;
  static_assert(kSlot * kPitch * 4 <= kStages * kStage && kRed <= kMany, "the sums take the stages' place");
};

// kMany: some slot may have more than sixteen tokens.  tm_s and tm_x: x in copies of kSlot and kBox tokens.
template <typename T, int R, bool kMany>
__global__ void __launch_bounds__(kThreads, 2)
    multi_lora_shrink_kernel(const __grid_constant__ CUtensorMap tm_s, const __grid_constant__ CUtensorMap tm_x,
                             const __grid_constant__ CUtensorMap tm_a, const MultiLoraParams p) {
  constexpr int NT = R / 8;
  constexpr int kUnroll = R == 16 ? 4 : R == 32 ? 3 : 2;  // what the registers hold beside the sums
  using L = ShrinkSmem<R>;
  float* red = reinterpret_cast<float*>(g_lora_smem);     // [warps][16][R]
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int part = blockIdx.x % p.parts;
  int64_t first;
  int count, l, begin = 0, end = 0;
  // starts that fall or leave the tokens are recorded: there are as many slots as sequences, or more
  const bool looks = p.q_start != nullptr && part == 0 && threadIdx.x == kThreads - 1 && blockIdx.x / p.parts < p.batch;
  if (looks) {
    begin = p.q_start[blockIdx.x / p.parts];
    end = p.q_start[blockIdx.x / p.parts + 1];
  }
  const bool own = slot_of<kSlot>(p, blockIdx.x / p.parts, lane, first, count, l, part == 0 && warp == 0);
  if (looks && (begin < 0 || end < begin || end > p.tokens)) report_device_error(p.status, FITQ_ERR_ARG);
  if (!own || l < 0) return;  // the whole cluster
  const int k0 = part * p.part_cols, k1 = min(p.k, k0 + p.part_cols);
  const T* x = static_cast<const T*>(p.x) + first * p.x_stride;
  const T* a = static_cast<const T*>(p.a) + static_cast<int64_t>(l) * R * p.k;
  const bool few = !kMany || count <= 16;
  float acc[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
  if (few) {
    // ---- every warp has all tokens and columns of its own, loaded straight into fragments
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const bool has0 = g < count, has1 = g + 8 < count;
    const T* x0 = x + (has0 ? g : 0) * p.x_stride;
    const T* x1 = x + (has1 ? g + 8 : 0) * p.x_stride;
    const T* ag = a + static_cast<int64_t>(g) * p.k;
    for (int c0 = k0 + warp * 32; c0 < k1; c0 += kWarps * 32 * kUnroll) {
      uint4 xv[kUnroll][2], av[kUnroll][NT];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int col = c0 + u * kWarps * 32 + 8 * q;
        const bool in = col < k1;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          av[u][t] = in ? __ldg(reinterpret_cast<const uint4*>(ag + static_cast<int64_t>(8 * t) * p.k + col)) : zero;
        xv[u][0] = in && has0 ? __ldg(reinterpret_cast<const uint4*>(x0 + col)) : zero;
        xv[u][1] = in && has1 ? __ldg(reinterpret_cast<const uint4*>(x1 + col)) : zero;
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma_16816<T>(acc[t], xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y, av[u][t].x, av[u][t].y);
          mma_16816<T>(acc[t], xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w, av[u][t].z, av[u][t].w);
        }
    }
  } else if constexpr (kMany) {
    // ---- 64 columns at a time: TMA by warp 0, MMAs of 128 tokens x R by warp 1.  Rows of the tile behind the
    // slot's tokens hold another sequence's or nothing that was written: only their own sums see them.
    __shared__ uint64_t b_full[L::kStages], b_free[L::kStages], b_done;
    __shared__ uint32_t sh_tmem;
    __shared__ int sh_abort;
    const int steps = k1 > k0 ? (k1 - k0 + 63) / 64 : 0;
    uint8_t* ring = reinterpret_cast<uint8_t*>(g_lora_smem) + ((1024u - (smem_u32(g_lora_smem) & 1023u)) & 1023u);
    red = reinterpret_cast<float*>(ring);
    if (threadIdx.x == 0) {
      for (int i = 0; i < L::kStages; ++i) {
        mbar_init(&b_full[i], 1);
        mbar_init(&b_free[i], 1);
      }
      mbar_init(&b_done, 1);
      fence_mbar_init();
      sh_abort = 0;
    }
    if (warp == 1) {
      tmem_alloc(&sh_tmem, L::kTmem);
      tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh_tmem;
    if (warp == 0) {
      const int rows = count > kSlot - kBox ? kSlot : kBox;
      const int boxes = (count + rows - 1) / rows;
      const CUtensorMap* map = lane < boxes ? (rows == kSlot ? &tm_s : &tm_x) : &tm_a;  // a lane per copy
      const int y = lane < boxes ? static_cast<int>(first) + lane * rows : l * R;
      uint8_t* dst = ring + (lane < boxes ? lane * (rows * 128) : L::kX);
      int s = 0, at = 0;
      uint32_t phase = 1;  // of the stage's release
      bool ok = true;
      for (; s < steps; ++s) {
        if (s >= L::kStages) ok = mbar_wait_warp(&b_free[at], phase, &sh_abort, p.status);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&b_full[at], boxes * (rows * 128) + L::kA);
        __syncwarp();
        if (lane <= boxes) tma_load_2d(dst + at * L::kStage, map, &b_full[at], k0 + 64 * s, y);
        if (++at == L::kStages) {
          at = 0;
          phase ^= 1;
        }
      }
      if (!ok) {  // the copies in flight land before their place is used again
        int never = 0;
        for (int i = s > L::kStages ? s - L::kStages : 0; i < s; ++i)
          mbar_wait_warp(&b_full[i % L::kStages], i / L::kStages & 1, &never, p.status);
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) |
                                 (static_cast<uint32_t>(R >> 3) << 17) | (static_cast<uint32_t>(kSlot >> 4) << 24);
      const uint64_t dx = umma_smem_desc_sw128(smem_u32(ring)), da = umma_smem_desc_sw128(smem_u32(ring) + L::kX);
      uint32_t at = 0, phase = 0;
      for (int s = 0; s < steps; ++s) {
        if (!mbar_wait_warp(&b_full[at], phase, &sh_abort, p.status)) break;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          umma_f16_ss(tmem, dx + ((at * L::kStage + kk * 32) >> 4), da + ((at * L::kStage + kk * 32) >> 4), idesc,
                      s > 0 || kk > 0 ? 1u : 0u);
        commit_warp(&b_free[at]);
        if (++at == static_cast<uint32_t>(L::kStages)) {
          at = 0;
          phase ^= 1;
        }
      }
      commit_warp(&b_done);
      int never = 0;
      mbar_wait_warp(&b_done, 0, &never, p.status);
    }
    __syncthreads();  // the stages' place becomes the sums'
    tc_fence_after();
    const int row = 32 * (warp & 3) + lane;
    for (int c = 16 * (warp >> 2); c < R; c += 32) {
      uint32_t v[16];
      tmem_ld_x16(tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(red + row * L::kPitch + c + i) =
            steps > 0 ? make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]))
                      : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
      tc_fence_after();
      tmem_dealloc(tmem, L::kTmem);
    }
  }
  const int cells = count * (R / 4);
  float4* red4 = reinterpret_cast<float4*>(red);
  if (few) {  // the warps' sums in order, into the first warp's place
    float* mine = red + warp * 16 * R;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      *reinterpret_cast<float2*>(mine + g * R + 8 * t + 2 * q) = make_float2(acc[t][0], acc[t][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * R + 8 * t + 2 * q) = make_float2(acc[t][2], acc[t][3]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < cells; e += kThreads) {
      float4 s = red4[e];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 v = red4[e + w * 16 * (R / 4)];
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      red4[e] = s;
    }
  }
  float4* out = reinterpret_cast<float4*>(p.t + first * R);
  auto cell = [&](int e) { return few ? e : e + e / (R / 4) * ((L::kPitch - R) / 4); };
  if (p.parts == 1) {
    __syncthreads();
    for (int e = threadIdx.x; e < cells; e += kThreads) out[e] = red4[cell(e)];
    return;
  }
  cluster_barrier();
  for (int e = threadIdx.x * p.parts + part; e < cells; e += kThreads * p.parts) {
    const float* at = reinterpret_cast<const float*>(red4 + cell(e));
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

// Groups of 32 columns that a warp of a slot of few tokens loads at once.
template <int R>
constexpr int few_groups() { return R == 16 ? 4 : R == 32 ? 2 : 1; }

// kMany as above; the grid has p.chunks parts of N for every slot, of kCols columns or, where
// no slot has more than sixteen tokens, of all that eight warps load at once.
template <typename T, int R, bool kMany>
__global__ void __launch_bounds__(kThreads, 2) multi_lora_expand_kernel(const MultiLoraParams p) {
  constexpr int KS = R / 16;   // steps of the contraction
  constexpr int kPer = R / 4;  // its elements that a lane holds: [q kPer, (q + 1) kPer), four to a step
  constexpr int kGroups = few_groups<R>(), kFewCols = kGroups * 32 * kWarps;
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  int64_t first;
  int count, l;
  if (!slot_of<kSlot>(p, blockIdx.x / p.chunks, lane, first, count, l, false)) return;
  const bool few = !kMany || count <= 16;
  const int chunk = blockIdx.x % p.chunks, cols = few ? kFewCols : kCols;
  const int64_t c_first = static_cast<int64_t>(chunk) * cols;
  if (c_first >= p.n) return;  // the slot has fewer parts than the grid
  const int c_lo = static_cast<int>(c_first), c_hi = min(p.n, c_lo + cols);
  const int nw = few ? kWarps : 1, m0 = few ? 0 : warp * 16, wn = few ? warp : 0;
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
  const T* b = static_cast<const T*>(p.b) + static_cast<int64_t>(l) * p.n * R;
  // many tokens: the CTA's columns of B in shared memory, rows of 2 R bytes, 16-byte piece c of row r at
  // c ^ (the bits of r in which a load's eight rows differ)
  const uint32_t s_b = smem_u32(g_lora_smem);
  auto b_at = [&](int row, int piece) {
    const int mix = ((row & 1) | ((row >> 3) & 3) << 1) & (R % 64 == 0 ? 7 : R % 32 == 0 ? 3 : R == 16 ? 1 : 0);
    return s_b + row * (2 * R) + ((piece ^ mix) << 4);
  };
  if (kMany && !few) {
    for (int e = threadIdx.x; e < kCols * (R / 8); e += kThreads) {
      const int row = e / (R / 8), piece = e % (R / 8);
      const bool in = c_lo + row < p.n;
      cp16_zfill(b_at(row, piece), b + static_cast<int64_t>(in ? c_lo + row : 0) * R + piece * 8, in ? 16u : 0u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // column 2 q' + e of MMA j is column 8 q' + 2 j + e of the thirty-two
  constexpr int kSets = kMany && kAhead > kGroups ? kAhead : kGroups;
  uint2 bv[kGroups][4][KS];
  uint4 v0[kSets], v1[kSets];
  auto load_y = [&](int u, int cu) {
    const int c = cu + 8 * q;
    v0[u] = c < c_hi && has0 ? *reinterpret_cast<const uint4*>(add0 + c) : zero;
    v1[u] = c < c_hi && has1 ? *reinterpret_cast<const uint4*>(add1 + c) : zero;
  };
  auto load = [&](int c0) {
#pragma unroll
    for (int u = 0; u < kGroups; ++u) {
      const int cu = c0 + u * nw * 32;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = cu + 8 * (g >> 1) + 2 * j + (g & 1);
        const uint2* src = reinterpret_cast<const uint2*>(b + static_cast<int64_t>(col < c_hi ? col : 0) * R + q * kPer);
        if constexpr (KS % 2 == 0) {
#pragma unroll
          for (int s = 0; s < KS; s += 2) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + s));
            bv[u][j][s] = make_uint2(v.x, v.y);
            bv[u][j][s + 1] = make_uint2(v.z, v.w);
          }
        } else {
#pragma unroll
          for (int s = 0; s < KS; ++s) bv[u][j][s] = __ldg(src + s);
        }
      }
      load_y(u, cu);
    }
  };
  const int c0 = c_lo + wn * 32;
  if (few)  // on their way while T is made ready
    load(c0);
  else if constexpr (kMany) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) load_y(u, c0 + 32 * u);
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
  auto finish = [&](int u, int c, const uint2 (&w)[4][KS]) {  // y of the eight columns from c on
    float o0[8], o1[8];
    unpack8<T>(v0[u], o0);
    unpack8<T>(v1[u], o1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KS; ++s) mma_16816<T>(d, lo[s][0], lo[s][1], lo[s][2], lo[s][3], w[j][s].x, w[j][s].y);
#pragma unroll
      for (int s = 0; s < KS; ++s) mma_16816<T>(d, hi[s][0], hi[s][1], hi[s][2], hi[s][3], w[j][s].x, w[j][s].y);
      o0[2 * j] = fmaf(f0, d[0], o0[2 * j]);
      o0[2 * j + 1] = fmaf(f0, d[1], o0[2 * j + 1]);
      o1[2 * j] = fmaf(f1, d[2], o1[2 * j]);
      o1[2 * j + 1] = fmaf(f1, d[3], o1[2 * j + 1]);
    }
    if (c < c_hi && has0) *reinterpret_cast<uint4*>(y0 + c) = pack8<T>(o0);
    if (c < c_hi && has1) *reinterpret_cast<uint4*>(y1 + c) = pack8<T>(o1);
  };
  if (few) {
#pragma unroll
    for (int u = 0; u < kGroups; ++u) finish(u, c0 + u * nw * 32 + 8 * q, bv[u]);
  } else if constexpr (kMany) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
#pragma unroll 1
    for (int g0 = 0; g0 < kCols / 32; g0 += kAhead) {
      if (c_lo + 32 * g0 >= c_hi) break;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        uint2 w[4][KS];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 32 * (g0 + u) + 8 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int byte = q * 2 * kPer + 8 * s;
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[j][s].x), "=r"(w[j][s].y) : "r"(b_at(row, byte >> 4) + (byte & 15)));
          }
        }
        const int c = c_lo + 32 * (g0 + u);
        finish(u, c + 8 * q, w);
        load_y(u, c + 32 * kAhead);
      }
    }
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
  // Parts of K, of 256 columns at least.  Slots are counted as a batch of any lengths has them on average (a
  // sequence's last one half full), so that the sums do not depend on how the lengths were passed.  Few
  // tokens: as many parts as find room at once, two CTAs on an SM, a power of two.  Many: a CTA for every SM, or
  // two parts where that leaves some without (36 slots, K = 27,648, rank 64, 1 to 8 parts: 131, 77, 63, 59,
  // 57, 59, 76 us; 118 slots: 158, 140, 161, 150; 47 slots, K = 5,120: 32, 24, 25, 25, 27).
  const int64_t half = p.tokens / kSlot + p.batch / 2, real = half > p.batch ? half : p.batch;
  const bool prompts = p.tokens > 16ll * p.batch;
  int parts = 1;
  if (prompts) {
    while (parts < kMaxParts && real * (parts + 1) <= (parts == 1 ? 2ll * num_sms : num_sms) && p.k > 256 * parts) ++parts;
  } else {
    while (parts < kMaxParts && real * parts * 2 <= 2ll * num_sms && p.k > 256 * parts) parts *= 2;
  }
  p.parts = parts;
  p.part_cols = ((p.k + parts - 1) / parts + 63) / 64 * 64;
  const bool many = p.q_start != nullptr ? p.tokens > 16 : p.t_new > 16;
  CUtensorMap ts{}, tx{}, ta{};
  if (many) {
    const auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    if (!encode_tmap_2d(&ts, type, p.x, p.k, p.tokens, p.x_stride * 2, 64, kSlot, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
        !encode_tmap_2d(&tx, type, p.x, p.k, p.tokens, p.x_stride * 2, 64, kBox, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B) ||
        !encode_tmap_2d(&ta, type, p.a, p.k, static_cast<uint64_t>(p.adapters) * R, p.k * 2, 64, R, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B))
      return FITQ_ERR_CUDA;
  }
  const int smem = many ? ShrinkSmem<R>::kMany : ShrinkSmem<R>::kRed;
  auto* shrink = many ? multi_lora_shrink_kernel<T, R, true> : multi_lora_shrink_kernel<T, R, false>;
  if (many && !set_smem_limit(shrink, ShrinkSmem<R>::kMany)) return FITQ_ERR_CUDA;
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, shrink, ts, tx, ta, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  const int cols = many ? kCols : few_groups<R>() * 32 * kWarps;
  p.chunks = (p.n + cols - 1) / cols;
  auto* expand = many ? multi_lora_expand_kernel<T, R, true> : multi_lora_expand_kernel<T, R, false>;
  e = launch_pdl(expand, dim3(static_cast<unsigned>(slots * p.chunks)), dim3(kThreads), many ? kCols * R * 2 : 0, st, p);
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
