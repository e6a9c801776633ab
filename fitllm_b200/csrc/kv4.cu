// Append to and read from the 4-bit paged key/value cache (layout: kv4.cuh).
//
// kv4_append_kernel: for every new token the queries and keys are rotated
// (rotate-half, fp32 tables indexed by the token's absolute position), the
// queries are written out in their own type, and the rotated keys (in fp32, not
// rounded first) and the values are coded in groups of 64:
//   low = fp16(min), scale = fp16((max - low) / 15),
//   code = round((x - low) * (1 / scale)) in 0..15, 0 where scale is 0,
// every difference, product and quotient rounded to fp32 on its own (no fused
// multiply-add: a code next to a border is then the same wherever it is
// computed).  A group that holds a NaN, an infinity or a value fp16 cannot
// reach gets a non-finite scale and reads back as NaN.
//
// Bound: HBM (q, k, v in, q and the blocks out) for prompts, the launch for a
// decode step.
#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kAppThreads = 256;

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Kv4AppendParams {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements per token
  void* q_out;                           // [tokens, H, D]
  uint8_t* pool;
  const float *cs, *sn;  // [rope_len, D / 2]
  int rope_len, heads;
  int* status;
  Kv4Seq seq;
};

// Eight codes of x under (low, inv), packed low nibble first.
__device__ __forceinline__ uint32_t code8(const float (&x)[8], float low, float inv) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int c = __float2int_rn(__fmul_rn(__fsub_rn(x[i], low), inv));
    c = c < 0 ? 0 : (c > 15 ? 15 : c);
    w |= static_cast<uint32_t>(c) << (4 * i);
  }
  return w;
}

// One CTA per token (blockIdx.x) and share of its head slots (blockIdx.y); a
// team of D / 16 lanes holds one head: lane i elements 8 i .. 8 i + 7 of each
// half, so the rotation pairs meet in one lane and the group extrema take
// log2(team) shuffles.
template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int kTeam = D / 16;
  constexpr int kTeams = kAppThreads / kTeam;
  constexpr int kHalf = D / 2;
  const int lane = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
  pdl_launch_dependents();
  pdl_wait();  // q, k, v come from the previous kernel
  const int64_t n = blockIdx.x;
  const Kv4Seq& s = p.seq;
  const int b = kv4_sequence(s, n);
  if (b < 0) return;  // a token of no sequence: left as it is
  const int64_t first = s.q_start ? s.q_start[b] : static_cast<int64_t>(b) * s.t_new;
  const int pre = s.prefix[b];
  const int64_t pos = pre + (n - first);
  const int pg = pre < 0 ? -1 : kv4_page(s, b, pos);
  const bool ok = pg >= 0 && pos < p.rope_len;
  if (!ok && threadIdx.x == 0) report_device_error(p.status, FITQ_ERR_ARG);
  float c[8], sv[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = sv[i] = 0.f;  // a refused token's query reads as zeros
  if (ok) {
    const float4* cp = reinterpret_cast<const float4*>(p.cs + pos * kHalf + lane * 8);
    const float4* sp = reinterpret_cast<const float4*>(p.sn + pos * kHalf + lane * 8);
    const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
    c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
    sv[0] = s0.x; sv[1] = s0.y; sv[2] = s0.z; sv[3] = s0.w; sv[4] = s1.x; sv[5] = s1.y; sv[6] = s1.z; sv[7] = s1.w;
  }
  const int slots = p.heads + 2 * s.kv_heads;
  const int bp = static_cast<int>(pos & 15);
  for (int s0 = blockIdx.y * kTeams; s0 < slots; s0 += gridDim.y * kTeams) {
    const int slot = s0 + team;
    const bool is_q = slot < p.heads, is_k = !is_q && slot < p.heads + s.kv_heads;
    const bool is_kv = slot >= p.heads && slot < slots;
    const int kh = is_k ? slot - p.heads : slot - p.heads - s.kv_heads;
    float a[8], bb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = bb[i] = 0.f;
    if (slot < slots) {
      const T* src = is_q ? static_cast<const T*>(p.q) + n * p.q_stride + slot * D
                          : (is_k ? static_cast<const T*>(p.k) + n * p.k_stride
                                  : static_cast<const T*>(p.v) + n * p.v_stride) + kh * D;
      unpack8<T>(*reinterpret_cast<const uint4*>(src + lane * 8), a);
      unpack8<T>(*reinterpret_cast<const uint4*>(src + kHalf + lane * 8), bb);
    }
    if (is_q || is_k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = bb[i];
        a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, sv[i]));
        bb[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, sv[i]));
      }
    }
    if (is_q) {
      if (!ok) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = bb[i] = 0.f;
      }
      T* dst = static_cast<T*>(p.q_out) + (n * p.heads + slot) * D;
      *reinterpret_cast<uint4*>(dst + lane * 8) = pack8<T>(a);
      *reinterpret_cast<uint4*>(dst + kHalf + lane * 8) = pack8<T>(bb);
    }
    if (__any_sync(0xffffffffu, is_kv)) {
      // extrema of the lane's pieces: D = 128 has one group per half, D = 64 one in all
      float lo0 = a[0], hi0 = a[0], lo1 = bb[0], hi1 = bb[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        lo0 = min_nan(lo0, a[i]);
        hi0 = max_nan(hi0, a[i]);
        lo1 = min_nan(lo1, bb[i]);
        hi1 = max_nan(hi1, bb[i]);
      }
      if (D == 64) {
        lo0 = min_nan(lo0, lo1);
        hi0 = max_nan(hi0, hi1);
      }
#pragma unroll
      for (int o = kTeam / 2; o > 0; o >>= 1) {
        lo0 = min_nan(lo0, __shfl_xor_sync(0xffffffffu, lo0, o));
        hi0 = max_nan(hi0, __shfl_xor_sync(0xffffffffu, hi0, o));
        if (D == 128) {
          lo1 = min_nan(lo1, __shfl_xor_sync(0xffffffffu, lo1, o));
          hi1 = max_nan(hi1, __shfl_xor_sync(0xffffffffu, hi1, o));
        }
      }
      if (D == 64) {
        lo1 = lo0;
        hi1 = hi0;
      }
      if (is_kv && ok) {
        const __half l0 = __float2half_rn(lo0), l1 = __float2half_rn(lo1);
        const float f0 = __half2float(l0), f1 = __half2float(l1);
        const __half c0 = __float2half_rn(__fdiv_rn(__fsub_rn(hi0, f0), 15.f));
        const __half c1 = __float2half_rn(__fdiv_rn(__fsub_rn(hi1, f1), 15.f));
        const float g0 = __half2float(c0), g1 = __half2float(c1);
        const uint32_t w0 = code8(a, f0, g0 > 0.f ? __frcp_rn(g0) : 0.f);
        const uint32_t w1 = code8(bb, f1, g1 > 0.f ? __frcp_rn(g1) : 0.f);
        uint32_t* blk = reinterpret_cast<uint32_t*>(p.pool + kv4_block_offset(s, pg, kh, pos, D));
        const __half2 p0 = __halves2half2(c0, l0), p1 = __halves2half2(c1, l1);
        const int side = is_k ? 0 : 1;
        if (D == 128) {
          blk[is_k ? kv4_key_word<D>(bp, 0, lane) : kv4_value_word<D>(bp, 0, lane)] = w0;
          blk[is_k ? kv4_key_word<D>(bp, 1, lane) : kv4_value_word<D>(bp, 1, lane)] = w1;
          if (lane == 0) {
            blk[kv4_param_word<D>(bp, side, 0)] = *reinterpret_cast<const uint32_t*>(&p0);
            blk[kv4_param_word<D>(bp, side, 1)] = *reinterpret_cast<const uint32_t*>(&p1);
          }
        } else {
          blk[is_k ? kv4_key_word<D>(bp, 0, lane) : kv4_value_word<D>(bp, 0, lane)] = w0;
          blk[is_k ? kv4_key_word<D>(bp, 0, 4 + lane) : kv4_value_word<D>(bp, 0, 4 + lane)] = w1;
          if (lane == 0) blk[kv4_param_word<D>(bp, side, 0)] = *reinterpret_cast<const uint32_t*>(&p0);
        }
      }
    }
  }
}

struct Kv4GatherParams {
  const uint8_t* pool;
  void *k, *v;  // [tokens, KVH, D]
  int* status;
  Kv4Seq seq;
};

// One thread per (token, KV head, side, 8 elements): value = scale * code + low
// in fp32, rounded once.
template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads) kv4_gather_kernel(const Kv4GatherParams p) {
  pdl_launch_dependents();
  pdl_wait();  // the pool is written by the previous kernel
  const Kv4Seq& s = p.seq;
  constexpr int kWords = D / 8;
  const int64_t n = blockIdx.x;
  const int b = kv4_sequence(s, n);
  if (b < 0) return;
  const int64_t first = s.q_start ? s.q_start[b] : static_cast<int64_t>(b) * s.t_new;
  const int pre = s.prefix[b];
  const int64_t pos = pre + (n - first);
  const int pg = pre < 0 ? -1 : kv4_page(s, b, pos);
  if (pg < 0 && threadIdx.x == 0) report_device_error(p.status, FITQ_ERR_ARG);
  const int bp = static_cast<int>(pos & 15);
  const int items = s.kv_heads * 2 * kWords;
  for (int i = blockIdx.y * kAppThreads + threadIdx.x; i < items; i += gridDim.y * kAppThreads) {
    const int e = i % kWords, side = (i / kWords) & 1, kh = i / (2 * kWords);
    const int g = e / 8, e8 = e % 8;
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    if (pg >= 0) {
      const uint32_t* blk = reinterpret_cast<const uint32_t*>(p.pool + kv4_block_offset(s, pg, kh, pos, D));
      const uint32_t w = blk[side ? kv4_value_word<D>(bp, g, e8) : kv4_key_word<D>(bp, g, e8)];
      const uint32_t pr = blk[kv4_param_word<D>(bp, side, g)];
      const float2 sl = Half16<__half>::unpack(pr);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = __fadd_rn(__fmul_rn(sl.x, static_cast<float>((w >> (4 * j)) & 15u)), sl.y);
    }
    T* dst = static_cast<T*>(side ? p.v : p.k) + (n * s.kv_heads + kh) * D + e * 8;
    *reinterpret_cast<uint4*>(dst) = pack8<T>(f);
  }
}

// CTAs along y: a call of few tokens spreads the work of each over several CTAs
// (a decode step of one token is one pass deep); from two tokens per SM on, one
// CTA per token keeps its rotary row in registers over its passes.
unsigned split_y(int64_t tokens, int passes, int num_sms) {
  return tokens >= 2ll * num_sms ? 1u : static_cast<unsigned>(passes);
}

template <typename T, int D>
int append_t(const Kv4AppendParams& p, cudaStream_t st, int num_sms) {
  constexpr int kTeams = kAppThreads / (D / 16);
  const int passes = (p.heads + 2 * p.seq.kv_heads + kTeams - 1) / kTeams;
  const dim3 grid(static_cast<unsigned>(p.seq.tokens), split_y(p.seq.tokens, passes, num_sms));
  const cudaError_t e = launch_pdl(kv4_append_kernel<T, D>, grid, dim3(kAppThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T, int D>
int gather_t(const Kv4GatherParams& p, cudaStream_t st, int num_sms) {
  const int passes = (p.seq.kv_heads * 2 * (D / 8) + kAppThreads - 1) / kAppThreads;
  const dim3 grid(static_cast<unsigned>(p.seq.tokens), split_y(p.seq.tokens, passes, num_sms));
  const cudaError_t e = launch_pdl(kv4_gather_kernel<T, D>, grid, dim3(kAppThreads), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace

int launch_kv4_append(const Kv4Seq& seq, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                      const void* v, int64_t v_stride, void* q_out, void* pool, const float* cs,
                      const float* sn, int rope_len, int heads, int dim, int dtype, int* status,
                      cudaStream_t st, int num_sms) {
  const Kv4AppendParams p{q, k, v, q_stride, k_stride, v_stride, q_out, static_cast<uint8_t*>(pool), cs, sn,
                          rope_len, heads, status, seq};
  if (dtype == FITQ_DTYPE_BF16)
    return dim == 128 ? append_t<__nv_bfloat16, 128>(p, st, num_sms) : append_t<__nv_bfloat16, 64>(p, st, num_sms);
  return dim == 128 ? append_t<__half, 128>(p, st, num_sms) : append_t<__half, 64>(p, st, num_sms);
}

int launch_kv4_gather(const Kv4Seq& seq, const void* pool, void* k, void* v, int dim, int dtype, int* status,
                      cudaStream_t st, int num_sms) {
  const Kv4GatherParams p{static_cast<const uint8_t*>(pool), k, v, status, seq};
  if (dtype == FITQ_DTYPE_BF16)
    return dim == 128 ? gather_t<__nv_bfloat16, 128>(p, st, num_sms) : gather_t<__nv_bfloat16, 64>(p, st, num_sms);
  return dim == 128 ? gather_t<__half, 128>(p, st, num_sms) : gather_t<__half, 64>(p, st, num_sms);
}

}  // namespace fitq
