// Append to and read from the 4-bit paged key/value cache (layout: kv4.cuh).
//
// kv4_append_kernel: for every new token the queries and keys are rotated
// (rotate-half, fp32 tables indexed by the token's absolute position), the
// queries are written out in their own type, and the rotated keys (in fp32, not
// rounded first) and the values are coded in groups of 64:
//   low = fp16(min), scale = fp16((max - low) * (1 / 15)),
//   code = round((x - low) * (1 / scale)) in 0..15, 0 where scale is 0,
// every difference, product and reciprocal rounded to fp32 on its own (no fused
// multiply-add: a code next to a border is then the same wherever it is
// computed).  A group that holds a NaN, an infinity or a value fp16 cannot
// reach gets a non-finite scale and reads back as NaN.
//
// Bound: HBM (q, k, v in, q and the blocks out) for prompts (three of up to 4,001
// tokens, 40 heads on 8, with a read back of what was written: 58 us, 4.8 TB/s), the
// launch for a decode step (64 tokens with the read back: 4.8 us).  A CTA takes up to four tokens: their places (sequence, position,
// page: a chain of dependent loads) are found once, by one thread each, while the
// first heads are already on their way, and each team of lanes loads its next head
// before it works on the current one.
#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kAppThreads = 256;
constexpr float kFifteenth = 1.f / 15.f;

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

// Eight codes of x under (low, inv), packed low nibble first.  A sum with 1.5 * 2^23
// rounds to the nearest whole number, ties to even, and leaves it in the low bits;
// the eight words add up to the codes plus a constant.
__device__ __forceinline__ uint32_t code8(const float (&x)[8], float low, float inv) {
  constexpr uint32_t kBias = 0x4B400000u;  // the bits of 1.5 * 2^23
  uint32_t w = 0, shifted = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], low), inv), 0.f), 15.f);
    w += __float_as_uint(__fadd_rn(c, 12582912.f)) << (4 * i);
    shifted += kBias << (4 * i);
  }
  return w - shifted;
}

constexpr int kAppTokens = 4;  // tokens of a CTA, at most

// Where a new token goes: its sequence's page and position; page < -1: no sequence,
// -1: refused.
struct TokenPlace {
  int page, pos;
};
__device__ __forceinline__ TokenPlace token_place(const Kv4Seq& s, int64_t n, int limit, int* status) {
  TokenPlace r{-2, 0};
  if (n >= s.tokens) return r;
  const int b = kv4_sequence(s, n);
  if (b < 0) return r;  // a token of no sequence: left as it is
  const int64_t first = s.q_start ? s.q_start[b] : static_cast<int64_t>(b) * s.t_new;
  const int pre = s.prefix[b];
  const int64_t pos = pre + (n - first);
  r.page = (pre < 0 || pos >= limit) ? -1 : kv4_page(s, b, pos);
  r.pos = r.page < 0 ? 0 : static_cast<int>(pos);
  if (r.page < 0) report_device_error(status, FITQ_ERR_ARG);
  return r;
}

// A CTA's heads (q, then k, then v slots of each of its tokens) go round its teams
// of D / 16 lanes (blockIdx.y: one of several CTAs of the same tokens).  Lane i of a
// team holds elements 8 i .. 8 i + 7 of each half of the head, so the rotation pairs
// meet in one lane and the group extrema take log2(team) shuffles.
template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads, 4) kv4_append_kernel(const Kv4AppendParams p, int per_cta) {
  constexpr int kTeam = D / 16;
  constexpr int kTeams = kAppThreads / kTeam;
  constexpr int kHalf = D / 2;
  __shared__ TokenPlace sh_place[kAppTokens];
  const int lane = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
  pdl_launch_dependents();
  pdl_wait();  // q, k, v come from the previous kernel
  const Kv4Seq& s = p.seq;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * per_cta;
  const int slots = p.heads + 2 * s.kv_heads;
  const int count = static_cast<int>(n0 + per_cta <= s.tokens ? per_cta : s.tokens - n0);
  const int step = kTeams * gridDim.y;

  uint4 ra = make_uint4(0, 0, 0, 0), rb = ra;  // this lane's elements of the next head
  auto fetch = [&](int tok, int slot) {
    if (tok >= count) return;
    const int64_t n = n0 + tok;
    const T* src = slot < p.heads ? static_cast<const T*>(p.q) + n * p.q_stride + slot * D
                   : slot < p.heads + s.kv_heads
                       ? static_cast<const T*>(p.k) + n * p.k_stride + (slot - p.heads) * D
                       : static_cast<const T*>(p.v) + n * p.v_stride + (slot - p.heads - s.kv_heads) * D;
    ra = *reinterpret_cast<const uint4*>(src + lane * 8);
    rb = *reinterpret_cast<const uint4*>(src + kHalf + lane * 8);
  };
  // (token, slot) of the team's current and next head, stepped without a division
  int tok_next = 0, slot_next = blockIdx.y * kTeams + team;
  auto wrap = [&]() {
    while (slot_next >= slots) {
      slot_next -= slots;
      ++tok_next;
    }
  };
  wrap();
  fetch(tok_next, slot_next);
  if (threadIdx.x < per_cta) sh_place[threadIdx.x] = token_place(s, n0 + threadIdx.x, p.rope_len, p.status);
  __syncthreads();

  while (__any_sync(0xffffffffu, tok_next < count)) {
    const bool have = tok_next < count;
    const int tok = have ? tok_next : 0, slot = slot_next;
    const TokenPlace at = sh_place[tok];
    const bool ok = have && at.page >= 0;
    const bool is_q = have && slot < p.heads;
    const bool is_kv = have && !is_q;
    const bool is_k = is_kv && slot < p.heads + s.kv_heads;
    float a[8], bb[8];
    unpack8<T>(ra, a);
    unpack8<T>(rb, bb);
    slot_next += step;
    wrap();
    fetch(tok_next, slot_next);
    if (is_q || is_k) {
      const float4* cp = reinterpret_cast<const float4*>(p.cs + static_cast<int64_t>(at.pos) * kHalf + lane * 8);
      const float4* sp = reinterpret_cast<const float4*>(p.sn + static_cast<int64_t>(at.pos) * kHalf + lane * 8);
      const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
      const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
      const float sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = bb[i];
        a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, sv[i]));
        bb[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, sv[i]));
      }
    }
    if (is_q && at.page >= -1) {  // a refused token's query reads as zeros
      T* dst = static_cast<T*>(p.q_out) + ((n0 + tok) * p.heads + slot) * D;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(dst + lane * 8) = ok ? pack8<T>(a) : zero;
      *reinterpret_cast<uint4*>(dst + kHalf + lane * 8) = ok ? pack8<T>(bb) : zero;
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
        const __half c0 = __float2half_rn(__fmul_rn(__fsub_rn(hi0, f0), kFifteenth));
        const __half c1 = __float2half_rn(__fmul_rn(__fsub_rn(hi1, f1), kFifteenth));
        const float g0 = __half2float(c0), g1 = __half2float(c1);
        const uint32_t w0 = code8(a, f0, g0 > 0.f ? __frcp_rn(g0) : 0.f);
        const uint32_t w1 = code8(bb, f1, g1 > 0.f ? __frcp_rn(g1) : 0.f);
        const int kh = is_k ? slot - p.heads : slot - p.heads - s.kv_heads;
        const int bp = at.pos & 15;
        uint32_t* blk = reinterpret_cast<uint32_t*>(p.pool + kv4_block_offset(s, at.page, kh, at.pos, D));
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
// in fp32, rounded once.  A thread's words of the CTA's tokens are all on their way
// before the first is used.
template <typename T, int D>
__global__ void __launch_bounds__(kAppThreads) kv4_gather_kernel(const Kv4GatherParams p, int per_cta) {
  __shared__ TokenPlace sh_place[kAppTokens];
  pdl_launch_dependents();
  pdl_wait();  // the pool is written by the previous kernel
  const Kv4Seq& s = p.seq;
  constexpr int kWords = D / 8;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * per_cta;
  if (threadIdx.x < kAppTokens)
    sh_place[threadIdx.x] = static_cast<int>(threadIdx.x) < per_cta
                                ? token_place(s, n0 + threadIdx.x, 0x7fffffff, p.status)
                                : TokenPlace{-2, 0};
  __syncthreads();
  const int items = s.kv_heads * 2 * kWords;
  for (int i = blockIdx.y * kAppThreads + threadIdx.x; i < items; i += gridDim.y * kAppThreads) {
    const int e = i % kWords, side = (i / kWords) & 1, kh = i / (2 * kWords);
    const int g = e / 8, e8 = e % 8;
    uint32_t w[kAppTokens], pr[kAppTokens];
#pragma unroll
    for (int t = 0; t < kAppTokens; ++t) {
      const TokenPlace at = sh_place[t];
      w[t] = pr[t] = 0;
      if (at.page >= 0) {
        const uint32_t* blk = reinterpret_cast<const uint32_t*>(p.pool + kv4_block_offset(s, at.page, kh, at.pos, D));
        const int bp = at.pos & 15;
        w[t] = blk[side ? kv4_value_word<D>(bp, g, e8) : kv4_key_word<D>(bp, g, e8)];
        pr[t] = blk[kv4_param_word<D>(bp, side, g)];
      }
    }
#pragma unroll
    for (int t = 0; t < kAppTokens; ++t) {
      if (sh_place[t].page < -1) continue;
      const float2 sl = Half16<__half>::unpack(pr[t]);
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = __fadd_rn(__fmul_rn(sl.x, static_cast<float>((w[t] >> (4 * j)) & 15u)), sl.y);
      T* dst = static_cast<T*>(side ? p.v : p.k) + ((n0 + t) * s.kv_heads + kh) * D + e * 8;
      *reinterpret_cast<uint4*>(dst) = pack8<T>(f);
    }
  }
}

// Tokens per CTA and CTAs along y: few tokens spread each over several CTAs (a decode
// step is one pass deep); from eight per SM on a CTA takes four.
struct TokenGrid {
  int per_cta;
  dim3 grid;
};
TokenGrid token_grid(int64_t tokens, int passes, int num_sms) {
  TokenGrid g;
  g.per_cta = tokens >= 8ll * num_sms ? kAppTokens : 1;
  g.grid = dim3(static_cast<unsigned>((tokens + g.per_cta - 1) / g.per_cta),
                tokens >= 2ll * num_sms ? 1u : static_cast<unsigned>(passes));
  return g;
}

template <typename T, int D>
int append_t(const Kv4AppendParams& p, cudaStream_t st, int num_sms) {
  constexpr int kTeams = kAppThreads / (D / 16);
  const TokenGrid g = token_grid(p.seq.tokens, (p.heads + 2 * p.seq.kv_heads + kTeams - 1) / kTeams, num_sms);
  const cudaError_t e = launch_pdl(kv4_append_kernel<T, D>, g.grid, dim3(kAppThreads), 0, st, p, g.per_cta);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T, int D>
int gather_t(const Kv4GatherParams& p, cudaStream_t st, int num_sms) {
  const TokenGrid g = token_grid(p.seq.tokens, (p.seq.kv_heads * 2 * (D / 8) + kAppThreads - 1) / kAppThreads, num_sms);
  const cudaError_t e = launch_pdl(kv4_gather_kernel<T, D>, g.grid, dim3(kAppThreads), 0, st, p, g.per_cta);
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
