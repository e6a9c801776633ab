// The 4-bit paged key/value cache: block layout and addressing shared by the
// append, gather and attention kernels (kv4.cu, kv4_attn.cu, kv4_prompt.cu).
//
// A pool holds pages of page_size positions, uint8
// [pages, KVH, page_size / 16, 18 D]: one block per 16 positions of a KV head.
// Each group of 64 elements of a key or value is value = scale * code + low
// (code 0..15, fp16 scale and low): 4.5 bits an element.  Inside a block, with
// G = D / 64 groups and eight elements per 4-byte word (element j in bits 4j):
//   keys    [16 positions][4 c][G g][2 w] words: elements 64 g + 16 c + 8 w + j.
//           Lane (r, c) of a warp reads its A-fragment row r of every k-step of
//           S^T = K.Q^T as one 8 G-byte load; the contraction index is permuted
//           alike in Q's fragments, so no element moves between lanes.
//   values  [2 h][8 e][4 q][2 o][G g] words: elements 64 g + 8 e + j of position
//           8 h + 2 q + o.  Lane (e, q) reads the positions of its A-fragment
//           columns of O^T = V^T.P^T as one 8 G-byte load per half h, at
//           consecutive addresses over the warp (no bank conflicts, whole lines).
//   params  [16 positions][key, value][G][scale, low] fp16.
// A word belongs to one position, so positions are written independently.
#pragma once
#include "common.cuh"

namespace fitq {

constexpr int kKv4Block = 16;  // positions per block

// Addressing of a call's new tokens and of the cache behind the page table.
struct Kv4Seq {
  const int32_t* page_table;  // [batch, max_pages]
  const int32_t* prefix;      // [batch] cached positions before the new tokens
  const int32_t* q_start;     // [batch + 1] or null: tokens / batch tokens each
  int64_t tokens;
  int batch, t_new;           // t_new: tokens of each sequence when q_start is null
  int max_pages, page_shift;  // page_size = 1 << page_shift
  int64_t num_pages;
  int kv_heads;
};

__host__ __device__ constexpr int kv4_block_bytes(int dim) { return 18 * dim; }

// Word index (4 bytes) of eight elements 8 e8 .. 8 e8 + 7 of group g at block position p.
template <int D>
__device__ __forceinline__ int kv4_key_word(int p, int g, int e8) {
  return ((p * 4 + (e8 >> 1)) * (D / 64) + g) * 2 + (e8 & 1);
}
template <int D>
__device__ __forceinline__ int kv4_value_word(int p, int g, int e8) {
  return 2 * D + ((((p >> 3) * 8 + e8) * 4 + ((p & 7) >> 1)) * 2 + (p & 1)) * (D / 64) + g;
}
// Word index of the (scale, low) pair of group g: side 0 keys, 1 values.
template <int D>
__device__ __forceinline__ int kv4_param_word(int p, int side, int g) {
  return 4 * D + (p * 2 + side) * (D / 64) + g;
}

// Tokens of sequence b: [first, first + count), clamped to the packed tokens so
// that a bad q_start never leads out of q.
__device__ __forceinline__ void kv4_tokens(const Kv4Seq& s, int b, int64_t& first, int& count) {
  if (s.q_start == nullptr) {
    first = static_cast<int64_t>(b) * s.t_new;
    count = s.t_new;
    return;
  }
  int64_t a = s.q_start[b], e = s.q_start[b + 1];
  a = a < 0 ? 0 : a;
  e = e > s.tokens ? s.tokens : e;
  first = a;
  count = e > a ? static_cast<int>(e - a) : 0;
}

// Sequence of packed token n under q_start: the last b with q_start[b] <= n, or
// -1 where n lies before the first or behind the last sequence.
__device__ __forceinline__ int kv4_sequence(const Kv4Seq& s, int64_t n) {
  if (s.q_start == nullptr) return static_cast<int>(n / s.t_new);
  int lo = 0, hi = s.batch;  // answer + 1 in [lo, hi]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s.q_start[mid] <= n)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int b = lo - 1;
  return (b >= 0 && n < s.q_start[b + 1]) ? b : -1;
}

// Page of position pos of sequence b, or -1 (position outside the table, or an
// entry that names no page).
__device__ __forceinline__ int kv4_page(const Kv4Seq& s, int b, int64_t pos) {
  if (pos < 0 || (pos >> s.page_shift) >= s.max_pages) return -1;
  const int pg = s.page_table[static_cast<int64_t>(b) * s.max_pages + (pos >> s.page_shift)];
  return (pg >= 0 && pg < s.num_pages) ? pg : -1;
}

// Byte offset of the block of position pos (page pg, KV head kvh) in the pool.
__device__ __forceinline__ int64_t kv4_block_offset(const Kv4Seq& s, int pg, int kvh, int64_t pos, int dim) {
  const int64_t per = 1ll << (s.page_shift - 4);
  const int64_t in_page = (pos & ((1ll << s.page_shift) - 1)) >> 4;
  return ((static_cast<int64_t>(pg) * s.kv_heads + kvh) * per + in_page) * kv4_block_bytes(dim);
}

// A warp's wait: every lane goes on, or none (a wait ran out).  A lane decides by its own
// view of the barrier, the abort flag and the clock; behind the wait stand shuffles, votes
// and MMAs of the whole warp, which lanes that had given up would never reach.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status));
}

// 16-bit activations: bf16 or fp16.
template <typename T>
struct Half16;
template <>
struct Half16<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t u) { return unpack_bf16x2(u); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <>
struct Half16<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Half16<T>::unpack(w[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Half16<T>::pack(f[0], f[1]), Half16<T>::pack(f[2], f[3]), Half16<T>::pack(f[4], f[5]),
                    Half16<T>::pack(f[6], f[7]));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in a register pair, one instruction for both.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// The codes as fp16 subnormals: 2^-24 c of the low nibble of each half, 2^-20 c of the
// second one.
__device__ __forceinline__ uint32_t tiny_even(uint32_t x) { return x & 0x000f000fu; }
__device__ __forceinline__ uint32_t tiny_odd(uint32_t x) { return x & 0x00f000f0u; }
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) { return Half16<__half>::pack(lo, hi); }

// 2^k with k in [-126, 127].
__device__ __forceinline__ float pow2(int k) { return __int_as_float((k + 127) << 23); }

}  // namespace fitq
