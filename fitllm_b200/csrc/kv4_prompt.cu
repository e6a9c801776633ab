// Attention of many new tokens (prompts) over the 4-bit paged cache, on tcgen05.
//
// The same product as kv4_attn.cu for calls whose rows (tokens x heads of a KV head)
// fill tensor-core tiles: a CTA takes 256 rows of a (sequence, KV head) pair as two
// tiles of 128 and walks the positions they see in tiles of 128.  Per tile and row
// tile r:  S_r = Q_r.K^T (tcgen05, both operands in shared memory), P_r = 2^(S_r c -
// m) on 128 threads that own a row each, O_r += P_r.V with P_r as the tensor-memory
// operand, written over S_r.  While one row tile's exponentials are taken the other's
// products run.
//
// Roles: warps 0-3 and 4-7 the softmax of row tiles 0 and 1, warps 8-11 decode the
// cache, warp 12 issues the MMAs.  The decoders read blocks straight into registers,
// one tile ahead, and write K [position][D] and V^T [D][position] as fp16 in the
// 128-byte-swizzled K-major layout, two buffers each.  A value of the cache is rounded
// once more, to fp16's 2^-12 (bf16 would round to 2^-9); all are halved, so that a
// group that ends at fp16's largest value stays finite, and the factors go back in with
// the scores' scale and the final 1 / l.  Queries are scaled per row by a power of
// two as in kv4_attn.cu.
//
// The reference m of a row moves only when a weight would exceed 2^15 (fp16's range for
// P); the thread that moves it rescales its row of O_r, which no MMA touches then (the
// products of the tile before completed with S_r).  A thread reads its scores twice
// (the maximum, the weights), the next 32 on their way while it works on 32.
//
// A group of V whose scale or low is not finite must only reach the rows that see it,
// and 0 x NaN would reach all: it enters as zeros, its first position is noted per
// tile, and rows that see the position answer NaN for the group.
//
// Bound: the exponentials (16 per cycle and SM: 2,048 cycles per 256 x 128 tile) and
// the MMAs (4 x 128^3: 2,048 cycles) alike.
#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kPRows = 128;       // rows of a row tile (TMEM lanes)
constexpr int kPTile = 128;       // positions of a tile
constexpr int kPThreads = 416;
constexpr int kPDecoders = 128;
constexpr float kPFloor = -3.0e38f;
constexpr float kPRoom = 15.f;    // weights stay below 2^15

template <int D>
struct PromptSmem {
  static constexpr int kQ = kPRows * D * 2;    // one row tile's queries
  static constexpr int kK = kPTile * D * 2;
  static constexpr int kV = kPTile * D * 2;
  static constexpr int kOffK = 2 * kQ;
  static constexpr int kOffV = kOffK + 2 * kK;
  static constexpr int kBytes = kOffV + 2 * kV + 1024;  // the tiles start on a 1,024-byte boundary
};

struct Kv4PromptParams {
  const void* q;
  int64_t q_stride;
  void* out;
  const uint8_t* pool;
  int heads, group, row_pairs;
  float scale_log2;
  int* status;
  Kv4Seq seq;
};

// Instruction descriptor for kind::f16 with fp16 A/B, fp32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  umma_bf16_ss(tmem_d, adesc, bdesc, idesc, accumulate);  // the type is the descriptor's
}
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t hfma2_u(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_of(uint32_t a) {  // both halves times 1/2
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), __floats2half2_rn(0.5f, 0.5f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Codes 0..15 as half2 from the low / second nibble of each half.
__device__ __forceinline__ uint32_t plain_even(uint32_t x) {
  const uint32_t u = codes_even(x);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(1024.f, 1024.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t plain_odd(uint32_t x) {
  const uint32_t u = codes_odd(x);
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(0.0625f, 0.0625f),
                            __floats2half2_rn(-64.f, -64.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Two fp32 operations in one instruction.
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

extern __shared__ uint8_t g_prompt_smem[];

template <typename T, int D>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prompt_kernel(const Kv4PromptParams p) {
  using L = PromptSmem<D>;
  constexpr int G = D / 64;
  __shared__ uint64_t b_qready, b_kfull[2], b_kfree[2], b_vfull[2], b_vfree[2], b_sfull[2], b_pready[2], b_ofull, b_done;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort;
  __shared__ int sh_bad[2][2];         // per buffer and group: first position that is not finite
  __shared__ uint32_t sh_pages[2];     // per buffer: which of the tile's blocks have a page
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(g_prompt_smem) + 1023u) & ~1023u;

  pdl_launch_dependents();
  pdl_wait();  // q and the cache append come from the previous kernels
  const Kv4Seq& s = p.seq;
  // the row pairs with the most positions come first
  const int per_pair = s.batch * s.kv_heads;
  const int rp = p.row_pairs - 1 - static_cast<int>(blockIdx.x) / per_pair;
  const int pair = static_cast<int>(blockIdx.x) % per_pair;
  const int b = pair / s.kv_heads, kvh = pair % s.kv_heads;
  int64_t first;
  int count;
  kv4_tokens(s, b, first, count);
  const int pre = s.prefix[b];
  const int64_t room = static_cast<int64_t>(s.max_pages) << s.page_shift;
  const int64_t rows_all = static_cast<int64_t>(count) * p.group;
  if (rp == 0 && kvh == 0 && tid == 0 && count > 0 &&
      (pre < 0 || static_cast<int64_t>(pre) + count > room ||
       rows_all > static_cast<int64_t>(p.row_pairs) * 2 * kPRows))
    report_device_error(p.status, FITQ_ERR_ARG);
  const int64_t row0 = static_cast<int64_t>(rp) * 2 * kPRows;
  if (row0 >= rows_all) return;
  const int rows = static_cast<int>(rows_all - row0 < 2 * kPRows ? rows_all - row0 : 2 * kPRows);
  const bool two = rows > kPRows;
  int64_t len64 = pre < 0 ? 0 : static_cast<int64_t>(pre) + (row0 + rows - 1) / p.group + 1;
  if (len64 > room) len64 = room;
  const int len = static_cast<int>(len64);
  const int tiles = (len + kPTile - 1) / kPTile;

  if (tid == 0) {
    sh_abort = 0;
    mbar_init(&b_qready, 2 * kPRows);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b_kfull[i], kPDecoders);
      mbar_init(&b_vfull[i], kPDecoders);
      mbar_init(&b_kfree[i], 1);
      mbar_init(&b_vfree[i], 1);
      mbar_init(&b_sfull[i], 1);
      mbar_init(&b_pready[i], kPRows);
    }
    mbar_init(&b_ofull, 1);
    mbar_init(&b_done, 1);
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sh_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh_tmem;  // S_0, S_1 (128 columns each), O_0, O_1 (D each, 128 apart)
  const uint32_t s_q = base, s_k = base + L::kOffK, s_v = base + L::kOffV;

  // a warp's wait: all of its lanes go on, or none (a wait ran out)
  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, &sh_abort, p.status));
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax: a row per thread
    const int r = warp >> 2;
    const int lr = tid & 127;
    const bool active = r == 0 || two;
    const int64_t row = row0 + r * kPRows + lr;
    const bool has = r * kPRows + lr < rows;
    const int tok = has ? static_cast<int>(row / p.group) : 0;
    const int hd = kvh * p.group + (has ? static_cast<int>(row % p.group) : 0);
    // ---- the row's queries: scaled, fp16, swizzled
    float cn;
    {
      const T* src = static_cast<const T*>(p.q) + (first + tok) * p.q_stride + static_cast<int64_t>(hd) * D;
      uint4 u[D / 8];
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        u[i] = make_uint4(0, 0, 0, 0);
        if (has) u[i] = reinterpret_cast<const uint4*>(src)[i];
        float f[8];
        unpack8<T>(u[i], f);
#pragma unroll
        for (int x = 0; x < 8; ++x) mx = fmaxf(mx, fabsf(f[x]));
      }
      int e = (__float_as_int(mx) >> 23) - 127;
      e = (mx == 0.f || e > 127) ? 12 : (e < -100 ? -100 : e);
      const float up = pow2(12 - e);
      cn = p.scale_log2 * pow2(e - 11);  // keys enter halved
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float f[8];
        unpack8<T>(u[i], f);
        sts128(s_q + r * L::kQ + (i >> 3) * (kPRows * 128) + lr * 128 + (((i & 7) ^ (lr & 7)) << 4),
               pack_half2(f[0] * up, f[1] * up), pack_half2(f[2] * up, f[3] * up), pack_half2(f[4] * up, f[5] * up),
               pack_half2(f[6] * up, f[7] * up));
      }
    }
    fence_async_proxy();
    mbar_arrive(&b_qready);
    const uint32_t t_lane = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t t_s = tmem + t_lane + r * 128, t_o = tmem + t_lane + 256 + r * 128;
    int lim = pre + tok;  // last visible position
    if (lim >= len) lim = len - 1;
    // every row of the CTA sees the positions before this one
    const int64_t sure64 = static_cast<int64_t>(pre) + row0 / p.group + 1;
    const int sure = sure64 < len ? static_cast<int>(sure64) : len;
    float m = kPFloor, l = 0.f;
    uint32_t nan_groups = 0;
    bool ok = active && tiles > 0;
    const uint64_t cn2 = pack2(cn, cn);
    for (int j = 0; ok && j < tiles; ++j) {
      const int buf = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      // the tile's notes are there once V is decoded
      ok = wait_all(&b_vfull[buf], ph) && wait_all(&b_sfull[r], j & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t pages = sh_pages[buf];
      const int pos0 = j * kPTile;
      const bool masked = pos0 + kPTile > sure || pages != 0xffu;
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        if (sh_bad[buf][gr] <= lim) nan_groups |= 1u << gr;
      // ---- the largest score; hidden ones become -inf in tensor memory too
      float raw = -INFINITY;
      {
        uint32_t v[2][32];
        tmem_ld_32x32b_x32(t_s, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t(&x)[32] = v[c & 1];
          tmem_ld_wait();
          if (c < 3) tmem_ld_32x32b_x32(t_s + 32 * (c + 1), v[(c + 1) & 1]);
          if (masked) {
            const uint32_t pg = pages >> (2 * c);
            const int left = lim - pos0 - 32 * c;  // elements 0 .. left are visible
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i > left || !(pg & (i < 16 ? 1u : 2u))) x[i] = 0xff800000u;
            tmem_st_x32(t_s + 32 * c, x);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            raw = fmaxf(raw, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
        }
        if (masked) tmem_st_done();
      }
      raw *= cn;
      if (__any_sync(0xffffffffu, raw > m + kPRoom)) {
        const float m_new = fmaxf(m, raw);
        const float al = exp2_approx(m - m_new);
        m = m_new;
        l *= al;
        if (j > 0) {
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(t_o + 32 * c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * al);
            tmem_st_x32(t_o + 32 * c, v);
          }
        }
      }
      // ---- weights, written over the scores (chunk c's lie where chunk c / 2's were)
      {
        const uint64_t m2 = pack2(-m, -m);
        uint64_t s2 = 0;
        uint32_t v[2][32];
        tmem_ld_32x32b_x32(t_s, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t(&x)[32] = v[c & 1];
          tmem_ld_wait();
          if (c < 3) tmem_ld_32x32b_x32(t_s + 32 * (c + 1), v[(c + 1) & 1]);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), cn2, m2), x0, x1);
            const float w0 = exp2_approx(x0), w1 = exp2_approx(x1);
            s2 = add2(s2, pack2(w0, w1));
            pk[i / 2] = pack_half2(w0, w1);
          }
          tmem_st_x16(t_s + 16 * c, pk);
        }
        float a, c;
        unpack2(s2, a, c);
        l += a + c;
      }
      tmem_st_done();
      tc_fence_before();
      mbar_arrive(&b_pready[r]);
    }
    if (ok) ok = wait_all(&b_ofull, 0);
    if (active && (ok || tiles == 0)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 2.f / l;  // values entered halved
      T* dst = static_cast<T*>(p.out) + ((first + tok) * p.heads + hd) * D;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (tiles > 0) {
          tmem_ld_32x32b_x32(t_o + 32 * c, v);
          tmem_ld_wait();
        }
        const bool bad = (nan_groups >> (c / 2)) & 1u;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) f[x] = bad ? NAN : (l == 0.f ? 0.f : __uint_as_float(v[i + x]) * inv);
          if (has) *reinterpret_cast<uint4*>(dst + 32 * c + i) = pack8<T>(f);
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------ decoders
    const int dt = tid - 256;
    // keys: positions 32 i + dt / 4, sixteen-byte unit c = dt % 4 of each group; values:
    // eight positions of half block h16, elements 8 e .. 8 e + 7 of each group
    const int kc = dt & 3, kp = dt >> 2;
    const int h16 = dt & 15, ve = dt >> 4;
    uint32_t kw[4][2 * G], kpar[4][G], vw[8 * G], vpar[8][G];
    auto look_up = [&](int j) -> int64_t {  // lane i (mod 8): block i of tile j
      int64_t off = -1;
      const int64_t pos = static_cast<int64_t>(j) * kPTile + (lane & 7) * kKv4Block;
      if (j < tiles && pos < len) {
        const int pg = kv4_page(s, b, pos);
        if (pg >= 0)
          off = kv4_block_offset(s, pg, kvh, pos, D);
        else if (dt < 8)
          report_device_error(p.status, FITQ_ERR_ARG);
      }
      return off;
    };
    auto load_k = [&](int64_t off) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = 32 * i + kp;
        const int64_t o = __shfl_sync(0xffffffffu, off, pos >> 4);
#pragma unroll
        for (int w = 0; w < 2 * G; ++w) kw[i][w] = 0;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) kpar[i][gr] = 0;
        if (o >= 0) {
          const uint8_t* blk = p.pool + o;
          const int bp = pos & 15;
          if (G == 2) {
            *reinterpret_cast<uint4*>(kw[i]) = *reinterpret_cast<const uint4*>(blk + (bp * 4 + kc) * 16);
            *reinterpret_cast<uint2*>(kpar[i]) = *reinterpret_cast<const uint2*>(blk + 16 * D + bp * 16);
          } else {
            *reinterpret_cast<uint2*>(kw[i]) = *reinterpret_cast<const uint2*>(blk + (bp * 4 + kc) * 8);
            kpar[i][0] = *reinterpret_cast<const uint32_t*>(blk + 16 * D + bp * 8);
          }
        }
      }
    };
    auto load_v = [&](int64_t off) {
      const int64_t o = __shfl_sync(0xffffffffu, off, h16 >> 1);
      const int h = h16 & 1;
#pragma unroll
      for (int i = 0; i < 8 * G; ++i) vw[i] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) vpar[i][gr] = 0;
      if (o >= 0) {
        const uint8_t* blk = p.pool + o;
        const uint4* src = reinterpret_cast<const uint4*>(blk + 8 * D + (h * 8 + ve) * 32 * G);
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) *reinterpret_cast<uint4*>(vw + 4 * i) = src[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint8_t* ps = blk + 16 * D + (8 * h + i) * 8 * G + 4 * G;
          if (G == 2)
            *reinterpret_cast<uint2*>(vpar[i]) = *reinterpret_cast<const uint2*>(ps);
          else
            vpar[i][0] = *reinterpret_cast<const uint32_t*>(ps);
        }
      }
    };
    bool ok = tiles > 0;
    int64_t off_now = look_up(0), off_next = look_up(1);
    if (ok) {
      load_k(off_now);
      load_v(off_now);
    }
    for (int j = 0; ok && j < tiles; ++j) {
      const int buf = j & 1;
      const uint32_t ph = (j >> 1) & 1;
      const uint32_t pages = __ballot_sync(0xffffffffu, off_now >= 0) & 0xffu;
      off_now = off_next;
      off_next = look_up(j + 2);
      // ---- keys
      if (j >= 2) ok = wait_all(&b_kfree[buf], ph ^ 1u);
      if (!ok) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pos = 32 * i + kp;
        const uint32_t dst = s_k + buf * L::kK + pos * 128;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          const uint32_t par = half_of(kpar[i][gr]);
          const uint32_t sc = __byte_perm(par, par, 0x1010), lo = __byte_perm(par, par, 0x3232);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = kw[i][2 * gr + w], y = x >> 8;
            // pairs (e, e + 4): put in order by halves
            const uint32_t a = hfma2_u(plain_even(x), sc, lo), c = hfma2_u(plain_odd(x), sc, lo);
            const uint32_t d = hfma2_u(plain_even(y), sc, lo), f = hfma2_u(plain_odd(y), sc, lo);
            sts128(dst + gr * (kPTile * 128) + (((2 * kc + w) ^ (pos & 7)) << 4), __byte_perm(a, c, 0x5410),
                   __byte_perm(d, f, 0x5410), __byte_perm(a, c, 0x7632), __byte_perm(d, f, 0x7632));
          }
        }
      }
      fence_async_proxy();
      mbar_arrive(&b_kfull[buf]);
      if (j + 1 < tiles) load_k(off_now);
      // ---- values
      if (j >= 2) ok = wait_all(&b_vfree[buf], ph ^ 1u);
      if (!ok) break;
      int bad[G];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) bad[gr] = 0x7fffffff;
      const int vpos = j * kPTile + 8 * h16;
      uint32_t sc[4][G], lo[4][G];  // of position pairs
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          // an exponent of all ones in either half: not finite
          const uint32_t e = vpar[i][gr] & 0x7c007c00u;
          if (vpos + i >= len) {
            vpar[i][gr] = 0;
          } else if ((e & 0xffffu) == 0x7c00u || (e >> 16) == 0x7c00u) {
            vpar[i][gr] = 0;
            bad[gr] = min(bad[gr], vpos + i);
          }
        }
      if (warp == 8) {  // its lanes 0-15 hold every position of the tile
#pragma unroll
        for (int gr = 0; gr < G; ++gr) bad[gr] = __reduce_min_sync(0xffffffffu, bad[gr]);
        if (lane == 0) {
          sh_pages[buf] = pages;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) sh_bad[buf][gr] = bad[gr];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          sc[i][gr] = half_of(__byte_perm(vpar[2 * i][gr], vpar[2 * i + 1][gr], 0x5410));
          lo[i][gr] = half_of(__byte_perm(vpar[2 * i][gr], vpar[2 * i + 1][gr], 0x7632));
        }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        const uint32_t dst = s_v + buf * L::kV + (h16 >> 3) * (D * 128) + (64 * gr + 8 * ve) * 128;
#pragma unroll
        for (int z = 0; z < 2; ++z) {  // elements 4 z .. 4 z + 3
          uint32_t o[4][4];            // element, position pair
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = __byte_perm(vw[(2 * i) * G + gr], vw[(2 * i + 1) * G + gr], z ? 0x7632 : 0x5410);
            const uint32_t y = x >> 8;
            o[0][i] = hfma2_u(plain_even(x), sc[i][gr], lo[i][gr]);
            o[1][i] = hfma2_u(plain_odd(x), sc[i][gr], lo[i][gr]);
            o[2][i] = hfma2_u(plain_even(y), sc[i][gr], lo[i][gr]);
            o[3][i] = hfma2_u(plain_odd(y), sc[i][gr], lo[i][gr]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int d = 4 * z + x;  // row 64 gr + 8 ve + d: its swizzle is d
            sts128(dst + d * 128 + (((h16 & 7) ^ d) << 4), o[x][0], o[x][1], o[x][2], o[x][3]);
          }
        }
      }
      fence_async_proxy();
      mbar_arrive(&b_vfull[buf]);
      if (j + 1 < tiles) load_v(off_now);
    }
  } else {
    if (lane == 0 && tiles > 0) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc_s = idesc_f16_f32(kPRows, kPTile), idesc_o = idesc_f16_f32(kPRows, D);
    const uint64_t dq = umma_smem_desc_sw128(s_q), dk = umma_smem_desc_sw128(s_k), dv = umma_smem_desc_sw128(s_v);
    auto issue_s = [&](int r, int buf) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t qa = dq + ((r * L::kQ + (kk >> 2) * (kPRows * 128) + (kk & 3) * 32) >> 4);
        const uint64_t kb = dk + ((buf * L::kK + (kk >> 2) * (kPTile * 128) + (kk & 3) * 32) >> 4);
        umma_f16_ss(tmem + r * 128, qa, kb, idesc_s, kk > 0 ? 1u : 0u);
      }
    };
    auto issue_o = [&](int r, int buf, bool add) {
#pragma unroll
      for (int kk = 0; kk < kPTile / 16; ++kk) {
        const uint64_t vb = dv + ((buf * L::kV + (kk >> 2) * (D * 128) + (kk & 3) * 32) >> 4);
        umma_f16_ts(tmem + 256 + r * 128, tmem + r * 128 + kk * 8, vb, idesc_o, add || kk > 0 ? 1u : 0u);
      }
    };
    bool ok = mbar_wait(&b_qready, 0, &sh_abort, p.status) && mbar_wait(&b_kfull[0], 0, &sh_abort, p.status);
    if (ok) {
      tc_fence_after();
      issue_s(0, 0);
      umma_commit(&b_sfull[0]);
      if (two) {
        issue_s(1, 0);
        umma_commit(&b_sfull[1]);
      }
      umma_commit(&b_kfree[0]);
    }
    for (int j = 0; ok && j < tiles; ++j) {
      const int buf = j & 1, nbuf = buf ^ 1;
      const bool more = j + 1 < tiles;
      if (!mbar_wait(&b_vfull[buf], (j >> 1) & 1, &sh_abort, p.status)) break;
      for (int r = 0; ok && r < (two ? 2 : 1); ++r) {
        if (!mbar_wait(&b_pready[r], j & 1, &sh_abort, p.status) ||
            (more && r == 0 && !mbar_wait(&b_kfull[nbuf], ((j + 1) >> 1) & 1, &sh_abort, p.status))) {
          ok = false;
          break;
        }
        tc_fence_after();
        issue_o(r, buf, j > 0);
        if (r == (two ? 1 : 0)) umma_commit(&b_vfree[buf]);
        if (more) {
          issue_s(r, nbuf);
          umma_commit(&b_sfull[r]);
          if (r == (two ? 1 : 0)) umma_commit(&b_kfree[nbuf]);
        }
      }
    }
    if (ok) umma_commit(&b_ofull);
    // every MMA has retired before tensor memory is given back
    umma_commit(&b_done);
    int never = 0;
    mbar_wait(&b_done, 0, &never, p.status);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D>
int prompt_t(const Kv4PromptParams& p, cudaStream_t st) {
  constexpr int smem = PromptSmem<D>::kBytes;
  if (!set_smem_limit(kv4_prompt_kernel<T, D>, smem)) return FITQ_ERR_CUDA;
  const int64_t ctas = static_cast<int64_t>(p.row_pairs) * p.seq.batch * p.seq.kv_heads;
  const cudaError_t e =
      launch_pdl(kv4_prompt_kernel<T, D>, dim3(static_cast<unsigned>(ctas)), dim3(kPThreads), smem, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

}  // namespace

int launch_kv4_prompt(const Kv4Seq& seq, const void* q, int64_t q_stride, const void* pool, void* out, int heads,
                      int dim, int dtype, int64_t max_new, int* status, cudaStream_t st) {
  const int group = heads / seq.kv_heads;
  const int row_pairs = static_cast<int>((group * max_new + 2 * kPRows - 1) / (2 * kPRows));
  const Kv4PromptParams p{q, q_stride, out, static_cast<const uint8_t*>(pool), heads, group, row_pairs,
                          1.4426950408889634f / sqrtf(static_cast<float>(dim)), status, seq};
  if (dtype == FITQ_DTYPE_BF16) return dim == 128 ? prompt_t<__nv_bfloat16, 128>(p, st) : prompt_t<__nv_bfloat16, 64>(p, st);
  return dim == 128 ? prompt_t<__half, 128>(p, st) : prompt_t<__half, 64>(p, st);
}

}  // namespace fitq
