// Attention of many new tokens (prompts) over the 4-bit paged cache, on tcgen05.
//
// The same product as kv4_attn.cu for calls whose rows (tokens x heads of a KV head)
// fill tensor-core tiles: a CTA takes 256 rows of a (sequence, KV head) pair as two
// tiles of 128 and walks the positions they see in steps of 64.  Per step and row
// tile r:  S_r = Q_r.K^T (tcgen05, both operands in shared memory), P_r = 2^(S_r c -
// m) on 128 threads that own a row each, O_r += P_r.V with P_r as the tensor-memory
// operand, written over S_r.  Tensor memory holds two steps of S for each row tile:
// while a thread takes the exponentials of one, the MMAs before and behind the other
// run (with one step of 128 positions the two waited for each other, 5,200 cycles
// per 128 positions).
//
// Roles: warps 0-3 and 4-7 the softmax of row tiles 0 and 1, warps 8-15 decode the
// cache (with four of them a tile took 5,400 cycles, their own instructions' latency),
// warp 16 issues the MMAs.  The decoders read blocks straight into registers,
// one tile ahead, and write K [position][D] and V^T [D][position] as fp16 in the
// 128-byte-swizzled K-major layout, two buffers each.  A value of the cache is rounded
// once more, by half a step of fp16, 2^-11 (bf16's is 2^-8); all are halved, so that a
// group that ends at fp16's largest value stays finite, and the factors go back in with
// the scores' scale and the final 1 / l.  It is the codes that are halved, which is
// exact: a halved scale would lose a bit below 2^-13, fifteen times over in a value.  What
// remains there is the rounding of the halved low and of the sum: 2^-23 of a value at most.
// fp16 results would show it, once of the keys and once of the values (relative error
// 4.2e-4 where the result's rounding and the weights' alone give 2.9e-4): there a value is
// the sum of two fp16 numbers, computed in fp32, tiles are 64 positions of two rows (columns
// of V^T) each, half of the decoders decode keys and half values, and both products take twice
// the MMAs: 176 -> 279 us for the two sequences below.  Queries are scaled per row by a power of two as in kv4_attn.cu.
//
// The reference m of a row moves only when a weight would exceed 2^15 (fp16's range for
// P), and then to 2^7 below the row's largest, so that eight more bits of growth move
// nothing; the thread that moves it rescales its row of O_r once the step before has been
// added to it.  Weights keep fp16's 11 bits down to 2^-21 of the largest met and some of
// them down to 2^-32: behind a first position with 99.9% of the mass, 131,000 others
// still count (with the reference at the largest itself all of them rounded to zero).
//
// A group of V whose scale or low is not finite must only reach the rows that see it,
// and 0 x NaN would reach all: it enters as zeros, its first position is noted per
// tile, and rows that see the position answer NaN for the group.
//
// Where the pairs' row tiles are fewer than the SMs, a pair's positions are cut into up
// to kPMaxSplits parts of equal tiles, a CTA each; they leave (O, m, l) per row in the
// workspace and kv4_prompt_combine_kernel joins them in order (deterministic).  After
// window_steps O_r joins the rows' sums in the workspace and begins anew.  Where the parts or
// sums of all rows would take more than kPScratch, the call goes in several launches.
//
// Bound: the exponentials (16 per cycle and SM: 2,048 cycles per 256 x 128 tile) and
// the MMAs (4 x 128^3: 2,048 cycles) alike; measured, the chain of a step (wait, read S,
// maximum, exponentials, write P) and its hand-overs, some 2,000 cycles of 64 positions
// that two row tiles per SM cover in part.  Two sequences of up to 2,048 tokens (40 heads
// on 8) behind up to 513: 175.5 us, 0.56 PFLOP/s.  Half the exponentials as a polynomial
// on the FMA pipe made it 183 us, sixteen softmax warps (two threads a row) 200 us.
#include <type_traits>

#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kPRows = 128;       // rows of a row tile (TMEM lanes)
constexpr int kPTile = 128;       // rows of a decoded tile
constexpr int kPStep = 64;        // positions of a step
constexpr int kPThreads = 640;     // five warpgroups
// Registers per thread: 96 at launch (61,440 in all), then softmax 128, decoders 80,
// issuer 64: 2 x 128 + 2 x 80 + 64 = 480 per lane of a warpgroup.
constexpr int kPRegsSoftmax = 128, kPRegsDecode = 80, kPRegsIssue = 64;
static_assert(2 * kPRegsSoftmax + 2 * kPRegsDecode + kPRegsIssue <= 5 * 96, "more registers than the launch has");
constexpr float kPFloor = -3.0e38f;
constexpr float kPRoom = 15.f;    // weights stay below 2^15
constexpr float kPSlack = 8.f;    // a reference that moves leaves this much (log2) to the weights that follow
constexpr int kPMaxSplits = 32;   // a lane of the combining warp each
// Steps after which O_r joins its rows' sums in the workspace.  An accumulation in tensor
// memory rounds towards zero at the accumulator's size, some 2^-24 of it each time, which adds
// up to 5e-4 of the output over 131,072 positions and 5e-3 over a million.
template <typename T>
constexpr int window_steps() { return std::is_same<T, __half>::value ? 1 << 8 : 1 << 10; }
constexpr int64_t kPScratch = 256ll << 20;  // bytes of such sums and of parts that a launch needs, about, at most

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
  float* ml_part;  // [CTAs of the launch without splits][splits][256 rows][2], splits > 1 only
  float* o_part;   // [..][D], splits > 1 or where a call may have more than window_steps
  int heads, group, row_pairs;
  int max_new;  // the most new tokens of a sequence that the launch covers
  int cta0;     // CTA (without splits) that this launch begins with
  float scale_log2;
  int* status;
  Kv4Seq seq;
};

// Instruction descriptor for kind::f16 with fp16 A/B, fp32 D, both K-major.
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// MMAs and commits of a warp that runs as one, issued by its elected lane: with the
// loop around them uniform the operands are computed in uniform registers (from one
// lane's branch every MMA took nine moves there, 90 cycles an MMA).
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void commit_warp(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
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
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
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
// (x & mask) | 512 in both halves, in one instruction (two constants in one
// expression would be split in two).
template <uint32_t kMask>
__device__ __forceinline__ uint32_t nibbles(uint32_t x) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "n"(kMask), "r"(0x60006000u));
  return d;
}
// 512 + c / 2 of the low nibble of each half (fp16's steps are 1/2 there); 512 + 8 c of
// the second one.
__device__ __forceinline__ uint32_t codes_even(uint32_t x) { return nibbles<0x000f000fu>(x); }
__device__ __forceinline__ uint32_t codes_odd(uint32_t x) { return nibbles<0x00f000f0u>(x); }
// Half the codes, 0, 1/2 .. 15/2, as half2 from the low / second nibble of each half.
__device__ __forceinline__ uint32_t halved_even(uint32_t x) {
  const uint32_t u = codes_even(x);
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(512.f, 512.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t halved_odd(uint32_t x) {
  const uint32_t u = codes_odd(x);
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&u), __floats2half2_rn(0.0625f, 0.0625f),
                            __floats2half2_rn(-32.f, -32.f));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t a) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(a) : "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }


// v / 2 = hi + lo, both fp16, of two values: from their codes' halves, scales and halved lows.
struct Pair2 {
  uint32_t hi, lo;
};
__device__ __forceinline__ Pair2 value_pair(uint32_t codes, float s0, float s1, float l0, float l1) {
  const float2 c = Half16<__half>::unpack(codes);
  const float a = fmaf(c.x, s0, l0), b = fmaf(c.y, s1, l1);
  Pair2 r;
  r.hi = pack_half2(a, b);
  const float2 h = Half16<__half>::unpack(r.hi);
  r.lo = pack_half2(a - h.x, b - h.y);
  return r;
}

extern __shared__ uint8_t g_prompt_smem[];

// kLong: a row may see more than window_steps.
template <typename T, int D, bool kLong>
__global__ void __launch_bounds__(kPThreads, 1) kv4_prompt_kernel(const Kv4PromptParams p) {
  using L = PromptSmem<D>;
  constexpr int G = D / 64;
  // two fp16 numbers a value, hi in the tile's first half and lo in its second
  constexpr bool kTwo = std::is_same<T, __half>::value;
  constexpr int kTile = kTwo ? kPTile / 2 : kPTile;  // positions of a decoded tile
  constexpr int kSteps = kTile / kPStep;             // steps of one
  constexpr int kBlocks = kTile / kKv4Block;         // blocks of one, a warp each
  constexpr int kWindow = window_steps<T>();
  __shared__ uint64_t b_qready, b_kfull[2], b_kfree[2], b_vfull[2], b_vfree[2], b_sfull[2][2], b_pready[2][2], b_odone[2][2], b_done;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort;
  // per buffer and block: 1 if it has a page, and from bit 8 and 16 the first position
  // at which a value of group 0 and 1 is not finite (16: none)
  __shared__ __align__(16) uint32_t sh_note[2][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(g_prompt_smem) + 1023u) & ~1023u;

  pdl_launch_dependents();
  pdl_wait();  // q and the cache append come from the previous kernels
  const Kv4Seq& s = p.seq;
  // the row pairs with the most positions come first
  const int per_pair = s.batch * s.kv_heads;
  const int cta = p.cta0 + static_cast<int>(blockIdx.x);
  const int rp = p.row_pairs - 1 - cta / per_pair, pair = cta % per_pair;
  const int b = pair / s.kv_heads, kvh = pair % s.kv_heads;
  int64_t first;
  int count;
  kv4_tokens(s, b, first, count);
  const int pre = s.prefix[b];
  const int64_t room = static_cast<int64_t>(s.max_pages) << s.page_shift;
  const int64_t rows_all = static_cast<int64_t>(min(count, p.max_new)) * p.group;
  if (rp == 0 && kvh == 0 && blockIdx.y == 0 && tid == 0 && count > 0 &&
      (pre < 0 || static_cast<int64_t>(pre) + count > room || count > p.max_new))
    report_device_error(p.status, FITQ_ERR_ARG);
  const int64_t row0 = static_cast<int64_t>(rp) * 2 * kPRows;
  if (row0 >= rows_all) return;
  const int rows = static_cast<int>(rows_all - row0 < 2 * kPRows ? rows_all - row0 : 2 * kPRows);
  const bool two = rows > kPRows;
  int64_t len64 = pre < 0 ? 0 : static_cast<int64_t>(pre) + (row0 + rows - 1) / p.group + 1;
  if (len64 > room) len64 = room;
  // This CTA's part: `tiles` tiles from position at0 on.  Positions below are relative to at0.
  const int len_all = static_cast<int>(len64);
  const int tiles_all = (len_all + kTile - 1) / kTile;
  const int share = (tiles_all + static_cast<int>(gridDim.y) - 1) / static_cast<int>(gridDim.y);
  const int tile0 = min(static_cast<int>(blockIdx.y) * share, tiles_all);
  const int tiles = min(share, tiles_all - tile0);
  const int at0 = tile0 * kTile;
  const int len = min(len_all - at0, tiles * kTile);

  if (tid == 0) {
    sh_abort = 0;
    mbar_init(&b_qready, 8);  // one arrival per warp
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b_kfull[i], kBlocks);
      mbar_init(&b_vfull[i], kBlocks);
      mbar_init(&b_kfree[i], 1);
      mbar_init(&b_vfree[i], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&b_sfull[i][h], 1);
        mbar_init(&b_pready[i][h], kPRows / 32);
        mbar_init(&b_odone[i][h], 1);
      }
    }
    mbar_init(&b_done, 1);
    fence_mbar_init();
  }
  if (warp == 16) {
    tmem_alloc(&sh_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh_tmem;  // S_0, S_1 (128 columns each), O_0, O_1 (D each, 128 apart)
  const uint32_t s_q = base, s_k = base + L::kOffK, s_v = base + L::kOffV;

  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
    return mbar_wait_warp(bar, parity, &sh_abort, p.status);
  };

  auto arrive_warp = [&](uint64_t* bar) {  // behind every lane's stores and fences
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPRegsSoftmax));
    // ------------------------------------------------------------ softmax: a row per thread
    const int r = warp >> 2;
    const int lr = tid & 127;
    const bool active = r == 0 || two;
    const int64_t row = row0 + r * kPRows + lr;
    const bool has = r * kPRows + lr < rows;
    const int tok = has ? static_cast<int>(row / p.group) : 0;
    const int hd = kvh * p.group + (has ? static_cast<int>(row % p.group) : 0);
    // ---- the row's queries: scaled, fp16, swizzled, elements as the keys'
    float cn;
    {
      const T* src = static_cast<const T*>(p.q) + (first + tok) * p.q_stride + static_cast<int64_t>(hd) * D;
      const uint4* qv = reinterpret_cast<const uint4*>(src);
      float mx = 0.f;
      if (has) {
#pragma unroll 4
        for (int i = 0; i < D / 8; ++i) {
          float f[8];
          unpack8<T>(qv[i], f);
#pragma unroll
          for (int x = 0; x < 8; ++x) mx = fmaxf(mx, fabsf(f[x]));
        }
      }
      int e = (__float_as_int(mx) >> 23) - 127;
      e = (mx == 0.f || e > 127) ? 12 : (e < -100 ? -100 : e);
      const float up = pow2(12 - e);
      cn = p.scale_log2 * pow2(e - 11);  // keys enter halved
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (has) u = qv[i];
        float f[8];
        unpack8<T>(u, f);
        sts128(s_q + r * L::kQ + (i >> 3) * (kPRows * 128) + lr * 128 + (((i & 7) ^ (lr & 7)) << 4),
               pack_half2(f[0] * up, f[4] * up), pack_half2(f[1] * up, f[5] * up), pack_half2(f[2] * up, f[6] * up),
               pack_half2(f[3] * up, f[7] * up));
      }
    }
    fence_async_proxy();
    arrive_warp(&b_qready);
    const uint32_t t_lane = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t t_s = tmem + t_lane + r * 128, t_o = tmem + t_lane + 256 + r * 128;
    const int lim = min(pre + tok, len_all - 1) - at0;  // last visible position
    // every row of the CTA sees the positions before this one
    const int64_t sure64 = static_cast<int64_t>(pre) + row0 / p.group + 1;
    const int sure = (sure64 < len_all ? static_cast<int>(sure64) : len_all) - at0;
    float m = kPFloor, l = 0.f, m_kept = kPFloor;
    const int64_t part = (static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y) * (2 * kPRows) + r * kPRows + lr;
    uint32_t nan_groups = 0;
    bool ok = active && tiles > 0;
    const uint64_t cn2 = pack2(cn, cn);
    const int steps = (len + kPStep - 1) / kPStep;
    for (int t0 = 0; ok && t0 < steps;) {
      if (kLong && t0 > 0) {  // O_r joins the row's sums, whose columns are its own, and begins anew
        ok = wait_all(&b_odone[r][(t0 - 1) & 1], ((t0 - 1) >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        const float k = exp2_approx(m_kept - m);
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t x[16];
          tmem_ld_x16(t_o + 16 * c, x);
          tmem_ld_wait();
          if (has) {
            float4* sum = reinterpret_cast<float4*>(p.o_part + part * D + 16 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float4 v = t0 > kWindow ? sum[i] : make_float4(0.f, 0.f, 0.f, 0.f);
              v.x = fmaf(k, v.x, __uint_as_float(x[4 * i]));
              v.y = fmaf(k, v.y, __uint_as_float(x[4 * i + 1]));
              v.z = fmaf(k, v.z, __uint_as_float(x[4 * i + 2]));
              v.w = fmaf(k, v.w, __uint_as_float(x[4 * i + 3]));
              sum[i] = v;
            }
          }
          __syncwarp();
        }
        m_kept = m;
      }
      const int t1 = kLong && steps - t0 > kWindow ? t0 + kWindow : steps;
      for (int t = t0; ok && t < t1; ++t) {
        const int j = t / kSteps, sub = t % kSteps, buf = j & 1, h = t & 1;
        const int pos0 = t * kPStep;
        // the tile's notes are there once V is decoded
        if (sub == 0) {
          ok = wait_all(&b_vfull[buf], (j >> 1) & 1);
          if (!ok) break;
        }
        ok = wait_all(&b_sfull[r][h], (t >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld_32x32b_x32(t_s + h * kPStep, v[0]);
        tmem_ld_32x32b_x32(t_s + h * kPStep + 32, v[1]);
        uint32_t pages = 0xfu;  // which of the step's blocks are there
        const uint4 nt = *reinterpret_cast<const uint4*>(&sh_note[buf][4 * sub]);
        constexpr uint32_t kClean = 1u | (kKv4Block << 8) | (kKv4Block << 16);
        if (((nt.x ^ kClean) | (nt.y ^ kClean) | (nt.z ^ kClean) | (nt.w ^ kClean)) != 0) {
          pages = 0;
          for (int i = 0; i < 4; ++i) {
            const uint32_t note = sh_note[buf][4 * sub + i];
            pages |= (note & 1u) << i;
            for (int gr = 0; gr < G; ++gr) {
              const int at = static_cast<int>((note >> (8 + 8 * gr)) & 0xffu);
              if (at < kKv4Block && pos0 + i * kKv4Block + at <= lim) nan_groups |= 1u << gr;
            }
          }
        }
        tmem_ld_wait();
        if (pos0 + kPStep > sure || pages != 0xfu) {  // hidden positions
          const int left = lim - pos0;                // elements 0 .. left are visible
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (32 * c + i > left || !(pages & (1u << (2 * c + (i >> 4))))) v[c][i] = 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) top[x] = -INFINITY;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 8)
#pragma unroll
            for (int x = 0; x < 4; ++x)
              top[x] = fmaxf(top[x], fmaxf(__uint_as_float(v[c][i + 2 * x]), __uint_as_float(v[c][i + 2 * x + 1])));
        const float raw = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * cn;
        if (__any_sync(0xffffffffu, raw > m + kPRoom)) {
          const float m_new = fmaxf(m, raw - (kPRoom - kPSlack));
          const float al = exp2_approx(m - m_new);
          m = m_new;
          l *= al;
          if (t > t0) {
            ok = wait_all(&b_odone[r][h ^ 1], ((t - 1) >> 1) & 1);  // the step before has been added
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t x[16];
              tmem_ld_x16(t_o + 16 * c, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * al);
              tmem_st_x16(t_o + 16 * c, x);
            }
          }
        }
        // ---- weights, written over the scores
        const uint64_t m2 = pack2(-m, -m);
        uint64_t s2[2] = {0, 0};
        uint32_t pk[32];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1;
            unpack2(fma2(pack2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), cn2, m2), x0, x1);
            const float w0 = exp2_approx(x0), w1 = exp2_approx(x1);
            s2[(i >> 1) & 1] = add2(s2[(i >> 1) & 1], pack2(w0, w1));
            pk[16 * c + i / 2] = pack_half2(w0, w1);
          }
        tmem_st_x32(t_s + h * kPStep, pk);
        float a, c2;
        unpack2(add2(s2[0], s2[1]), a, c2);
        l += a + c2;
        tmem_st_done();
        tc_fence_before();
        arrive_warp(&b_pready[r][h]);
      }
      t0 = t1;
      }
    // the last step's products (and those before them).  A wait by parity tells a phase from
    // its neighbours only: the steps take two barriers in turn, so that the last phase of
    // each has none behind it and the one before it was done when S of this step came.
    if (ok) ok = wait_all(&b_odone[r][(steps - 1) & 1], ((steps - 1) >> 1) & 1);
    if (active && (ok || tiles == 0)) {
      tc_fence_after();
      const bool whole = gridDim.y == 1;
      const float inv = !whole ? 2.f : (l == 0.f ? 0.f : 2.f / l);  // values entered halved
      T* dst = static_cast<T*>(p.out) + ((first + tok) * p.heads + hd) * D;
      const float kept = exp2_approx(m_kept - m);
      if (!whole && has) *reinterpret_cast<float2*>(p.ml_part + part * 2) = make_float2(m, l);
#pragma unroll 1
      for (int gr = 0; gr < G; ++gr) {
        uint32_t v[2][32];
        if (tiles > 0) {
          tmem_ld_32x32b_x32(t_o + 64 * gr, v[0]);
          tmem_ld_32x32b_x32(t_o + 64 * gr + 32, v[1]);
          tmem_ld_wait();
          if (kLong && steps > kWindow && has) {  // what joined the sums before
            const float4* sum = reinterpret_cast<const float4*>(p.o_part + part * D + 64 * gr);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float4 x = sum[i];
              uint32_t* to = &v[i >> 3][4 * (i & 7)];
              to[0] = __float_as_uint(fmaf(kept, x.x, __uint_as_float(to[0])));
              to[1] = __float_as_uint(fmaf(kept, x.y, __uint_as_float(to[1])));
              to[2] = __float_as_uint(fmaf(kept, x.z, __uint_as_float(to[2])));
              to[3] = __float_as_uint(fmaf(kept, x.w, __uint_as_float(to[3])));
            }
          }
        }
        const bool bad = (nan_groups >> gr) & 1u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // element 8 e + x of the group stands in column 8 x + e
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x)
            f[x] = bad ? NAN : (l == 0.f ? 0.f : __uint_as_float(v[x >> 2][8 * (x & 3) + e]) * inv);
          if (!has) continue;
          if (whole) {
            *reinterpret_cast<uint4*>(dst + 64 * gr + 8 * e) = pack8<T>(f);
          } else {
            float* po = p.o_part + part * D + 64 * gr + 8 * e;
            *reinterpret_cast<float4*>(po) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(po + 4) = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
      }
    }
  } else if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsDecode));
    // ------------------------------------------------------------ decoders
    // Warp dw decodes block dw of every tile (kTwo: its keys or its values).  Keys: lane
    // (r, c) = (lane / 4, lane % 4) takes positions r and r + 8, unit c of each group; values:
    // lane (e, q) takes positions 2 q, 2 q + 1 of each half, elements 8 e .. 8 e + 7 of each
    // group.  Either way a warp reads 512 consecutive bytes at a time.  V^T's row of element 8 e + i of a group is
    // 8 i + e, so that the lanes of a store lie in eight rows of different swizzle.
    const int dw = (warp - 8) % kBlocks;
    const int hi = lane >> 2, lo2 = lane & 3;
    auto decode = [&](auto keys_tag, auto values_tag) {
      constexpr bool does_k = decltype(keys_tag)::value, does_v = decltype(values_tag)::value;
      uint32_t kw[2][2 * G], kpar[2][G], vw[2][2][G], vpar[2][2][G];
      // The page table's entry for this warp's block of tile j, and, one tile later (a use at
      // once would wait for the load), the block; null: no page.
      auto entry = [&](int j) -> int {
        const int pos = j * kTile + dw * kKv4Block;
        return j < tiles && pos < len
                   ? s.page_table[static_cast<int64_t>(b) * s.max_pages + ((at0 + pos) >> s.page_shift)]
                   : -2;
      };
      auto block = [&](int j, int pg) -> const uint8_t* {
        const int64_t pos = static_cast<int64_t>(at0) + j * kTile + dw * kKv4Block;
        const bool there = pg >= 0 && pg < s.num_pages;
        if (!there && pg != -2 && lane == 0) report_device_error(p.status, FITQ_ERR_ARG);
        return there ? p.pool + kv4_block_offset(s, pg, kvh, pos, D) : nullptr;
      };
      // A block without a page reads the pool's first one with scale and low 0.
      auto load_k = [&](const uint8_t* blk) {
        if (blk == nullptr) blk = p.pool;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (G == 2) {
            *reinterpret_cast<uint4*>(kw[i]) = *reinterpret_cast<const uint4*>(blk + i * 512 + lane * 16);
            *reinterpret_cast<uint2*>(kpar[i]) = *reinterpret_cast<const uint2*>(blk + 16 * D + (8 * i + hi) * 16);
          } else {
            *reinterpret_cast<uint2*>(kw[i]) = *reinterpret_cast<const uint2*>(blk + i * 256 + lane * 8);
            kpar[i][0] = *reinterpret_cast<const uint32_t*>(blk + 16 * D + (8 * i + hi) * 8);
          }
        }
      };
      auto load_v = [&](const uint8_t* blk) {
        if (blk == nullptr) blk = p.pool;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (G == 2)
            *reinterpret_cast<uint4*>(vw[h]) = *reinterpret_cast<const uint4*>(blk + 8 * D + h * 512 + lane * 16);
          else
            *reinterpret_cast<uint2*>(vw[h]) = *reinterpret_cast<const uint2*>(blk + 8 * D + h * 256 + lane * 8);
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const uint8_t* ps = blk + 16 * D + (8 * h + 2 * lo2 + o) * 8 * G + 4 * G;
            if (G == 2)
              *reinterpret_cast<uint2*>(vpar[h][o]) = *reinterpret_cast<const uint2*>(ps);
            else
              vpar[h][o][0] = *reinterpret_cast<const uint32_t*>(ps);
          }
        }
      };
      bool ok = tiles > 0;
      int pg_next = entry(1);
      const uint8_t* blk = block(0, entry(0));
      if (ok && does_k) load_k(blk);
      if (ok && does_v) load_v(blk);
      for (int j = 0; ok && j < tiles; ++j) {
        const int buf = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        const bool there = blk != nullptr;
        blk = block(j + 1, pg_next);
        pg_next = entry(j + 2);
        if (does_k) {
          // ---- keys
          if (j >= 2) ok = wait_all(&b_kfree[buf], ph ^ 1u);
          if (!ok) break;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int pos = dw * kKv4Block + 8 * i + hi;  // its swizzle is hi
            const uint32_t dst = s_k + buf * L::kK + pos * 128;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              const uint32_t par = there ? kpar[i][gr] : 0u, half = half_of(par);
              const uint32_t sc = __byte_perm(par, par, 0x1010), lo = __byte_perm(half, half, 0x3232);
              const float2 sl = Half16<__half>::unpack(par);
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const uint32_t x = kw[i][2 * gr + w], y = x >> 8;
                // the eight elements in the order 0 4 1 5 2 6 3 7, as the queries'
                const uint32_t c[4] = {halved_even(x), halved_odd(x), halved_even(y), halved_odd(y)};
                const uint32_t at = dst + gr * (kPTile * 128) + (((2 * lo2 + w) ^ hi) << 4);
                if (kTwo) {
                  Pair2 v[4];
#pragma unroll
                  for (int u = 0; u < 4; ++u) v[u] = value_pair(c[u], sl.x, sl.x, 0.5f * sl.y, 0.5f * sl.y);
                  sts128(at, v[0].hi, v[1].hi, v[2].hi, v[3].hi);
                  sts128(at + kTile * 128, v[0].lo, v[1].lo, v[2].lo, v[3].lo);
                } else {
                  sts128(at, hfma2_u(c[0], sc, lo), hfma2_u(c[1], sc, lo), hfma2_u(c[2], sc, lo), hfma2_u(c[3], sc, lo));
                }
              }
            }
          }
          fence_async_proxy();
          arrive_warp(&b_kfull[buf]);
          if (j + 1 < tiles) load_k(blk);
        }
        if (!does_v) continue;
        // ---- values
        if (j >= 2) ok = wait_all(&b_vfree[buf], ph ^ 1u);
        if (!ok) break;
        int bad[G];  // the block's first position that is not finite, 16: none
#pragma unroll
        for (int gr = 0; gr < G; ++gr) bad[gr] = kKv4Block;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int vpos = j * kTile + dw * kKv4Block + 8 * h + 2 * lo2;
#pragma unroll
          for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              // an exponent of all ones in either half: not finite
              const uint32_t e = vpar[h][o][gr] & 0x7c007c00u;
              if (vpos + o >= len || !there) {
                vpar[h][o][gr] = 0;
              } else if ((e & 0xffffu) == 0x7c00u || (e >> 16) == 0x7c00u) {
                vpar[h][o][gr] = 0;
                bad[gr] = min(bad[gr], 8 * h + 2 * lo2 + o);
              }
            }
        }
        uint32_t note = there ? 1u : 0u;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) note |= __reduce_min_sync(0xffffffffu, static_cast<unsigned>(bad[gr])) << (8 + 8 * gr);
        if (G == 1) note |= kKv4Block << 16;
        if (lane == 0) sh_note[buf][dw] = note;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int h16 = 2 * dw + h;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            const uint32_t sc = __byte_perm(vpar[h][0][gr], vpar[h][1][gr], 0x5410);
            const uint32_t lo = half_of(__byte_perm(vpar[h][0][gr], vpar[h][1][gr], 0x7632));
            const float2 s2 = Half16<__half>::unpack(sc);
            const float2 l2 = Half16<__half>::unpack(__byte_perm(vpar[h][0][gr], vpar[h][1][gr], 0x7632));
            // row 64 gr + 8 i + e, positions 8 h16 + 2 q, + 1
            const uint32_t dst =
                s_v + buf * L::kV + (h16 >> 3) * (D * 128) + (64 * gr + hi) * 128 + (((h16 & 7) ^ hi) << 4) + lo2 * 4;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t x = __byte_perm(vw[h][0][gr], vw[h][1][gr], z ? 0x7632 : 0x5410);
              const uint32_t y = x >> 8;
              const uint32_t c[4] = {halved_even(x), halved_odd(x), halved_even(y), halved_odd(y)};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                if (kTwo) {
                  const Pair2 v = value_pair(c[u], s2.x, s2.y, 0.5f * l2.x, 0.5f * l2.y);
                  sts32(dst + (4 * z + u) * 1024, v.hi);
                  sts32(dst + D * 128 + (4 * z + u) * 1024, v.lo);
                } else {
                  sts32(dst + (4 * z + u) * 1024, hfma2_u(c[u], sc, lo));
                }
              }
            }
          }
        }
        fence_async_proxy();
        arrive_warp(&b_vfull[buf]);
        if (j + 1 < tiles) load_v(blk);
      }
    };
    if constexpr (!kTwo)
      decode(std::true_type{}, std::true_type{});
    else if (warp - 8 < kBlocks)
      decode(std::true_type{}, std::false_type{});
    else
      decode(std::false_type{}, std::true_type{});
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPRegsIssue));
    if (warp == 16 && tiles > 0) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc_s = idesc_f16_f32(kPRows, kPStep), idesc_o = idesc_f16_f32(kPRows, D);
    const uint64_t dq = umma_smem_desc_sw128(s_q), dk = umma_smem_desc_sw128(s_k), dv = umma_smem_desc_sw128(s_v);
    const int steps = (len + kPStep - 1) / kPStep, last = two ? 1 : 0;
    auto issue_s = [&](int r, int t) {  // scores of step t into its half of S_r
      const int h = t & 1, sub = t % kSteps, buf = (t / kSteps) & 1;
#pragma unroll 1
      for (int part = 0; part < (kTwo ? 2 : 1); ++part)
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint64_t qa = dq + ((r * L::kQ + (kk >> 2) * (kPRows * 128) + (kk & 3) * 32) >> 4);
          const uint64_t kb =
              dk + ((buf * L::kK + (kk >> 2) * (kPTile * 128) + (sub + part) * (kPStep * 128) + (kk & 3) * 32) >> 4);
          umma_f16_ss(tmem + r * 128 + h * kPStep, qa, kb, idesc_s, kk > 0 || part > 0 ? 1u : 0u);
        }
      commit_warp(&b_sfull[r][h]);
      // the tile's last scores: its keys' buffer is free
      if (r == last && (sub == kSteps - 1 || t == steps - 1)) commit_warp(&b_kfree[buf]);
    };
    auto issue_o = [&](int r, int t) {  // step t's weights times its values
      const int h = t & 1, sub = t % kSteps, buf = (t / kSteps) & 1;
#pragma unroll 1
      for (int part = 0; part < (kTwo ? 2 : 1); ++part)
#pragma unroll
        for (int kk = 0; kk < kPStep / 16; ++kk) {
          const uint64_t vb = dv + ((buf * L::kV + (sub + part) * (D * 128) + kk * 32) >> 4);
          umma_f16_ts(tmem + 256 + r * 128, tmem + r * 128 + h * kPStep + kk * 8, vb, idesc_o,
                      (kLong ? t % kWindow : t) != 0 || kk > 0 || part > 0 ? 1u : 0u);
        }
      commit_warp(&b_odone[r][h]);
      if (r == last && (sub == kSteps - 1 || t == steps - 1)) commit_warp(&b_vfree[buf]);
    };
    // keys of the tile that step t opens
    auto keys_here = [&](int t) -> bool {
      return t >= steps || t % kSteps != 0 || wait_all(&b_kfull[(t / kSteps) & 1], (t / kSteps >> 1) & 1);
    };
    bool ok = wait_all(&b_qready, 0);
    for (int t = 0; ok && t < 2 && t < steps; ++t) {
      ok = keys_here(t);
      if (!ok) break;
      tc_fence_after();
      for (int r = 0; r <= last; ++r) issue_s(r, t);
    }
    for (int t = 0; ok && t < steps; ++t) {
      const int h = t & 1;
      if (t % kSteps == 0)
        ok = wait_all(&b_vfull[(t / kSteps) & 1], (t / kSteps >> 1) & 1) && (kTwo || keys_here(t + 2));
      for (int r = 0; ok && r <= last; ++r) {
        ok = wait_all(&b_pready[r][h], (t >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        issue_o(r, t);
        if (kTwo && r == 0) {
          ok = keys_here(t + 2);
          tc_fence_after();
        }
        if (ok && t + 2 < steps) issue_s(r, t + 2);
      }
    }
    // every MMA has retired before tensor memory is given back
    commit_warp(&b_done);
    int never = 0;
    mbar_wait(&b_done, 0, &never, p.status);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the parts of the rows.  A CTA takes eight rows of a row pair, a warp each: lane
// c holds the weight of part c, then every lane D / 32 elements.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_prompt_combine_kernel(const Kv4PromptParams p, int splits) {
  constexpr int kE = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();  // the partials
  const Kv4Seq& s = p.seq;
  const int cta = p.cta0 + static_cast<int>(blockIdx.x);
  const int per_pair = s.batch * s.kv_heads;
  const int rp = p.row_pairs - 1 - cta / per_pair, pair = cta % per_pair;
  const int b = pair / s.kv_heads, kvh = pair % s.kv_heads;
  int64_t first;
  int count;
  kv4_tokens(s, b, first, count);
  const int in_cta = static_cast<int>(blockIdx.y) * 8 + warp;
  const int64_t row = static_cast<int64_t>(rp) * 2 * kPRows + in_cta;
  if (row >= static_cast<int64_t>(min(count, p.max_new)) * p.group) return;
  const int64_t part0 = static_cast<int64_t>(blockIdx.x) * splits * (2 * kPRows) + in_cta;  // part c: + c * 256
  float2 ml = make_float2(kPFloor, 0.f);
  if (lane < splits) ml = *reinterpret_cast<const float2*>(p.ml_part + (part0 + lane * (2 * kPRows)) * 2);
  float mx = ml.y == 0.f ? kPFloor : ml.x;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  // a part that saw nothing weighs 0, whatever its rows hold
  const float w = ml.y == 0.f ? 0.f : exp2_approx(ml.x - mx);
  float l = ml.y == 0.f ? 0.f : w * ml.y;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
  const uint32_t live = __ballot_sync(0xffffffffu, ml.y != 0.f);
  float f[kE];
#pragma unroll
  for (int x = 0; x < kE; ++x) f[x] = 0.f;
#pragma unroll 4
  for (int c = 0; c < splits; ++c) {
    const float k = __shfl_sync(0xffffffffu, w, c);
    if (!((live >> c) & 1u)) continue;
    const float* src = p.o_part + (part0 + static_cast<int64_t>(c) * (2 * kPRows)) * D + lane * kE;
    float v[kE];
    if (kE == 4)
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
    else
      *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
    for (int x = 0; x < kE; ++x) f[x] = fmaf(k, v[x], f[x]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* dst = static_cast<T*>(p.out) + ((first + row / p.group) * p.heads + kvh * p.group + row % p.group) * D + lane * kE;
  if (kE == 4)
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(Half16<T>::pack(f[0] * inv, f[1] * inv), Half16<T>::pack(f[kE - 2] * inv, f[kE - 1] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = Half16<T>::pack(f[0] * inv, f[1] * inv);
}

struct PromptPlan {
  int row_pairs, splits;
  bool long_sums;
  int64_t ctas, per_launch;  // without the splits
  size_t o_off, bytes;
};

// steps: window_steps of the type
PromptPlan prompt_plan(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim, int steps,
                       int num_sms) {
  PromptPlan a;
  a.row_pairs = static_cast<int>((group * max_new + 2 * kPRows - 1) / (2 * kPRows));
  a.ctas = static_cast<int64_t>(a.row_pairs) * batch * kv_heads;
  // as many parts as leave no SM a second CTA, of four tiles or more
  int64_t splits = num_sms / a.ctas;
  const int64_t most = (max_len + 4 * kPTile - 1) / (4 * kPTile);
  if (splits > most) splits = most;
  if (splits > kPMaxSplits) splits = kPMaxSplits;
  a.splits = static_cast<int>(splits < 1 ? 1 : splits);
  a.long_sums = max_len > static_cast<int64_t>(steps) * kPStep;
  a.per_launch = a.ctas;
  a.o_off = 0;
  a.bytes = 16;
  if (a.splits > 1 || a.long_sums) {
    const int64_t fits = kPScratch / (2 * kPRows * (dim + 2) * static_cast<int64_t>(sizeof(float)) * a.splits);
    if (a.per_launch > fits) a.per_launch = fits;
    const size_t rows = static_cast<size_t>(a.per_launch) * a.splits * 2 * kPRows;
    a.o_off = (rows * 2 * sizeof(float) + 255) & ~static_cast<size_t>(255);
    a.bytes = a.o_off + rows * dim * sizeof(float);
  }
  return a;
}

template <typename T, int D>
int prompt_t(Kv4PromptParams p, const PromptPlan& a, cudaStream_t st) {
  constexpr int smem = PromptSmem<D>::kBytes;
  // joining sums costs every step registers: 0.6% in bf16, 4% in fp16
  auto* kernel = a.long_sums ? kv4_prompt_kernel<T, D, true> : kv4_prompt_kernel<T, D, false>;
  if (!set_smem_limit(kernel, smem)) return FITQ_ERR_CUDA;
  for (int64_t at = 0; at < a.ctas; at += a.per_launch) {
    const unsigned ctas = static_cast<unsigned>(a.ctas - at < a.per_launch ? a.ctas - at : a.per_launch);
    p.cta0 = static_cast<int>(at);
    cudaError_t e = launch_pdl(kernel, dim3(ctas, a.splits), dim3(kPThreads), smem, st, p);
    note_launch();
    if (e != cudaSuccess) return FITQ_ERR_CUDA;
    if (a.splits == 1) continue;
    e = launch_pdl(kv4_prompt_combine_kernel<T, D>, dim3(ctas, 2 * kPRows / 8), dim3(256), 0, st, p, a.splits);
    note_launch();
    if (e != cudaSuccess) return FITQ_ERR_CUDA;
  }
  return launch_result();
}

}  // namespace

size_t kv4_prompt_workspace(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim,
                            int num_sms) {
  // the query does not know the type
  const size_t a = prompt_plan(batch, kv_heads, group, max_new, max_len, dim, window_steps<__nv_bfloat16>(), num_sms).bytes;
  const size_t b = prompt_plan(batch, kv_heads, group, max_new, max_len, dim, window_steps<__half>(), num_sms).bytes;
  return a > b ? a : b;
}

int launch_kv4_prompt(const Kv4Seq& seq, const void* q, int64_t q_stride, const void* pool, void* out, int heads,
                      int dim, int dtype, int64_t max_new, int64_t max_len, void* workspace, int* status,
                      cudaStream_t st, int num_sms) {
  const int group = heads / seq.kv_heads;
  const int steps = dtype == FITQ_DTYPE_BF16 ? window_steps<__nv_bfloat16>() : window_steps<__half>();
  const PromptPlan a = prompt_plan(seq.batch, seq.kv_heads, group, max_new, max_len, dim, steps, num_sms);
  float* ml = static_cast<float*>(workspace);
  float* o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + a.o_off);
  const Kv4PromptParams p{q, q_stride, out, static_cast<const uint8_t*>(pool), ml, o, heads, group, a.row_pairs,
                          static_cast<int>(max_new), 0, 1.4426950408889634f / sqrtf(static_cast<float>(dim)), status, seq};
  if (dtype == FITQ_DTYPE_BF16)
    return dim == 128 ? prompt_t<__nv_bfloat16, 128>(p, a, st) : prompt_t<__nv_bfloat16, 64>(p, a, st);
  return dim == 128 ? prompt_t<__half, 128>(p, a, st) : prompt_t<__half, 64>(p, a, st);
}

}  // namespace fitq
