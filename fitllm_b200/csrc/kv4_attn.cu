// Attention of new tokens over the 4-bit paged cache (layout: kv4.cuh).
//
//   o[n] = sum_p w_p v_p / sum_p w_p,  w_p = exp(q_n . k_p / sqrt(D)) over the
//   positions p <= prefix + i that token i of its sequence sees; query head h
//   reads KV head h / G, G = H / KVH.
//
// A KV head's G heads and R / G tokens fold into R = 8 NT columns (column =
// token * G + head).  With s, l the scale and low of a group and c its codes,
//   q . k = sum_g s_g (q_g . c_g) + l_g sum(q_g),
//   o     = sum_g [sum_p (w_p s_pg) (c_pg - 8)] + sum_p w_p (l_pg + 8 s_pg),
// so the tensor cores multiply the codes themselves and scales and lows are
// applied in fp32 to scores and weights.  A code becomes a bf16 or fp16 operand
// by OR-ing it into the mantissa of 128 (1024): bf16 keys keep that offset, it is
// taken off with l (one fp32 term per score), values have it subtracted because
// their sums run over the whole cache, where it would cancel badly.
//
// kv4_attn_kernel.  Both products have the cache as the 16-row operand of
// mma.m16n8k16 (S^T = K.Q^T, O^T = V^T.P^T), the R columns as the n8 operand, so
// eight columns cost one MMA; its fragments come straight out of the block
// layout (two 16-byte shared loads per 16 keys, two per 16 values), and P turns
// from accumulator to operand with movmatrix.  Every warp streams its own blocks
// (2,304 B at D = 128, one bulk copy each) through a private ring and keeps its
// own running maximum, sum and output; the warps of a CTA meet once per segment.
//
// Work split.  The 64-position tiles of all (sequence, KV head) pairs form one
// list, cut into equal runs, one per CTA, whatever the sequences' lengths; a CTA
// finds its first pair from the device-side lengths.  A pair that lies in one
// run is written out; one cut between runs leaves partials that
// kv4_attn_combine_kernel joins in run order (deterministic).
//
// Bound: HBM, 18 D / 16 B per position and KV head.
#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

constexpr int kAWarps = 4;
constexpr int kAThreads = 32 * kAWarps;
constexpr int kATile = kKv4Block * kAWarps;  // positions per tile: one block per warp
constexpr int kAStages = 4;                  // blocks in flight per warp
// Running maxima start finite, so that masked scores (-inf) never meet -inf - -inf.
constexpr float kFloor = -3.0e38f;

struct Kv4AttnParams {
  const void* q;
  int64_t q_stride;  // elements per token
  void* out;         // [tokens, H, D]
  const uint8_t* pool;
  float* o_part;  // [row tiles][runs + pairs][R][D]
  float* ml_part; // [row tiles][runs + pairs][R][2]
  int* base;      // [row tiles][batch + 1] first tile of each sequence (per KV head)
  int heads, group;
  float scale_log2;  // log2(e) / sqrt(D)
  int* status;
  Kv4Seq seq;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

template <typename T>
struct Mma16;
template <>
struct Mma16<__nv_bfloat16> {
  static constexpr uint32_t kMagic = 0x43004300u;   // 128 in both halves
  static constexpr uint32_t kCentre = 0x43084308u;  // 136
  static constexpr float kKeyOffset = 128.f;        // what a key operand adds to its code
  static __device__ __forceinline__ uint32_t key(uint32_t c) { return c | kMagic; }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};
template <>
struct Mma16<__half> {
  static constexpr uint32_t kMagic = 0x64006400u;   // 1024 in both halves
  static constexpr uint32_t kCentre = 0x64086408u;  // 1032
  // An offset of 1024 would leave scores of fp16 queries ten bits short of fp32's
  // 24: the key operand is centred too (one more instruction per pair).
  static constexpr float kKeyOffset = -8.f;
  static __device__ __forceinline__ uint32_t key(uint32_t c) { return sub(c | kMagic, kCentre); }
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
};

// Tiles of sequence b that columns [col0, col0 + R) see, and its lengths.
struct SeqSpan {
  int64_t first;  // packed token of the sequence's first new token
  int count;      // new tokens
  int pre;        // cached positions before them
  int cols;       // columns of this row tile that exist
  int len;        // positions the row tile's last column sees
  int tiles;
};

__device__ __forceinline__ SeqSpan seq_span(const Kv4Seq& s, int b, int group, int col0, int R) {
  SeqSpan r;
  kv4_tokens(s, b, r.first, r.count);
  r.pre = s.prefix[b];
  int64_t total = static_cast<int64_t>(r.count) * group - col0;
  r.cols = total <= 0 ? 0 : (total > R ? R : static_cast<int>(total));
  int64_t len = 0;
  if (r.cols > 0 && r.pre >= 0) {
    len = static_cast<int64_t>(r.pre) + (col0 + r.cols - 1) / group + 1;
    const int64_t room = static_cast<int64_t>(s.max_pages) << s.page_shift;
    if (len > room) len = room;
  }
  r.len = static_cast<int>(len);
  // a sequence with columns but no positions still has a tile: its rows are zeros
  r.tiles = r.cols == 0 ? 0 : (r.len == 0 ? 1 : (r.len + kATile - 1) / kATile);
  return r;
}

template <typename T, int D, int NT>
constexpr int kv4_attn_smem() {
  return kAWarps * kAStages * kv4_block_bytes(D) + kAWarps * 8 * NT * (D + 4) * 4 + kAWarps * 8 * NT * 2 * 4 +
         kAWarps * kAStages * 8 + 64;
}

extern __shared__ __align__(128) uint8_t g_kv4_smem[];

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kAThreads, NT == 1 ? 4 : (NT == 2 ? 3 : 2))
    kv4_attn_kernel(const Kv4AttnParams p) {
  constexpr int G = D / 64;            // groups of 64
  constexpr int R = 8 * NT;            // columns
  constexpr int kBlk = kv4_block_bytes(D);
  constexpr int kLd = D + 4;           // row pitch of the merge buffer (floats)
  using M = Mma16<T>;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, qd = lane & 3;
  const int col0 = blockIdx.y * R;

  uint8_t* ring = g_kv4_smem + warp * (kAStages * kBlk);
  float* mrg_o = reinterpret_cast<float*>(g_kv4_smem + kAWarps * kAStages * kBlk);
  float* mrg_ml = mrg_o + kAWarps * R * kLd;  // [warp][R][2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(mrg_ml + kAWarps * R * 2) + warp * kAStages;
  __shared__ int sh_scan[kAWarps], sh_b, sh_base, sh_total;
  __shared__ int sh_abort;

  if (tid == 0) sh_abort = 0;
  if (lane == 0) {
    for (int i = 0; i < kAStages; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  pdl_launch_dependents();
  pdl_wait();  // q and the cache append come from the previous kernels

  const Kv4Seq& s = p.seq;
  // ---- the list of tiles: every thread sums a run of sequences, then a scan
  const int per_thread = (s.batch + kAThreads - 1) / kAThreads;
  const int b_lo = tid * per_thread, b_hi = b_lo + per_thread < s.batch ? b_lo + per_thread : s.batch;
  int mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += seq_span(s, b, p.group, col0, R).tiles;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sh_scan[warp] = incl;
  __syncthreads();
  int before = incl - mine;
  for (int w = 0; w < warp; ++w) before += sh_scan[w];
  int all = 0;
  for (int w = 0; w < kAWarps; ++w) all += sh_scan[w];
  const int64_t total = static_cast<int64_t>(all) * s.kv_heads;
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;  // tiles per run
  int* base = p.base + static_cast<int64_t>(blockIdx.y) * (s.batch + 1);
  int64_t t_lo = per * blockIdx.x, t_hi = t_lo + per < total ? t_lo + per : total;
  if (tid == 0) {
    sh_b = s.batch;
    sh_total = all;
  }
  __syncthreads();
  {
    int at = before;
    for (int b = b_lo; b < b_hi; ++b) {
      const SeqSpan sp = seq_span(s, b, p.group, col0, R);
      if (blockIdx.x == 0) base[b] = at;
      // sequence b covers tiles [at * KVH, (at + tiles) * KVH) of the list
      if (t_lo < t_hi && static_cast<int64_t>(at) * s.kv_heads <= t_lo &&
          t_lo < static_cast<int64_t>(at + sp.tiles) * s.kv_heads) {
        sh_b = b;
        sh_base = at;
      }
      at += sp.tiles;
      // more columns than the launch covers, or positions outside the table
      if (blockIdx.x == 0 &&
          (sp.pre < 0 || (blockIdx.y == 0 && static_cast<int64_t>(sp.count) * p.group > static_cast<int64_t>(gridDim.y) * R) ||
           (blockIdx.y == 0 && sp.count > 0 &&
            static_cast<int64_t>(sp.pre) + sp.count > (static_cast<int64_t>(s.max_pages) << s.page_shift))))
        report_device_error(p.status, FITQ_ERR_ARG);
    }
    if (blockIdx.x == 0 && tid == 0) base[s.batch] = all;
  }
  __syncthreads();
  if (t_lo >= t_hi) return;
  int b = sh_b;
  int64_t seq_t0 = static_cast<int64_t>(sh_base) * s.kv_heads;  // first list tile of sequence b

  const int64_t slot0 = static_cast<int64_t>(blockIdx.y) * (gridDim.x + static_cast<int64_t>(s.batch) * s.kv_heads);
  uint32_t issued = 0, taken = 0;  // this warp's copies so far

  int64_t t = t_lo;
  while (t < t_hi) {
    SeqSpan sp = seq_span(s, b, p.group, col0, R);
    while (sp.tiles == 0 || t >= seq_t0 + static_cast<int64_t>(sp.tiles) * s.kv_heads) {  // next sequence with work
      seq_t0 += static_cast<int64_t>(sp.tiles) * s.kv_heads;
      ++b;
      sp = seq_span(s, b, p.group, col0, R);
    }
    const int kvh = static_cast<int>((t - seq_t0) / sp.tiles);
    const int64_t pair_t0 = seq_t0 + static_cast<int64_t>(kvh) * sp.tiles;
    const int ta = static_cast<int>(t - pair_t0);
    int tb = sp.tiles;
    if (pair_t0 + tb > t_hi) tb = static_cast<int>(t_hi - pair_t0);
    const bool whole = ta == 0 && tb == sp.tiles;

    // ---- this warp's blocks: block j at position ta * kATile + 16 (warp + 4 j)
    const int pos_first = ta * kATile + kKv4Block * warp;
    const int pos_end = tb * kATile < sp.len ? tb * kATile : sp.len;
    const int blocks = pos_first < pos_end ? (pos_end - pos_first + kATile - 1) / kATile : 0;
    int pages = -1;   // lane j: page of block 32 * (j / 32) + lane
    auto load_pages = [&](int j0) {
      const int j = j0 + lane;
      pages = -1;
      if (j < blocks) {
        pages = kv4_page(s, b, pos_first + static_cast<int64_t>(j) * kATile);
        if (pages < 0) report_device_error(p.status, FITQ_ERR_ARG);
      }
    };
    auto issue = [&](int pg, int j) {  // whole warp; pg uniform
      if (pg < 0) return;
      const int st = issued % kAStages;
      if (lane == 0) {
        mbar_arrive_expect_tx(&bars[st], kBlk);
        bulk_load(ring + st * kBlk,
                  p.pool + kv4_block_offset(s, pg, kvh, pos_first + static_cast<int64_t>(j) * kATile, D), kBlk,
                  &bars[st]);
      }
      ++issued;
    };
    load_pages(0);
    uint32_t valid = __ballot_sync(0xffffffffu, pages >= 0);  // blocks 32 k .. of the current page set
    int next = 0;                                             // next block to issue
    uint32_t next_valid = 0;  // validity of the page set that starts at next_set
    int cur_pages = pages;
    // blocks are consumed in order; the copies run at most kAStages ahead of block `done`
    auto issue_next = [&](int done) {
      while (next < blocks && next < done + kAStages) {
        if ((next & 31) == 0 && next > 0) {
          load_pages(next);
          cur_pages = pages;
          next_valid = __ballot_sync(0xffffffffu, pages >= 0);
        }
        const int pg = __shfl_sync(0xffffffffu, cur_pages, next & 31);
        issue(pg, next);
        ++next;
      }
    };
    issue_next(0);

    // ---- query fragments (column n = 8 nt + g), their group sums, column limits
    uint32_t qf[NT][G][2][4];
    float qs[NT][2][G];  // offset-corrected sums belong to the columns 2 qd, 2 qd + 1
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = 8 * nt + g;
      const bool has = n < sp.cols;
      const int tok = (col0 + n) / p.group, hd = (col0 + n) % p.group;
      const T* src = static_cast<const T*>(p.q) + (sp.first + tok) * p.q_stride +
                     static_cast<int64_t>(kvh * p.group + hd) * D;
      float sum[G];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        sum[gr] = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (has) u = *reinterpret_cast<const uint4*>(src + 64 * gr + 16 * qd + 8 * w);
          float f[8];
          unpack8<T>(u, f);
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[gr] += f[i];
          // pairs (e, e + 4): the order in which the codes leave their word
          qf[nt][gr][w][0] = __byte_perm(u.x, u.z, 0x5410);
          qf[nt][gr][w][1] = __byte_perm(u.x, u.z, 0x7632);
          qf[nt][gr][w][2] = __byte_perm(u.y, u.w, 0x5410);
          qf[nt][gr][w][3] = __byte_perm(u.y, u.w, 0x7632);
        }
        sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
        sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
        qs[nt][0][gr] = __shfl_sync(0xffffffffu, sum[gr], 8 * qd);
        qs[nt][1][gr] = __shfl_sync(0xffffffffu, sum[gr], 8 * qd + 4);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int l = sp.pre + (col0 + 8 * nt + 2 * qd + e) / p.group;
        lim[nt][e] = l < sp.len ? l : sp.len - 1;
      }
    }
    const int mask_from = sp.pre + col0 / p.group + 1;  // positions every column sees lie before it

    float m_run[NT][2], l_run[NT][2], corr[NT][2][G], o[NT][G][4][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m_run[nt][e] = kFloor;
        l_run[nt][e] = 0.f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) corr[nt][e][gr] = 0.f;
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][gr][i][e] = 0.f;
    }

    uint32_t cur_valid = valid;
    for (int j = 0; j < blocks; ++j) {
      if ((j & 31) == 0 && j > 0) cur_valid = next_valid;
      if (!((cur_valid >> (j & 31)) & 1u)) {  // no page: the block is hidden from every column
        issue_next(j + 1);
        continue;
      }
      const int st = taken % kAStages;
      if (!mbar_wait(&bars[st], (taken / kAStages) & 1u, &sh_abort, p.status)) break;
      const uint8_t* blk = ring + st * kBlk;
      const int pos0 = pos_first + j * kATile;

      // ---- S^T = K.Q^T, one accumulator set per group
      float acc[NT][G][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][gr][e] = 0.f;
      uint32_t kw[2][2 * G];
      if (G == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(kw[h]) = *reinterpret_cast<const uint4*>(blk + h * 512 + lane * 16);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint2*>(kw[h]) = *reinterpret_cast<const uint2*>(blk + h * 256 + lane * 8);
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t x = kw[0][2 * gr + w], y = kw[1][2 * gr + w];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t a0 = M::key((x >> (8 * h)) & 0x000f000fu);
            const uint32_t a1 = M::key((y >> (8 * h)) & 0x000f000fu);
            const uint32_t a2 = M::key((x >> (8 * h + 4)) & 0x000f000fu);
            const uint32_t a3 = M::key((y >> (8 * h + 4)) & 0x000f000fu);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              M::mma(acc[nt][gr], a0, a1, a2, a3, qf[nt][gr][w][2 * h], qf[nt][gr][w][2 * h + 1]);
          }
        }

      // ---- parameters of positions g and g + 8: {key, value} x groups x (scale, low)
      float ks[2][G], kl[2][G], vs[2][G], vl[2][G];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t pr[2 * G];
        const uint8_t* src = blk + 16 * D + (g + 8 * h) * 8 * G;
        if (G == 2)
          *reinterpret_cast<uint4*>(pr) = *reinterpret_cast<const uint4*>(src);
        else
          *reinterpret_cast<uint2*>(pr) = *reinterpret_cast<const uint2*>(src);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          const float2 a = Half16<__half>::unpack(pr[gr]);
          const float2 c = Half16<__half>::unpack(pr[G + gr]);
          ks[h][gr] = a.x;
          kl[h][gr] = fmaf(-M::kKeyOffset, a.x, a.y);
          vs[h][gr] = c.x;
          vl[h][gr] = fmaf(8.f, c.x, c.y);
        }
      }
      float sc[NT][4];  // (position g: columns 2 qd, 2 qd + 1; position g + 8: the same)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int h = e >> 1;
          float v = 0.f;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            v = fmaf(ks[h][gr], acc[nt][gr][e], v);
            v = fmaf(kl[h][gr], qs[nt][e & 1][gr], v);
          }
          sc[nt][e] = v;
        }
      const bool edge = pos0 + kKv4Block > mask_from;
      if (edge) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (pos0 + g + 8 * (e >> 1) > lim[nt][e & 1]) sc[nt][e] = -INFINITY;
      }

      // ---- running maximum per column (over the eight lanes that share qd)
      bool grew = false;
      float m_new[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(sc[nt][e], sc[nt][2 + e]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          m_new[nt][e] = fmaxf(m_run[nt][e], mx);
          grew |= m_new[nt][e] > m_run[nt][e];
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float al = exp2_approx((m_run[nt][e] - m_new[nt][e]) * p.scale_log2);
            m_run[nt][e] = m_new[nt][e];
            l_run[nt][e] *= al;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              corr[nt][e][gr] *= al;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[nt][gr][i][e] *= al;
                o[nt][gr][i][2 + e] *= al;
              }
            }
          }
      }

      // ---- weights, their scaled copies per group as the n8 operand of O^T
      uint32_t pb[NT][G][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = exp2_approx((sc[nt][e] - m_run[nt][e & 1]) * p.scale_log2);
          l_run[nt][e & 1] += w[e];
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          float ws[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1;
            ws[e] = w[e] * vs[h][gr];
            float add = w[e] * vl[h][gr];
            if (edge && pos0 + g + 8 * h > lim[nt][e & 1]) ws[e] = add = 0.f;  // whatever the hidden value holds
            corr[nt][e & 1][gr] += add;
          }
          pb[nt][gr][0] = movmatrix_t(Half16<T>::pack(ws[0], ws[1]));
          pb[nt][gr][1] = movmatrix_t(Half16<T>::pack(ws[2], ws[3]));
        }
      }

      // ---- O^T += (V - 8)^T.P^T: rows g, g + 8 of m-tile i are elements 2 i, 2 i + 1 of eight
      uint32_t vw[2][2][G];  // half h, position parity, group
      if (G == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint4*>(vw[h]) = *reinterpret_cast<const uint4*>(blk + 8 * D + h * 512 + lane * 16);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<uint2*>(vw[h]) = *reinterpret_cast<const uint2*>(blk + 8 * D + h * 256 + lane * 8);
      }
      __syncwarp();  // every lane has read the block
      ++taken;
      issue_next(j + 1);
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const uint32_t x = __byte_perm(vw[0][0][gr], vw[0][1][gr], z ? 0x7632 : 0x5410);
          const uint32_t y = __byte_perm(vw[1][0][gr], vw[1][1][gr], z ? 0x7632 : 0x5410);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t a0 = M::sub(((x >> (8 * i)) & 0x000f000fu) | M::kMagic, M::kCentre);
            const uint32_t a1 = M::sub(((x >> (8 * i + 4)) & 0x000f000fu) | M::kMagic, M::kCentre);
            const uint32_t a2 = M::sub(((y >> (8 * i)) & 0x000f000fu) | M::kMagic, M::kCentre);
            const uint32_t a3 = M::sub(((y >> (8 * i + 4)) & 0x000f000fu) | M::kMagic, M::kCentre);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              M::mma(o[nt][gr][2 * z + i], a0, a1, a2, a3, pb[nt][gr][0], pb[nt][gr][1]);
          }
        }
    }

    if (sh_abort) {  // a wait ran out: the copies still in flight land before the CTA leaves
      int none = 0;
      for (; taken != issued; ++taken)
        mbar_wait_for(&bars[taken % kAStages], (taken / kAStages) & 1u, &none, p.status, kWaitLimitNs);
    }

    // ---- the warps' results meet in shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l_run[nt][e] += __shfl_xor_sync(0xffffffffu, l_run[nt][e], x);
#pragma unroll
          for (int gr = 0; gr < G; ++gr) corr[nt][e][gr] += __shfl_xor_sync(0xffffffffu, corr[nt][e][gr], x);
        }
        const int n = 8 * nt + 2 * qd + e;
        float* row = mrg_o + (warp * R + n) * kLd;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          const float c = corr[nt][e][gr];
          float* dst = row + 64 * gr + 8 * g;
          *reinterpret_cast<float4*>(dst) =
              make_float4(o[nt][gr][0][e] + c, o[nt][gr][0][2 + e] + c, o[nt][gr][1][e] + c, o[nt][gr][1][2 + e] + c);
          *reinterpret_cast<float4*>(dst + 4) =
              make_float4(o[nt][gr][2][e] + c, o[nt][gr][2][2 + e] + c, o[nt][gr][3][e] + c, o[nt][gr][3][2 + e] + c);
        }
        if (g == 0) *reinterpret_cast<float2*>(mrg_ml + (warp * R + n) * 2) = make_float2(m_run[nt][e], l_run[nt][e]);
      }
    __syncthreads();
    const int64_t slot = slot0 + blockIdx.x + static_cast<int64_t>(b) * s.kv_heads + kvh;
    for (int i = tid; i < sp.cols * (D / 8); i += kAThreads) {
      const int n = i / (D / 8), d0 = (i % (D / 8)) * 8;
      float mx = kFloor;
#pragma unroll
      for (int w = 0; w < kAWarps; ++w) mx = fmaxf(mx, mrg_ml[(w * R + n) * 2]);
      float l = 0.f, f[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) f[x] = 0.f;
#pragma unroll
      for (int w = 0; w < kAWarps; ++w) {
        const float2 ml = *reinterpret_cast<const float2*>(mrg_ml + (w * R + n) * 2);
        if (ml.y == 0.f) continue;  // this warp saw no position of the column
        const float k = exp2_approx((ml.x - mx) * p.scale_log2);
        l += k * ml.y;
        const float* row = mrg_o + (w * R + n) * kLd + d0;
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = fmaf(k, row[x], f[x]);
      }
      if (whole) {
        const float inv = 1.f / l;
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = l == 0.f ? 0.f : f[x] * inv;
        const int tok = (col0 + n) / p.group, hd = (col0 + n) % p.group;
        T* dst = static_cast<T*>(p.out) + ((sp.first + tok) * p.heads + kvh * p.group + hd) * D + d0;
        *reinterpret_cast<uint4*>(dst) = pack8<T>(f);
      } else {
        float* dst = p.o_part + (slot * R + n) * D + d0;
        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        if (d0 == 0) *reinterpret_cast<float2*>(p.ml_part + (slot * R + n) * 2) = make_float2(mx, l);
      }
    }
    __syncthreads();  // the merge buffer is free again
    t = pair_t0 + tb;
    if (sh_abort) break;
  }
}

// Joins the runs that a pair was cut into, in run order.  Grid (batch * KVH, row
// tiles), D / 8 lanes per column.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) kv4_attn_combine_kernel(const Kv4AttnParams p, int runs) {
  constexpr int R = 8 * NT;
  pdl_launch_dependents();
  pdl_wait();  // the partials
  const Kv4Seq& s = p.seq;
  const int b = blockIdx.x / s.kv_heads, kvh = blockIdx.x % s.kv_heads;
  const int* base = p.base + static_cast<int64_t>(blockIdx.y) * (s.batch + 1);
  const int64_t total = static_cast<int64_t>(base[s.batch]) * s.kv_heads;
  const int tiles = base[b + 1] - base[b];
  if (tiles == 0) return;
  const int64_t per = (total + runs - 1) / runs;
  const int64_t t0 = static_cast<int64_t>(base[b]) * s.kv_heads + static_cast<int64_t>(kvh) * tiles;
  const int64_t c0 = t0 / per, c1 = (t0 + tiles - 1) / per;
  if (c0 == c1) return;  // written by its one run
  const int col0 = blockIdx.y * R;
  const SeqSpan sp = seq_span(s, b, p.group, col0, R);
  const int64_t slot0 = static_cast<int64_t>(blockIdx.y) * (runs + static_cast<int64_t>(s.batch) * s.kv_heads) +
                        static_cast<int64_t>(b) * s.kv_heads + kvh;
  for (int i = threadIdx.x; i < sp.cols * (D / 8); i += 128) {
    const int n = i / (D / 8), d0 = (i % (D / 8)) * 8;
    float mx = kFloor;
    for (int64_t c = c0; c <= c1; ++c) mx = fmaxf(mx, p.ml_part[((slot0 + c) * R + n) * 2]);
    float l = 0.f, f[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = 0.f;
    for (int64_t c = c0; c <= c1; ++c) {
      const float2 ml = *reinterpret_cast<const float2*>(p.ml_part + ((slot0 + c) * R + n) * 2);
      if (ml.y == 0.f) continue;
      const float k = exp2_approx((ml.x - mx) * p.scale_log2);
      l += k * ml.y;
      const float4* src = reinterpret_cast<const float4*>(p.o_part + ((slot0 + c) * R + n) * D + d0);
      const float4 a = src[0], c4 = src[1];
      f[0] = fmaf(k, a.x, f[0]); f[1] = fmaf(k, a.y, f[1]); f[2] = fmaf(k, a.z, f[2]); f[3] = fmaf(k, a.w, f[3]);
      f[4] = fmaf(k, c4.x, f[4]); f[5] = fmaf(k, c4.y, f[5]); f[6] = fmaf(k, c4.z, f[6]); f[7] = fmaf(k, c4.w, f[7]);
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int x = 0; x < 8; ++x) f[x] = l == 0.f ? 0.f : f[x] * inv;
    const int tok = (col0 + n) / p.group, hd = (col0 + n) % p.group;
    T* dst = static_cast<T*>(p.out) + ((sp.first + tok) * p.heads + kvh * p.group + hd) * D + d0;
    *reinterpret_cast<uint4*>(dst) = pack8<T>(f);
  }
}

// Columns of a call: tokens of a sequence x heads of a KV head, in n8 tiles.
int col_tiles(int group, int64_t max_new) {
  const int64_t cols = static_cast<int64_t>(group) * max_new;
  return cols <= 8 ? 1 : (cols <= 16 ? 2 : 4);
}

struct AttnPlan {
  int nt, row_tiles, runs;
  size_t base_off, ml_off, o_off, bytes;
};

AttnPlan attn_plan(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim, int num_sms) {
  AttnPlan a;
  a.nt = col_tiles(group, max_new);
  const int R = 8 * a.nt;
  a.row_tiles = static_cast<int>((group * max_new + R - 1) / R);
  const int ctas = a.nt == 1 ? 4 : (a.nt == 2 ? 3 : 2);
  const int64_t pairs = static_cast<int64_t>(batch) * kv_heads;
  const int64_t tiles = pairs * ((max_len + kATile - 1) / kATile);
  int64_t runs = static_cast<int64_t>(num_sms) * ctas;
  if (a.row_tiles > 1) runs = (runs + a.row_tiles - 1) / a.row_tiles;
  if (runs > tiles) runs = tiles;
  a.runs = static_cast<int>(runs < 1 ? 1 : runs);
  const size_t slots = static_cast<size_t>(a.row_tiles) * (a.runs + pairs);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  a.base_off = 0;
  a.ml_off = up(static_cast<size_t>(a.row_tiles) * (batch + 1) * sizeof(int));
  a.o_off = a.ml_off + up(slots * R * 2 * sizeof(float));
  a.bytes = a.o_off + slots * R * dim * sizeof(float);
  return a;
}

template <typename T, int D, int NT>
int attn_t(const Kv4AttnParams& p, const AttnPlan& a, cudaStream_t st) {
  constexpr int smem = kv4_attn_smem<T, D, NT>();
  if (!set_smem_limit(kv4_attn_kernel<T, D, NT>, smem)) return FITQ_ERR_CUDA;
  cudaError_t e = launch_pdl(kv4_attn_kernel<T, D, NT>, dim3(a.runs, a.row_tiles), dim3(kAThreads), smem, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  e = launch_pdl(kv4_attn_combine_kernel<T, D, NT>, dim3(p.seq.batch * p.seq.kv_heads, a.row_tiles), dim3(128), 0, st,
                 p, a.runs);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T, int D>
int attn_td(const Kv4AttnParams& p, const AttnPlan& a, cudaStream_t st) {
  return a.nt == 1 ? attn_t<T, D, 1>(p, a, st) : (a.nt == 2 ? attn_t<T, D, 2>(p, a, st) : attn_t<T, D, 4>(p, a, st));
}

}  // namespace

size_t kv4_attention_workspace(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim,
                               int num_sms) {
  return attn_plan(batch, kv_heads, group, max_new, max_len, dim, num_sms).bytes;
}

int launch_kv4_attention(const Kv4Seq& seq, const void* q, int64_t q_stride, const void* pool, void* out, int heads,
                         int dim, int dtype, int64_t max_new, int64_t max_len, void* workspace, int* status,
                         cudaStream_t st, int num_sms) {
  const int group = heads / seq.kv_heads;
  const AttnPlan a = attn_plan(seq.batch, seq.kv_heads, group, max_new, max_len, dim, num_sms);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Kv4AttnParams p;
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.pool = static_cast<const uint8_t*>(pool);
  p.base = reinterpret_cast<int*>(ws + a.base_off);
  p.ml_part = reinterpret_cast<float*>(ws + a.ml_off);
  p.o_part = reinterpret_cast<float*>(ws + a.o_off);
  p.heads = heads;
  p.group = group;
  p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(dim));
  p.status = status;
  p.seq = seq;
  if (dtype == FITQ_DTYPE_BF16)
    return dim == 128 ? attn_td<__nv_bfloat16, 128>(p, a, st) : attn_td<__nv_bfloat16, 64>(p, a, st);
  return dim == 128 ? attn_td<__half, 128>(p, a, st) : attn_td<__half, 64>(p, a, st);
}

}  // namespace fitq
