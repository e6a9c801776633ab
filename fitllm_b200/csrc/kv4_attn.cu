// Attention of new tokens over the 4-bit paged cache (layout: kv4.cuh).
//
//   o[n] = sum_p w_p v_p / sum_p w_p,  w_p = exp(q_n . k_p / sqrt(D)) over the
//   positions p <= prefix + i that token i of its sequence sees; query head h
//   reads KV head h / G, G = H / KVH.
//
// A KV head's G heads and R / G tokens fold into R = 8 NT columns (column =
// token * G + head).  With s, l the scale and low of a group and c its codes,
//   q . k = sum_g s_g (q_g . c_g) + sum_g l_g sum(q_g),
//   o     = sum_g [sum_p (w_p s_pg) c_pg - 8 sum_p (w_p s_pg)] + sum_p w_p (l_pg + 8 s_pg),
// so the tensor cores multiply the codes themselves: one logic instruction leaves two
// codes of a word as the fp16 subnormals 2^-24 c (even elements) or 2^-20 c (odd ones, q
// / 16 against them), exact in the product, and the factors go back in once per score
// and per output.  What else is a sum over positions or groups is an MMA of few rows as
// well: the lows against the queries' sums (in two fp16 pieces), the weights against the
// scales, lows and a one (the denominator: of the rounded weights, so that their rounding
// cancels where it is common), and the eights, whose product is taken off exactly where
// the scaled weights' own rounding would leave a constant behind.
// Both products run in fp16 whatever the type of q.  Queries are multiplied by a power of
// two per column (their largest element goes to 2^15, which keeps the eight bits of a
// bf16 value over 2^29 of range).  Weights are rounded to fp16 by half a step, 2^-11
// (bf16's is 2^-8), and for bf16 results, whose own rounding is eight times that, once
// more behind their product with the scale; for fp16 results that product is taken in
// fp32 and rounded once.  Both stay below 2^15.  Scores, maxima, denominators and outputs
// are fp32.
//
// An MMA's sum rounds towards zero at the accumulator's size, and sums of codes and lows grow
// with the positions where the output, their small difference, shrinks.  So every 32 blocks
// (fp16 results of more than 2^15 positions: 8) a warp adds what it has, the difference taken,
// to its part in shared memory, rounded to nearest, and starts anew.  Relative errors of 5 heads
// over 131,072 positions, 640 sequences: bf16 1.1e-2 -> 1.7e-3, fp16 1.3e-2 -> 3.0e-4; over a
// million, 16 sequences: 1.0e-2 -> 1.7e-3 and 1.1e-2 -> 3.8e-4.  It costs 1.4 us of 78 (64
// sequences), in registers rather than in its own work.
//
// A scale that is no number only makes its own group's elements of the columns that see
// it none: it reaches them through the parameters' products, and enters the scaled
// weights as zero.
//
// kv4_attn_kernel.  Both products have the cache as the 16-row operand of
// mma.m16n8k16 (S^T = K.Q^T, O^T = V^T.P^T), the R columns as the n8 operand, so
// eight columns cost one MMA; its fragments come straight out of the block
// layout (two 16-byte shared loads per 16 keys, two per 16 values), and P turns
// from accumulator to operand with movmatrix.  Every warp streams its own blocks
// (2,304 B at D = 128, one bulk copy each) through a private ring and keeps its
// own reference maximum, sum and output; the warps of a CTA meet once per segment.
// It takes two blocks at a time, so that one's products run in the other's latencies
// (64 sequences of 100 to 8,191 positions, 40 heads on 8: 86.1 -> 83.9 us; 131,072
// positions of one: 42.9 -> 40.3 us).  The reference only moves when a score exceeds it
// by 2^8 in weight: a vote per two blocks instead of a reduction, the sums have the range
// to spare.  Pages of the next segment are looked up and its queries fetched when a
// segment begins, its first copies take the places that the last blocks leave.
//
// Work split.  The tiles (one block per warp) of all (sequence, KV head) pairs
// form one list, cut into equal runs, one per CTA, whatever the sequences'
// lengths; a CTA finds its first pair from the device-side lengths.  A pair that
// lies in one run is written out; one cut between runs leaves partials that
// kv4_attn_combine_kernel joins in run order (deterministic).
//
// Few pairs of few positions (a single sequence's decode step) take the same kernel
// in clusters: eight CTAs share a pair's tiles and join their parts over distributed
// shared memory, one launch without partials in HBM and without the list (one sequence
// of 1,024 positions: 5.9 us).
//
// Bound: HBM, 18 D / 16 B per position and KV head, and the instructions of a block (some
// 310 for eight columns, of 380 that an SM's schedulers have time for at 6.5 TB/s).  The
// 64 sequences above take 78.8 us, 4.0 TB/s; 200 of them 217 us, 4.5 TB/s; inside the
// loop it is 5.5 TB/s, the rest is the start (5 us until the first block), the two CTAs
// of an SM ending apart and the join (4 us).
#include <type_traits>

#include "kv4.cuh"
#include "kernels.cuh"

namespace fitq {
namespace {

// Warps per CTA by column tiles; both shapes leave two CTAs to an SM.  Sixteen columns are
// the most a warp takes: with 32 the output alone is 128 registers a thread; more columns
// are further row tiles, whose reads hit L2.
template <int NT>
struct AttnShape {
  static constexpr int kWarps = NT == 1 ? 8 : 4;
  static constexpr int kCtas = 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kTile = kKv4Block * kWarps;  // positions per tile
  static constexpr int kStages = 4;                 // blocks in flight per warp
};
// Running maxima start finite, so that masked scores (-inf) never meet -inf - -inf.
constexpr float kFloor = -3.0e38f;

// The pair that a run opens and leaves to the runs behind it: `count` runs hold
// parts of it (0: none), the first in `slot`.
struct __align__(16) Kv4Cut {
  int64_t first;  // packed token of the sequence's first new token
  int count, cols, slot, kvh;
};

struct Kv4AttnParams {
  const void* q;
  int64_t q_stride;  // elements per token
  void* out;         // [tokens, H, D]
  const uint8_t* pool;
  float* o_part;  // [row tiles][runs + pairs][R][D]
  float* ml_part; // [row tiles][runs + pairs][R][2]
  Kv4Cut* cuts;   // [row tiles][runs]
  int heads, group;
  int max_new;    // the most new tokens of a sequence that the launch covers
  int group_mul;  // ceil(2^16 / group): n / group for n of a few hundred
  float scale_log2;  // log2(e) / sqrt(D)
  int* status;
  Kv4Seq seq;
};

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                        uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d = a.b.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// d = a.b with eight along k.
__device__ __forceinline__ void mma_f16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

// Two 8 x 8 matrices of 16-bit elements, transposed; lanes 0-15 give the rows' addresses.
__device__ __forceinline__ void ldmatrix2_t(uint32_t& a, uint32_t& b, const void* row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];"
               : "=r"(a), "=r"(b)
               : "r"(smem_u32(row))
               : "memory");
}

// N neighbouring words (1 or 2) of shared memory.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* at) {
  if (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    w[0] = v.x;
    w[N - 1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(at);
  }
}

__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(as_half2(a), as_half2(b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Tiles of sequence b that columns [col0, col0 + R) see, and its lengths.  Tokens from
// max_new on have no columns, whatever the device-side counts say.
struct Columns {
  int group, mul, max_new;
  __device__ __forceinline__ int token(int n) const { return (n * mul) >> 16; }
};

struct SeqSpan {
  int64_t first;  // packed token of the sequence's first new token
  int count;      // new tokens
  int pre;        // cached positions before them
  int cols;       // columns of this row tile that exist
  int len;        // positions the row tile's last column sees
  int tiles;
};

__device__ __forceinline__ SeqSpan seq_span(const Kv4Seq& s, int b, const Columns& c, int col0, int R, int tile) {
  SeqSpan r;
  kv4_tokens(s, b, r.first, r.count);
  r.pre = s.prefix[b];
  int64_t total = static_cast<int64_t>(min(r.count, c.max_new)) * c.group - col0;
  r.cols = total <= 0 ? 0 : (total > R ? R : static_cast<int>(total));
  int64_t len = 0;
  if (r.cols > 0 && r.pre >= 0) {
    len = static_cast<int64_t>(r.pre) + c.token(col0 + r.cols - 1) + 1;
    const int64_t room = static_cast<int64_t>(s.max_pages) << s.page_shift;
    if (len > room) len = room;
  }
  r.len = static_cast<int>(len);
  // a sequence with columns but no positions still has a tile: its rows are zeros
  r.tiles = r.cols == 0 ? 0 : (r.len == 0 ? 1 : (r.len + tile - 1) / tile);
  return r;
}

template <int D, int NT>
struct AttnSmem {
  using S = AttnShape<NT>;
  static constexpr int kR = 8 * NT;
  static constexpr int kLd = D + 4;  // row pitch of the merge buffer (floats)
  static constexpr int kRing = S::kWarps * S::kStages * kv4_block_bytes(D);
  static constexpr int kMerge = S::kWarps * kR * kLd * 4;
  static constexpr int kMl = kRing + kMerge;                        // [warp][R][2] floats
  // queries of two segments, each: fragments [group][word][nt][lane] uint4, then
  // group sums [R][D / 64] (half2: value, rest) and the exponent factors [R]
  static constexpr int kQ = kMl + S::kWarps * kR * 2 * 4;
  static constexpr int kQsum = (D / 64) * 2 * NT * 512;
  static constexpr int kQexp = kQsum + kR * (D / 64) * 4;
  static constexpr int kQBytes = (kQexp + kR * 4 + 15) & ~15;
  static constexpr int kRaw = kQ + 2 * kQBytes;  // queries of the next segment as they came [R][D]
  static constexpr int kBars = kRaw + kR * D * 2;
  static constexpr int kBytes = kBars + S::kWarps * S::kStages * 8;
};

// Weights, and weights times scales, stay below 2^15 in fp16; a reference that moves
// leaves this much (log2) to the weights that follow.
constexpr float kRoom = 15.f, kSlack = 8.f;
constexpr float kGaveUp = -1.f;  // the cap of a lane whose wait ran out
// A pair's first tile costs a run this many tiles more (the warps' meeting, the first
// blocks' reference): runs are cut by cost.  64 sequences of 100 to 8,191 positions take
// 83.9, 75.5, 78.5 us with 2, 4, 8.
constexpr int kPairCost = 4;
__device__ __forceinline__ int pair_cost(const SeqSpan& sp) { return sp.tiles ? sp.tiles + kPairCost : 0; }

extern __shared__ __align__(128) uint8_t g_kv4_smem[];

constexpr int kCluster = 8;  // CTAs per pair of a cluster launch

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Four floats of the same shared-memory address in another CTA of the cluster.
__device__ __forceinline__ float4 peer_float4(const float* p, uint32_t rank) {
  uint32_t a;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

template <typename T, int D, int NT, bool kClustered>
__global__ void __launch_bounds__(AttnShape<NT>::kThreads, AttnShape<NT>::kCtas)
    kv4_attn_kernel(const Kv4AttnParams p) {
  using S = AttnShape<NT>;
  using L = AttnSmem<D, NT>;
  constexpr int G = D / 64;   // groups of 64
  constexpr int R = 8 * NT;   // columns
  constexpr int kBlk = kv4_block_bytes(D);
  constexpr int kLd = L::kLd;
  constexpr int kWarps = S::kWarps, kTile = S::kTile, kStages = S::kStages, kThreads = S::kThreads;
  // fp16 results show the weights' rounding before their scaling: there they are scaled in fp32
  constexpr bool kOnce = std::is_same<T, __half>::value;
  constexpr int kLong = 1 << 15;  // positions from which fp16 sums are joined four times as often
  constexpr int kRowV = G == 2 ? 4 : 0;  // the values' first row among a position's quantities
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, qd = lane & 3;
  const int col0 = blockIdx.y * R;
  const Columns columns{p.group, p.group_mul, p.max_new};

  uint8_t* ring = g_kv4_smem + warp * (kStages * kBlk);
  float* mrg_o = reinterpret_cast<float*>(g_kv4_smem + L::kRing);
  float* mrg_ml = reinterpret_cast<float*>(g_kv4_smem + L::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(g_kv4_smem + L::kBars) + warp * kStages;
  // a run's segment: tiles [ta, tb) of a pair; tb = 0 behind the last one
  struct Segment {
    SeqSpan sp;
    int b, kvh, ta, tb;
  };
  __shared__ Segment sh_seg[3];  // segment i in place i % 3
  __shared__ uint32_t sh_walk_t, sh_walk_t0;  // the place in the list behind the last segment found
  __shared__ int sh_walk_b;
  __shared__ int sh_scan[kWarps];
  __shared__ int sh_abort;

  if (tid == 0) sh_abort = 0;
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  pdl_launch_dependents();
  pdl_wait();  // q and the cache append come from the previous kernels

  const Kv4Seq& s = p.seq;
  // a negative prefix, positions outside the table, more tokens than the launch covers
  auto check_sequence = [&](const SeqSpan& sp) {
    if (sp.count > 0 &&
        (sp.pre < 0 || static_cast<int64_t>(sp.pre) + sp.count > (static_cast<int64_t>(s.max_pages) << s.page_shift) ||
         sp.count > p.max_new))
      report_device_error(p.status, FITQ_ERR_ARG);
  };
  uint32_t total = 0, per = 0, t_lo = 0, t_hi = 0;
  Kv4Cut* cut = p.cuts + blockIdx.y * gridDim.x + blockIdx.x;  // the pair that this run opens and does not finish
  // ---- the run's segments, found one ahead of their use
  auto advance = [&](Segment& g) {
    uint32_t t = sh_walk_t, t0 = sh_walk_t0;
    int b = sh_walk_b;
    g.tb = 0;
    if (t < t_hi) {
      SeqSpan sp = seq_span(s, b, columns, col0, R, kTile);
      while (t < t_hi && g.tb == 0) {
        int cost = pair_cost(sp);
        while (t >= t0 + static_cast<uint32_t>(cost) * s.kv_heads) {  // next sequence with work
          t0 += static_cast<uint32_t>(cost) * s.kv_heads;
          sp = seq_span(s, ++b, columns, col0, R, kTile);
          cost = pair_cost(sp);
        }
        g.kvh = static_cast<int>((t - t0) / static_cast<uint32_t>(cost));
        const uint32_t pair_t0 = t0 + static_cast<uint32_t>(g.kvh) * cost;
        const int xa = static_cast<int>(t - pair_t0);
        const int xb = pair_t0 + cost < t_hi ? cost : static_cast<int>(t_hi - pair_t0);
        t = pair_t0 + xb;
        g.ta = xa > kPairCost ? xa - kPairCost : 0;
        g.tb = xb > kPairCost ? xb - kPairCost : 0;
        if (g.tb <= g.ta) g.tb = 0;  // the pair's first cost only, its tiles are the next run's
      }
      g.b = b;
      g.sp = sp;
    }
    sh_walk_t = t;
    sh_walk_t0 = t0;
    sh_walk_b = b;
  };

  if (!kClustered) {
    // ---- the list of pairs in units of cost: every thread sums a run of sequences, then a scan
    const int per_thread = (s.batch + kThreads - 1) / kThreads;
    const int b_lo = tid * per_thread, b_hi = b_lo + per_thread < s.batch ? b_lo + per_thread : s.batch;
    int mine = 0;
    for (int b = b_lo; b < b_hi; ++b) mine += pair_cost(seq_span(s, b, columns, col0, R, kTile));
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sh_scan[warp] = incl;
    __syncthreads();
    int before = incl - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int v = sh_scan[w];
      before += w < warp ? v : 0;
      all += v;
    }
    // (the host has checked that the list's length fits in 31 bits)
    total = static_cast<uint32_t>(all) * s.kv_heads;
    per = (total + gridDim.x - 1) / gridDim.x;  // cost of a run
    t_lo = per * blockIdx.x;
    t_hi = t_lo + per < total ? t_lo + per : total;
    if (tid == 0) cut->count = 0;
    {
      int at = before, found = -1, found_at = 0;
      for (int b = b_lo; b < b_hi; ++b) {
        const SeqSpan sp = seq_span(s, b, columns, col0, R, kTile);
        const int cost = pair_cost(sp);
        // sequence b covers [at * KVH, (at + cost) * KVH) of the list
        if (t_lo < t_hi && static_cast<uint32_t>(at) * s.kv_heads <= t_lo &&
            t_lo < static_cast<uint32_t>(at + cost) * s.kv_heads) {
          found = b;
          found_at = at;
        }
        if (blockIdx.x == 0 && blockIdx.y == 0) check_sequence(sp);
        at += cost;
      }
      if (found >= 0) {
        sh_walk_t = t_lo;
        sh_walk_t0 = static_cast<uint32_t>(found_at) * s.kv_heads;
        sh_walk_b = found;
        advance(sh_seg[0]);
      }
    }
    if (t_lo >= t_hi) return;
  }

  if (kClustered && tid == 0) {  // the CTA's share of its cluster's pair, and nothing behind it
    Segment& g = sh_seg[0];
    const int pair = static_cast<int>(blockIdx.x) / kCluster, rank = static_cast<int>(blockIdx.x) % kCluster;
    g.b = pair / s.kv_heads;
    g.kvh = pair % s.kv_heads;
    g.sp = seq_span(s, g.b, columns, col0, R, kTile);
    const int share = (g.sp.tiles + kCluster - 1) / kCluster;
    g.ta = min(rank * share, g.sp.tiles);
    g.tb = min(g.ta + share, g.sp.tiles);
    sh_seg[1].tb = 0;
    if (rank == 0 && g.kvh == 0 && blockIdx.y == 0) check_sequence(g.sp);
  }
  __syncthreads();
  if (kClustered && sh_seg[0].sp.cols == 0) return;  // the whole cluster

  const int64_t slot0 = static_cast<int64_t>(blockIdx.y) * (gridDim.x + static_cast<int64_t>(s.batch) * s.kv_heads);
  uint32_t issued = 0, taken = 0;  // this warp's copies so far

  // ---- this warp's blocks of the segment whose copies are under way: block j lies at
  // position ta * kTile + 16 (warp + kWarps j); lane j % 32 looks its page up and
  // issues its copy.
  const uint8_t* src = nullptr;  // this lane's block of the set of 32 that is being issued
  uint32_t valid = 0;            // which blocks of that set have a page
  auto first_position = [&](const Segment& g) { return g.ta * kTile + kKv4Block * warp; };
  auto block_count = [&](const Segment& g) {
    const int first = first_position(g), end = g.tb * kTile < g.sp.len ? g.tb * kTile : g.sp.len;
    return first < end ? (end - first + kTile - 1) / kTile : 0;
  };
  // the table's entry for block j0 + lane, and the set's blocks once it is there
  auto entry = [&](const Segment& g, int j0) {
    const int64_t pos = first_position(g) + static_cast<int64_t>(j0 + lane) * kTile;
    return j0 + lane < block_count(g) ? s.page_table[static_cast<int64_t>(g.b) * s.max_pages + (pos >> s.page_shift)] : -1;
  };
  auto resolve = [&](const Segment& g, int j0, int pg) -> uint32_t {
    const bool has = pg >= 0 && pg < s.num_pages;
    if (has)
      src = p.pool + kv4_block_offset(s, pg, g.kvh, first_position(g) + static_cast<int64_t>(j0 + lane) * kTile, D);
    else if (j0 + lane < block_count(g))
      report_device_error(p.status, FITQ_ERR_ARG);
    return __ballot_sync(0xffffffffu, has);
  };
  auto issue = [&](uint32_t set, int j) {
    if (!((set >> (j & 31)) & 1u)) return;
    if (lane == (j & 31)) {
      const uint32_t st = issued % kStages;
      mbar_arrive_expect_tx(&bars[st], kBlk);
      bulk_load(ring + st * kBlk, src, kBlk, &bars[st]);
    }
    ++issued;
  };
  // blocks [0, next) of this segment have been issued, and once they are all, [0, ahead) of
  // the one behind it, whose table entries are on their way since this one began
  int next = 0, ahead = 0, ahead_most = 0, ahead_entry = -1;
  uint32_t ahead_valid = 0;
  auto issue_ahead = [&](const Segment& g) {
    if (ahead == 0) ahead_valid = resolve(g, 0, ahead_entry);
    issue(ahead_valid, ahead);
    ++ahead;
  };

  // ---- a segment's queries: set out for shared memory, then into buffer `to`: columns
  // scaled to fp16's range, in the order in which the codes leave their words (element
  // pairs (e, e + 4) of eight), with their group sums
  uint8_t* raw = g_kv4_smem + L::kRaw;
  auto fetch_queries = [&](const Segment& g) {
    for (int i = tid; i < R * (D / 8); i += kThreads) {
      const int n = i / (D / 8), d0 = (i % (D / 8)) * 8;
      const int tok = columns.token(col0 + n), hd = col0 + n - tok * p.group;
      if (n < g.sp.cols)
        cp_async16(raw + i * 16, static_cast<const T*>(p.q) + (g.sp.first + tok) * p.q_stride +
                                     static_cast<int64_t>(g.kvh * p.group + hd) * D + d0);
      else
        *reinterpret_cast<uint4*>(raw + i * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto load_queries = [&](uint8_t* to) {
    uint4* sq = reinterpret_cast<uint4*>(to);
    uint32_t* sqsum = reinterpret_cast<uint32_t*>(to + L::kQsum);
    float* sqexp = reinterpret_cast<float*>(to + L::kQexp);
    // eight elements a thread, from the CTA's upper half on (the lower one joins the warps' parts)
    for (int i = (tid + kThreads / 2) % kThreads; i < R * 8 * G; i += kThreads) {
      const int n = i / (8 * G), gr = (i >> 3) % G, w = (i >> 2) & 1, c = i & 3;
      float f[8], mx = 0.f;
      unpack8<T>(*reinterpret_cast<const uint4*>(raw + (n * D + 64 * gr + 16 * c + 8 * w) * 2), f);
#pragma unroll
      for (int x = 0; x < 8; ++x) mx = fmaxf(mx, fabsf(f[x]));
#pragma unroll
      for (int x = 1; x < 8 * G; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      int e = (__float_as_int(mx) >> 23) - 127;
      e = (mx == 0.f || e > 127) ? 15 : (e < -100 ? -100 : e);
      const float up = pow2(15 - e);
      float even = 0.f, odd = 0.f;
#pragma unroll
      for (int x = 0; x < 8; x += 2) {
        f[x] *= up;
        f[x + 1] *= up * 0.0625f;
        even += f[x];
        odd += f[x + 1];
      }
      // lane 4 (n % 8) + c of the fragment of column tile n / 8
      sq[((gr * 2 + w) * NT + (n >> 3)) * 32 + (n & 7) * 4 + c] =
          make_uint4(pack_half2(f[0], f[4]), pack_half2(f[1], f[5]), pack_half2(f[2], f[6]), pack_half2(f[3], f[7]));
      float sum = fmaf(16.f, odd, even);
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      if ((i & 7) == 0) {
        sum *= pow2(-24);
        const float hi = __half2float(__float2half_rn(sum));
        sqsum[n * G + gr] = pack_half2(hi, sum - hi);
      }
      if (i % (8 * G) == 0) sqexp[n] = p.scale_log2 * pow2(min(e + 9, 127));
    }
  };
  auto queries_arrived = [&] { asm volatile("cp.async.wait_all;" ::: "memory"); };

  fetch_queries(sh_seg[0]);
  valid = resolve(sh_seg[0], 0, entry(sh_seg[0], 0));
  for (const int n = min(kStages, block_count(sh_seg[0])); next < n; ++next) issue(valid, next);
  if (!kClustered && tid == kThreads - 32) advance(sh_seg[1]);
  queries_arrived();
  __syncthreads();
  load_queries(g_kv4_smem + L::kQ);
  int buf = 0;
  // a clustered CTA without tiles of its own still joins the others'
  for (int seg = 0, after = 1; kClustered || sh_seg[seg].tb > 0; seg = after, after = after == 2 ? 0 : after + 1) {
    const Segment& sg = sh_seg[seg];
    const Segment& sn = sh_seg[after];
    const int pos_first = first_position(sg), blocks = block_count(sg), len = sg.sp.len;
    const uint8_t* sq_now = g_kv4_smem + L::kQ + buf * L::kQBytes;
    const uint4* sq = reinterpret_cast<const uint4*>(sq_now);
    const uint32_t* sqsum = reinterpret_cast<const uint32_t*>(sq_now + L::kQsum);
    const float* sqexp = reinterpret_cast<const float*>(sq_now + L::kQexp);
    buf ^= 1;
    __syncthreads();  // the queries are there, the merge buffer and the last segment's place are free
    if (!kClustered) {
      if (tid == kThreads - 32) advance(sh_seg[after == 2 ? 0 : after + 1]);
      ahead = ahead_most = 0;
      if (sn.tb > 0) {
        fetch_queries(sn);
        ahead_most = min(kStages, block_count(sn));
        ahead_entry = entry(sn, 0);
      }
    }
    float cn[NT][2];  // of the columns 2 qd, 2 qd + 1: exponent per score
    int lim[NT][2];   // and the last position they see
    uint32_t qb[NT];  // the group sums as the operand that the keys' lows meet: (0, value or rest)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = 8 * nt + 2 * qd + e;
        cn[nt][e] = sqexp[n];
        const int l = sg.sp.pre + columns.token(col0 + n);
        lim[nt][e] = l < len ? l : len - 1;
      }
      const uint32_t v = sqsum[(8 * nt + g) * G + (qd & (G - 1))];
      qb[nt] = qd < G ? v << 16 : (qd < 2 * G ? v & 0xffff0000u : 0u);
    }
    const int mask_from = sg.sp.pre + columns.token(col0) + 1;  // positions every column sees lie before it

    // m_run in log2 units; o of the codes, off of the eights taken from them (rows 0-7: group
    // 0, 8-15: group 1); sums: the weights' products with the parameters (rows 0-7) and with
    // one (rows 8-15)
    float m_run[NT][2], o[NT][G][4][4], off[NT][4], sums[NT][4];
    // no scale met so far exceeds cap (kGaveUp: below every scale); weights stay below 2^room
    float cap = 1.f, room = kRoom;
    auto clear = [&] {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sums[nt][e] = off[nt][e] = 0.f;
#pragma unroll
          for (int gr = 0; gr < G; ++gr)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][gr][i][e] = 0.f;
        }
    };
    clear();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) m_run[nt][e] = kFloor;

    uint32_t set_valid = 0;
    auto feed = [&] {  // a place in the ring is free
      if (next < blocks) {
        if ((next & 31) == 0) valid = resolve(sg, next, entry(sg, next));
        issue(valid, next);
        ++next;
      } else if (ahead < ahead_most) {
        issue_ahead(sn);
      }
    };
    // N blocks from j on; edge: some of their positions are hidden from some columns.  False
    // once a wait ran out.
    auto step = [&](int j, auto n_tag, auto edge_tag) -> bool {
      constexpr int N = decltype(n_tag)::value;
      constexpr bool edge = decltype(edge_tag)::value;
      const uint8_t* blk[N];
      // A wait that runs out is one lane's finding.  The others need it up to the vote below,
      // which its cap takes to the rare branch; what it reads until then is the ring's, and
      // thrown away.  (A vote of its own behind each wait: 77.8 -> 79.6 us for 64 sequences;
      // a loop of waits per block instead of one try for both first: 78.8.)
      bool here = true;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint32_t st = (taken + u) % kStages;
        here &= mbar_try_wait(&bars[st], ((taken + u) / kStages) & 1u);
        blk[u] = ring + st * kBlk;
      }
      if (!here) {
#pragma unroll 1
        for (int u = 0; u < N; ++u)
          if (!mbar_wait(&bars[(taken + u) % kStages], ((taken + u) / kStages) & 1u, &sh_abort, p.status)) cap = kGaveUp;
      }
      const int pos0 = pos_first + j * kTile;  // of the first block; an edge is one block

      // ---- keys' parameters of positions g and g + 8, and S^T = K.Q^T: one accumulator set
      // per group and one of the lows
      uint32_t kp[N][2][G];
      float acc[N][NT][G][4], accl[N][NT][4];
      uint32_t kw[N][2][2 * G];
#pragma unroll
      for (int u = 0; u < N; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* at = blk[u] + 16 * D + (g + 8 * h) * 8 * G;  // [position][K, V][group](scale, low)
          load_words(kp[u][h], at);
          if (G == 2)
            *reinterpret_cast<uint4*>(kw[u][h]) = *reinterpret_cast<const uint4*>(blk[u] + h * 512 + lane * 16);
          else
            *reinterpret_cast<uint2*>(kw[u][h]) = *reinterpret_cast<const uint2*>(blk[u] + h * 256 + lane * 8);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_f16_k8(accl[u][nt], qd & (G - 1) ? kp[u][0][G - 1] : kp[u][0][0],
                     qd & (G - 1) ? kp[u][1][G - 1] : kp[u][1][0], qb[nt]);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          uint4 bq[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) bq[nt] = sq[((gr * 2 + w) * NT + nt) * 32 + lane];
#pragma unroll
          for (int u = 0; u < N; ++u) {
            uint32_t x = kw[u][0][2 * gr + w], y = kw[u][1][2 * gr + w];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a0 = tiny_even(x), a1 = tiny_even(y), a2 = tiny_odd(x), a3 = tiny_odd(y);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                if (w == 0 && h == 0)
                  mma_f16_first(acc[u][nt][gr], a0, a1, a2, a3, bq[nt].x, bq[nt].y);
                else
                  mma_f16(acc[u][nt][gr], a0, a1, a2, a3, h ? bq[nt].z : bq[nt].x, h ? bq[nt].w : bq[nt].y);
              }
              x >>= 8;
              y >>= 8;
            }
          }
        }

      // ---- values' parameters: all eight quantities of a position as rows of an operand,
      // and the scales, of positions g, g + 8 (kOnce) or side by side of 2 qd, 2 qd + 1 and 8
      // behind them
      uint32_t vs[N][2][G], va[N][2];
      float vf[N][2][G];
      bool over = false;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* par = blk[u] + 16 * D;
        __half2 vmax = __float2half2_rn(0.f);
        if (G == 2) ldmatrix2_t(va[u][0], va[u][1], par + (lane & 15) * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[G], b[G];
          const uint8_t* at = par + (2 * qd + 8 * h) * 8 * G + 4 * G;
          if (G == 1 || !kOnce) {
            load_words(a, at);
            load_words(b, at + 8 * G);
          }
          if (G == 1) va[u][h] = __byte_perm(a[0], b[0], g & 1 ? 0x7632 : 0x5410);
          if (kOnce) load_words(a, par + (g + 8 * h) * 8 * G + 4 * G);
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            // whatever lies behind the last position must not matter
            if (kOnce) {
              vf[u][h][gr] = __low2float(as_half2(a[gr]));
              if (edge && pos0 + g + 8 * h >= len) vf[u][h][gr] = 0.f;
              over |= !(fabsf(vf[u][h][gr]) <= cap);
            } else {
              vs[u][h][gr] = __byte_perm(a[gr], b[gr], 0x5410);
              const int left = len - pos0 - 2 * qd - 8 * h;
              if (edge) vs[u][h][gr] &= left > 1 ? 0xffffffffu : (left > 0 ? 0xffffu : 0u);
              vmax = __hmax2_nan(vmax, __habs2(as_half2(vs[u][h][gr])));
            }
          }
        }
        if (!kOnce) over |= !(__half2float(__hmax_nan(__low2half(vmax), __high2half(vmax))) <= cap);
      }

      // ---- scores in log2 units less the reference (position g: columns 2 qd, 2 qd + 1;
      // position g + 8: the same)
      float sc[N][NT][4], x[N][NT][4];
      float largest = -INFINITY;
#pragma unroll
      for (int u = 0; u < N; ++u) {
        float ks[2][G];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int gr = 0; gr < G; ++gr) ks[h][gr] = __low2float(as_half2(kp[u][h][gr]));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int h = e >> 1;
            float v = fmaf(ks[h][0], acc[u][nt][0][e], accl[u][nt][e]);
            if (G == 2) v = fmaf(ks[h][G - 1], acc[u][nt][G - 1][e], v);
            sc[u][nt][e] = v;
            x[u][nt][e] = fmaf(v, cn[nt][e & 1], -m_run[nt][e & 1]);
            if (edge && pos0 + g + 8 * h > lim[nt][e & 1]) sc[u][nt][e] = x[u][nt][e] = -INFINITY;
            largest = fmaxf(largest, x[u][nt][e]);
          }
      }
      over |= largest > room;
      if (__any_sync(0xffffffffu, over)) {
        if (__any_sync(0xffffffffu, cap == kGaveUp)) return false;  // the warp as one
        // the largest finite scale of the blocks; the others reach their group's elements
        // through the sums, and as zeros nothing else
        float vm = 0.f;
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              float2 v = kOnce ? make_float2(vf[u][h][gr], 0.f) : Half16<__half>::unpack(vs[u][h][gr]);
              v.x = fabsf(v.x) <= 65504.f ? v.x : 0.f;
              v.y = fabsf(v.y) <= 65504.f ? v.y : 0.f;
              if (kOnce)
                vf[u][h][gr] = v.x;
              else
                vs[u][h][gr] = pack_half2(v.x, v.y);
              vm = fmaxf(vm, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
#pragma unroll
        for (int y = kOnce ? 4 : 1; y < (kOnce ? 32 : 4); y <<= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, y));
        if (vm > cap) {
          const int e = (__float_as_int(vm) >> 23) - 126;  // vm < 2^e
          cap = pow2(e);
          room = kRoom - static_cast<float>(e);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(sc[0][nt][e], sc[0][nt][2 + e]);
            if (N == 2) mx = fmaxf(mx, fmaxf(sc[N - 1][nt][e], sc[N - 1][nt][2 + e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mx = fmaxf(fmaf(mx, cn[nt][e], kSlack - room), m_run[nt][e]);
            const float al = exp2_approx(m_run[nt][e] - mx);
            m_run[nt][e] = mx;
#pragma unroll
            for (int u = 0; u < N; ++u) {
              x[u][nt][e] = fmaf(sc[u][nt][e], cn[nt][e], -mx);
              x[u][nt][2 + e] = fmaf(sc[u][nt][2 + e], cn[nt][e], -mx);
            }
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              sums[nt][h + e] *= al;
              off[nt][h + e] *= al;
#pragma unroll
              for (int gr = 0; gr < G; ++gr)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][gr][i][h + e] *= al;
            }
          }
      }

      // ---- weights as an n8 operand, their products with the scales as those of O^T
      uint32_t pb[N][NT][G][2];
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = exp2_approx(x[u][nt][e]);
          const uint32_t p0 = pack_half2(w[0], w[1]), p1 = pack_half2(w[2], w[3]);
          const uint32_t w0 = movmatrix_t(p0), w1 = movmatrix_t(p1);
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            if (kOnce) {
              pb[u][nt][gr][0] = movmatrix_t(pack_half2(w[0] * vf[u][0][gr], w[1] * vf[u][0][gr]));
              pb[u][nt][gr][1] = movmatrix_t(pack_half2(w[2] * vf[u][1][gr], w[3] * vf[u][1][gr]));
            } else {
              pb[u][nt][gr][0] = mul_half2(w0, vs[u][0][gr]);
              pb[u][nt][gr][1] = mul_half2(w1, vs[u][1][gr]);
            }
          }
          if (!edge) {
            mma_f16(sums[nt], va[u][0], 0x3c003c00u, va[u][1], 0x3c003c00u, w0, w1);
          } else {  // whatever a hidden value holds must not matter: visible ones one by one
            const int la = __shfl_sync(0xffffffffu, lim[nt][0], g >> 1), lb = __shfl_sync(0xffffffffu, lim[nt][1], g >> 1);
            const int last = (g & 1 ? lb : la) - pos0 - 2 * qd;  // column g's, from position 2 qd
            const uint32_t keep0 = (last >= 0 ? 0xffffu : 0u) | (last >= 1 ? 0xffff0000u : 0u),
                           keep1 = (last >= 8 ? 0xffffu : 0u) | (last >= 9 ? 0xffff0000u : 0u);
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              pb[u][nt][gr][0] &= keep0;
              pb[u][nt][gr][1] &= keep1;
            }
            const float2 r[2] = {Half16<__half>::unpack(p0), Half16<__half>::unpack(p1)};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float l = 0.f, c[G];
#pragma unroll
              for (int gr = 0; gr < G; ++gr) c[gr] = 0.f;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float we = e ? r[h].y : r[h].x;
                if (pos0 + g + 8 * h > lim[nt][e]) continue;
                l += we;
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                  const float2 v = Half16<__half>::unpack(
                      *reinterpret_cast<const uint32_t*>(blk[u] + 16 * D + (g + 8 * h) * 8 * G + 4 * G + 4 * gr));
                  c[gr] = fmaf(we, fmaf(8.f, v.x, v.y), c[gr]);
                }
              }
#pragma unroll
              for (int y = 4; y < 32; y <<= 1) {
                l += __shfl_xor_sync(0xffffffffu, l, y);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) c[gr] += __shfl_xor_sync(0xffffffffu, c[gr], y);
              }
              sums[nt][2 + e] += l;
#pragma unroll
              for (int gr = 0; gr < G; ++gr)
                if (g == kRowV + 2 * gr + 1) sums[nt][e] += c[gr];
            }
          }
          mma_f16(off[nt], 0x00080008u, 0u, 0x00080008u, 0u, pb[u][nt][0][0], pb[u][nt][0][1]);
          if (G == 2) mma_f16(off[nt], 0u, 0x00080008u, 0u, 0x00080008u, pb[u][nt][G - 1][0], pb[u][nt][G - 1][1]);
        }

      // ---- O^T += V^T.P^T: rows g, g + 8 of m-tile i are elements 2 i, 2 i + 1 of eight
#pragma unroll
      for (int u = 0; u < N; ++u) {
        uint32_t vw[2][2][G];  // half h, position parity, group
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (G == 2)
            *reinterpret_cast<uint4*>(vw[h]) = *reinterpret_cast<const uint4*>(blk[u] + 8 * D + h * 512 + lane * 16);
          else
            *reinterpret_cast<uint2*>(vw[h]) = *reinterpret_cast<const uint2*>(blk[u] + 8 * D + h * 256 + lane * 8);
        if (u == N - 1) {
          __syncwarp();  // every lane has read the blocks
          taken += N;
#pragma unroll
          for (int i = 0; i < N; ++i) feed();
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            uint32_t a = __byte_perm(vw[0][0][gr], vw[0][1][gr], z ? 0x7632 : 0x5410);
            uint32_t b = __byte_perm(vw[1][0][gr], vw[1][1][gr], z ? 0x7632 : 0x5410);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a0 = tiny_even(a), a1 = tiny_odd(a), a2 = tiny_even(b), a3 = tiny_odd(b);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16(o[nt][gr][2 * z + i], a0, a1, a2, a3, pb[u][nt][gr][0], pb[u][nt][gr][1]);
              a >>= 8;
              b >>= 8;
            }
          }
      }
      return true;
    };
    // ---- what the registers hold joins the warp's part in shared memory: the sums of codes less
    // eight, back at their size, and of w (low + 8 scale)
    auto flush = [&](bool first) {
      __syncwarp();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int n = 8 * nt + 2 * qd + e;
          float* ml = mrg_ml + (warp * R + n) * 2;
          float2 was = make_float2(0.f, 0.f);
          if (!first) {
            was = *reinterpret_cast<const float2*>(ml);
            was.x = exp2_approx(was.x - m_run[nt][e]);
          }
          float* row = mrg_o + (warp * R + n) * kLd;
#pragma unroll
          for (int gr = 0; gr < G; ++gr) {
            const int from = 4 * (kRowV + 2 * gr) + qd;
            const float c = fmaf(8.f, __shfl_sync(0xffffffffu, sums[nt][e], from),
                                 __shfl_sync(0xffffffffu, sums[nt][e], from + 4));
            float f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              f[2 * i] = fmaf(o[nt][gr][i][e] - off[nt][2 * gr + e], 16777216.f, c);
              f[2 * i + 1] = fmaf(fmaf(o[nt][gr][i][2 + e], 0.0625f, -off[nt][2 * gr + e]), 16777216.f, c);
            }
            float* dst = row + 64 * gr + 8 * g;
            if (!first) {
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = fmaf(was.x, dst[i], f[i]);
            }
            *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
          }
          __syncwarp();
          if (g == 0) *reinterpret_cast<float2*>(ml) = make_float2(m_run[nt][e], fmaf(was.x, was.y, sums[nt][2 + e]));
        }
    };
    // the blocks that every column sees to their end come first
    int inner = (mask_from - pos_first - kKv4Block) / kTile + 1;
    if (mask_from - pos_first < kKv4Block) inner = 0;
    if (inner > blocks) inner = blocks;
    bool fine = true;
    const int window = kOnce && len > kLong ? 8 : 32;
    for (int j = 0; j < blocks && fine;) {
      if ((j & 31) == 0) set_valid = valid;  // block j has been issued, its set is the current one
      const int stop = min((j | (window - 1)) + 1, blocks);  // (a pair may end one behind it)
      while (j < stop && fine) {
        const uint32_t has = set_valid >> (j & 31);
        if (j + 2 <= inner && (has & 3u) == 3u) {
          fine = step(j, std::integral_constant<int, 2>{}, std::false_type{});
          j += 2;
          continue;
        }
        if (!(has & 1u))  // no page: the block is hidden from every column
          feed();
        else
          fine = step(j, std::integral_constant<int, 1>{}, std::true_type{});
        ++j;
      }
      if (j < blocks) {
        flush(stop == window);
        clear();
      }
    }

    // ---- the rest of the next segment's first copies
    if (!kClustered) {
      while (fine && ahead < ahead_most) issue_ahead(sn);
      next = ahead;
      valid = ahead_valid;
      queries_arrived();
    }

    // ---- the warps' results meet in shared memory
    flush(blocks <= window);
    __syncthreads();
    if (!kClustered && sn.tb > 0) load_queries(g_kv4_smem + L::kQ + buf * L::kQBytes);
    const SeqSpan sp = sg.sp;
    const int b = sg.b, kvh = sg.kvh;
    const bool whole = sg.ta == 0 && sg.tb == sp.tiles;
    const int64_t slot = slot0 + blockIdx.x + static_cast<int64_t>(b) * s.kv_heads + kvh;
    if (!kClustered && tid == 0 && sg.ta == 0 && !whole) {
      // this run opens the pair; the last of its other tiles lies `rest` of cost behind the run's end
      const uint32_t rest = sp.tiles - sg.tb - 1;
      *cut = Kv4Cut{sp.first, static_cast<int>(2 + rest / per), sp.cols, static_cast<int>(slot), kvh};
    }
    for (int i = tid; i < sp.cols * (D / 8); i += kThreads) {
      const int n = i / (D / 8), d0 = (i % (D / 8)) * 8;
      float mx = kFloor;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, mrg_ml[(w * R + n) * 2]);
      float l = 0.f, f[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) f[x] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = *reinterpret_cast<const float2*>(mrg_ml + (w * R + n) * 2);
        if (ml.y == 0.f) continue;  // this warp saw no position of the column
        const float k = exp2_approx(ml.x - mx);
        l += k * ml.y;
        const float* row = mrg_o + (w * R + n) * kLd + d0;
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = fmaf(k, row[x], f[x]);
      }
      if (kClustered) {  // where the ring was: its copies have all been consumed
        float* dst = reinterpret_cast<float*>(g_kv4_smem) + n * D + d0;
        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        if (d0 == 0) *reinterpret_cast<float4*>(reinterpret_cast<float*>(g_kv4_smem) + R * D + n * 4) =
            make_float4(mx, l, 0.f, 0.f);
      } else if (whole) {
        const float inv = 1.f / l;
#pragma unroll
        for (int x = 0; x < 8; ++x) f[x] = l == 0.f ? 0.f : f[x] * inv;
        const int tok = columns.token(col0 + n), hd = col0 + n - tok * p.group;
        T* dst = static_cast<T*>(p.out) + ((sp.first + tok) * p.heads + kvh * p.group + hd) * D + d0;
        *reinterpret_cast<uint4*>(dst) = pack8<T>(f);
      } else {
        float* dst = p.o_part + (slot * R + n) * D + d0;
        *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
        if (d0 == 0) *reinterpret_cast<float2*>(p.ml_part + (slot * R + n) * 2) = make_float2(mx, l);
      }
    }
    if (kClustered) {
      cluster_barrier();
      // every CTA writes its share of the columns' elements
      const float* own_o = reinterpret_cast<const float*>(g_kv4_smem);
      const int rank = static_cast<int>(cluster_rank());
      for (int i = tid * kCluster + rank; i < sp.cols * (D / 4); i += kThreads * kCluster) {
        const int n = i / (D / 4), d0 = (i % (D / 4)) * 4;
        float4 ml[kCluster], v[kCluster];
        float mx = kFloor;
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
          ml[c] = peer_float4(own_o + R * D + n * 4, c);
          v[c] = peer_float4(own_o + n * D + d0, c);
        }
#pragma unroll
        for (int c = 0; c < kCluster; ++c) mx = fmaxf(mx, ml[c].x);
        float l = 0.f;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kCluster; ++c) {
          if (ml[c].y == 0.f) continue;
          const float k = exp2_approx(ml[c].x - mx);
          l += k * ml[c].y;
          f.x = fmaf(k, v[c].x, f.x);
          f.y = fmaf(k, v[c].y, f.y);
          f.z = fmaf(k, v[c].z, f.z);
          f.w = fmaf(k, v[c].w, f.w);
        }
        const float inv = 1.f / l;
        const int tok = columns.token(col0 + n), hd = col0 + n - tok * p.group;
        T* dst = static_cast<T*>(p.out) + ((sp.first + tok) * p.heads + kvh * p.group + hd) * D + d0;
        *reinterpret_cast<uint2*>(dst) =
            l == 0.f ? make_uint2(0u, 0u)
                     : make_uint2(Half16<T>::pack(f.x * inv, f.y * inv), Half16<T>::pack(f.z * inv, f.w * inv));
      }
      cluster_barrier();  // the parts stay until every CTA has read them
      break;
    }
    if (sh_abort) break;
  }
  if (sh_abort) {  // a wait ran out: the copies still in flight land before the CTA leaves
    int none = 0;
    for (; taken != issued; ++taken)
      mbar_wait_for(&bars[taken % kStages], (taken / kStages) & 1u, &none, p.status, kWaitLimitNs);
  }
}

// Joins the runs that a pair was cut into, in a fixed order.  Grid (runs, columns,
// row tiles): the CTA of the run that opens a pair joins one column of it; four
// warps take every fourth run each.
constexpr int kCWarps = 4;
constexpr int kCMaxRuns = 1024;  // more runs than a launch has

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * kCWarps) kv4_attn_combine_kernel(const Kv4AttnParams p) {
  constexpr int R = 8 * NT;
  constexpr int kE = D / 32;  // elements per lane
  __shared__ float sh_o[kCWarps][D];
  __shared__ float sh_ml[kCWarps][2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int run = blockIdx.x, n = blockIdx.y, runs = gridDim.x;
  pdl_launch_dependents();
  pdl_wait();  // the partials
  const Kv4Cut cut = p.cuts[blockIdx.z * runs + run];
  if (n >= cut.cols || cut.count == 0) return;
  const int col0 = blockIdx.z * R;
  const Columns columns{p.group, p.group_mul, p.max_new};
  const int64_t slot0 = cut.slot;
  const float2* ml = reinterpret_cast<const float2*>(p.ml_part) + slot0 * R + n;
  const float* row = p.o_part + (slot0 * R + n) * D + lane * kE;
  float mx = kFloor, l = 0.f, f[kE];
#pragma unroll
  for (int x = 0; x < kE; ++x) f[x] = 0.f;
#pragma unroll 4
  for (int c = warp; c < cut.count; c += kCWarps) {
    const float2 w = ml[static_cast<int64_t>(c) * R];
    float v[kE];
    if (kE == 4)
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(row + static_cast<int64_t>(c) * R * D);
    else
      *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(row + static_cast<int64_t>(c) * R * D);
    if (w.y == 0.f) continue;  // that run saw no position of the column
    const float m = fmaxf(mx, w.x), k0 = exp2_approx(mx - m), k1 = exp2_approx(w.x - m);
    mx = m;
    l = k0 * l + k1 * w.y;
#pragma unroll
    for (int x = 0; x < kE; ++x) f[x] = k0 * f[x] + k1 * v[x];
  }
#pragma unroll
  for (int x = 0; x < kE; ++x) sh_o[warp][lane * kE + x] = f[x];
  if (lane == 0) {
    sh_ml[warp][0] = mx;
    sh_ml[warp][1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  mx = kFloor;
#pragma unroll
  for (int w = 0; w < kCWarps; ++w) mx = fmaxf(mx, sh_ml[w][0]);
  float a = 0.f, b2 = 0.f;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kCWarps; ++w) {
    if (sh_ml[w][1] == 0.f) continue;
    const float k = exp2_approx(sh_ml[w][0] - mx);
    l += k * sh_ml[w][1];
    a = fmaf(k, sh_o[w][2 * threadIdx.x], a);
    b2 = fmaf(k, sh_o[w][2 * threadIdx.x + 1], b2);
  }
  const float inv = 1.f / l;
  const int tok = columns.token(col0 + n), hd = col0 + n - tok * p.group;
  T* dst = static_cast<T*>(p.out) + ((cut.first + tok) * p.heads + cut.kvh * p.group + hd) * D + 2 * threadIdx.x;
  *reinterpret_cast<uint32_t*>(dst) = l == 0.f ? 0u : Half16<T>::pack(a * inv, b2 * inv);
}

// Whether a call goes as clusters: all of them on the card at once, and no CTA with more
// than eight tiles.
template <int NT>
bool clusters_fit(int64_t pairs, int64_t cols, int64_t max_len, int num_sms) {
  const int64_t row_tiles = (cols + 8 * NT - 1) / (8 * NT);
  return pairs * kCluster * row_tiles <= static_cast<int64_t>(num_sms) * AttnShape<NT>::kCtas &&
         max_len <= 8ll * kCluster * AttnShape<NT>::kTile;
}

// Columns per warp, in n8 tiles.  Up to eight: one.  More: two, so that a block is decoded
// once for sixteen columns, unless all row tiles of eight fit on the card as clusters, which
// then end sooner: 5 tokens of 5 heads over 1,000 / 4,000 positions of one sequence take 8.1 /
// 10.6 us in four row tiles, 10.0 / 13.0 us in two; of two sequences, whose four no longer
// fit, 11.7 / 17.1 against 10.8 / 13.9 us.
int col_tiles(int64_t pairs, int64_t cols, int64_t max_len, int num_sms) {
  return cols <= 8 || clusters_fit<1>(pairs, cols, max_len, num_sms) ? 1 : 2;
}

struct AttnPlan {
  int nt, row_tiles, cols, runs;  // cols: columns of the fullest row tile; runs = 0: clusters
  size_t cuts_off, ml_off, o_off, bytes;
};

template <int NT>
int64_t plan_runs(int64_t pairs, int64_t max_len, int row_tiles, int num_sms) {
  const int64_t tiles = pairs * ((max_len + AttnShape<NT>::kTile - 1) / AttnShape<NT>::kTile);
  int64_t runs = static_cast<int64_t>(num_sms) * AttnShape<NT>::kCtas;
  if (row_tiles > 1) runs = (runs + row_tiles - 1) / row_tiles;
  if (runs > tiles) runs = tiles;
  if (runs > kCMaxRuns) runs = kCMaxRuns;
  return runs < 1 ? 1 : runs;
}

AttnPlan attn_plan(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim, int num_sms) {
  AttnPlan a;
  const int64_t pairs = static_cast<int64_t>(batch) * kv_heads, cols = static_cast<int64_t>(group) * max_new;
  a.nt = col_tiles(pairs, cols, max_len, num_sms);
  const int R = 8 * a.nt;
  a.row_tiles = static_cast<int>((cols + R - 1) / R);
  a.cols = static_cast<int>(cols < R ? cols : R);
  a.runs = static_cast<int>(a.nt == 1 ? plan_runs<1>(pairs, max_len, a.row_tiles, num_sms)
                                     : plan_runs<2>(pairs, max_len, a.row_tiles, num_sms));
  if (a.nt == 1 ? clusters_fit<1>(pairs, cols, max_len, num_sms) : clusters_fit<2>(pairs, cols, max_len, num_sms)) {
    a.runs = 0;
    a.cuts_off = a.ml_off = a.o_off = 0;
    a.bytes = 16;
    return a;
  }
  const size_t slots = static_cast<size_t>(a.row_tiles) * (a.runs + pairs);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  a.cuts_off = 0;
  a.ml_off = up(static_cast<size_t>(a.row_tiles) * a.runs * sizeof(Kv4Cut));
  a.o_off = a.ml_off + up(slots * R * 2 * sizeof(float));
  a.bytes = a.o_off + slots * R * dim * sizeof(float);
  return a;
}

template <typename T, int D, int NT>
int attn_t(const Kv4AttnParams& p, const AttnPlan& a, cudaStream_t st) {
  constexpr int smem = AttnSmem<D, NT>::kBytes;
  if (a.runs == 0) {
    auto* kernel = kv4_attn_kernel<T, D, NT, true>;
    if (!set_smem_limit(kernel, smem)) return FITQ_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.seq.batch * p.seq.kv_heads * kCluster, a.row_tiles);
    cfg.blockDim = dim3(AttnShape<NT>::kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
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
  auto* kernel = kv4_attn_kernel<T, D, NT, false>;
  if (!set_smem_limit(kernel, smem)) return FITQ_ERR_CUDA;
  cudaError_t e = launch_pdl(kernel, dim3(a.runs, a.row_tiles), dim3(AttnShape<NT>::kThreads), smem, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  e = launch_pdl(kv4_attn_combine_kernel<T, D, NT>, dim3(a.runs, a.cols, a.row_tiles), dim3(32 * kCWarps), 0, st, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  return launch_result();
}

template <typename T, int D>
int attn_td(const Kv4AttnParams& p, const AttnPlan& a, cudaStream_t st) {
  return a.nt == 1 ? attn_t<T, D, 1>(p, a, st) : attn_t<T, D, 2>(p, a, st);
}

// From 65 rows on the tensor-memory kernel takes the call.  45 rows of one sequence over
// 1,000 / 8,000 positions, of eight over 1,000 / 8,000: 10.7 / 20.8 / 27.7 / 79.8 us here,
// 18.0 / 19.8 / 19.6 / 82.4 us there; 65 rows: 14.6 / 27.0 / 32.0 / 197 and 18.7 / 21.3 /
// 20.2 / 83.3 us.
bool prompt_rows(int group, int64_t max_new) { return group * max_new > 64; }

}  // namespace

size_t kv4_attention_workspace(int batch, int kv_heads, int group, int64_t max_new, int64_t max_len, int dim,
                               int num_sms) {
  if (prompt_rows(group, max_new))
    return kv4_prompt_workspace(batch, kv_heads, group, max_new, max_len, dim, num_sms);
  return attn_plan(batch, kv_heads, group, max_new, max_len, dim, num_sms).bytes;
}

int launch_kv4_attention(const Kv4Seq& seq, const void* q, int64_t q_stride, const void* pool, void* out, int heads,
                         int dim, int dtype, int64_t max_new, int64_t max_len, void* workspace, int* status,
                         cudaStream_t st, int num_sms) {
  const int group = heads / seq.kv_heads;
  if (prompt_rows(group, max_new))
    return launch_kv4_prompt(seq, q, q_stride, pool, out, heads, dim, dtype, max_new, max_len, workspace, status, st,
                             num_sms);
  const AttnPlan a = attn_plan(seq.batch, seq.kv_heads, group, max_new, max_len, dim, num_sms);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Kv4AttnParams p;
  p.q = q;
  p.q_stride = q_stride;
  p.out = out;
  p.pool = static_cast<const uint8_t*>(pool);
  p.cuts = reinterpret_cast<Kv4Cut*>(ws + a.cuts_off);
  p.ml_part = reinterpret_cast<float*>(ws + a.ml_off);
  p.o_part = reinterpret_cast<float*>(ws + a.o_off);
  p.heads = heads;
  p.group = group;
  p.max_new = static_cast<int>(max_new);
  p.group_mul = (65536 + group - 1) / group;
  p.scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(dim));
  p.status = status;
  p.seq = seq;
  if (dtype == FITQ_DTYPE_BF16)
    return dim == 128 ? attn_td<__nv_bfloat16, 128>(p, a, st) : attn_td<__nv_bfloat16, 64>(p, a, st);
  return dim == 128 ? attn_td<__half, 128>(p, a, st) : attn_td<__half, 64>(p, a, st);
}

}  // namespace fitq
