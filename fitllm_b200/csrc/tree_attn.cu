// Attention of a tree of drafted tokens over a 16-bit key/value cache, on tcgen05.
//
// For token i of sequence b and head h on KV head h / group, with s_j = q.k_j / sqrt(D)
// over the cached positions and the ancestors of i (and i):
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   m = max s_j,
// in one pass with a running reference m.  The rows of a (sequence, KV head) pair are its
// tokens x group heads, 128 to a row tile, up to two row tiles at a time, so that keys and
// values are read once for all of them.
//
// Work: the 64-position tiles of all pairs (and pairs of row tiles) form one list, in which
// every CTA, one per SM, owns a run of equal length, found from the lengths on the device:
// short and long sequences share the card evenly and no length is known to the host.  A pair
// whose tiles lie in several runs leaves (O, m, l) of each piece in the workspace and
// tree_attn_combine_kernel joins them in order (deterministic).
//
// Roles: warps 0-3 and 4-7 are two softmax units, a thread per row (TMEM lane); warp 8
// loads K and V tiles by TMA into one ring, warps 9 and 11 issue the units' MMAs (one warp
// for both took 3,340 cycles a tile, 1,240 of waits and issues for each unit, where a unit's
// softmax takes 1,000), warp 10 cleans the values behind the cached positions.  Per step S = Q.K^T
// goes to one of two halves of the unit's columns of tensor memory, the unit writes P = 2^(S c - m)
// over it, and O += P.V takes P from there and V as loaded, position by position (an MN-major
// operand).  P is rounded to the values' type, which the MMA wants of its operands (relative errors
// of 2.1e-3 to 2.3e-3 in bf16 where the result's own rounding gives 1.7e-3; 2.9e-4 and 2.1e-4 in fp16);
// its sum is fp32 of what was not rounded.  As two numbers of that type, which would leave the result's rounding
// alone, P would have a second product: 512 more cycles of MMAs in the 2,000 of a tile for two row tiles.
// With one row tile the units take the tiles in turn, each with sums O, m and l of its own
// that are joined at the pair's end; with two, a unit is a row tile and both see every tile.
//
// m moves only when a weight would exceed 2^15, and then to 2^7 below the row's largest; the
// thread that moves it rescales its row of O once the step before has been added.
//
// Only a tile that reaches behind the cached positions needs a mask: a 64-bit word per row,
// the token's ancestors shifted to the tile.  There 0 x NaN must not reach rows that do
// not see a value, so warp 10 zeroes the rows that no token sees and the elements that are not
// finite; a row that sees such an element adds it at the end by itself.  The TMA of such a tile
// completes on a barrier of warp 10's own, and the slot's is completed by warp 10.
//
// Bound: with one row tile the loads (64 sequences of 8 tokens, 40 heads on 8 of 128, over 100 to 8,191
// positions: 197 us, 5.7 TB/s, at 1,965 MHz; 232 at the 1,627 MHz that a long run of them is left: its
// time follows the clock), and a pair's end, some 3 us that the ring covers in part.  With two the
// chain of a tile: some 2,000 cycles, of which both units' MMAs need 1,280 (48 for one of 32, which waits
// for Q from shared memory) and the exponentials 1,024 (8 sequences of 32 tokens over 3,500 to 4,099: 50 us;
// 64 tokens over 131,071 in fp16: 253 us, 298 at 1,605 MHz).  Few positions: 14 us for 5 tokens over 1,023.
#include <type_traits>

#include "kernels.cuh"
#include "tree.cuh"
#include "umma_warp.cuh"

namespace fitq {
namespace {

constexpr int kRows = 128;      // rows of a row tile (TMEM lanes)
constexpr int kStep = 64;       // positions of a tile
constexpr int kThreads = 384;
constexpr float kFloor = -3.0e38f;
constexpr float kRoom = 15.f;   // weights stay below 2^15
constexpr float kSlack = 8.f;   // a reference that moves leaves this much (log2) to the weights that follow

// Steps of a unit after which O joins its rows' sums in the workspace: an accumulation in
// tensor memory rounds towards zero at the accumulator's size, some 2^-24 of it each time.
template <typename T>
constexpr int window_steps() { return std::is_same<T, __half>::value ? 1 << 8 : 1 << 10; }

template <int D, bool kTwo>
struct TreeSmem {
  static constexpr int kPanel = kStep * 128;            // 64 elements of 64 positions
  static constexpr int kTile = D / 64 * kPanel;
  static constexpr int kQPanel = kRows * 128;
  static constexpr int kQ = D / 64 * kQPanel;           // one row tile's queries
  // A multiple of four: where the units take the tiles in turn a slot then stays with one unit,
  // whose issuer has seen each of its phases complete before it waits for the next (by parity).
  // 8 / 12 of them: 236 / 217 us for 64 sequences of 100 to 8,191.
  static constexpr int kStages = D == 64 ? 24 : kTwo ? 8 : 12;
  static constexpr int kOffRing = (kTwo ? 2 : 1) * kQ;
  static constexpr int kBytes = kOffRing + kStages * kTile + 1024;  // tiles start on a 1,024-byte boundary
  static_assert(kStages % 4 == 0 && kStages <= 32, "phases are kept in a word");
};

struct TreeAttnParams {
  TreeView tree;
  const void* q;
  const void* v_cache;
  void* out;
  int4* desc;      // [CTAs] pair that begins in a CTA's run and ends in a later one: sequence, head x rows, parts
  float2* ml_part; // [CTAs][2: the run's first pair, a later one][rows of a pair]
  float* o_part;   // [..][rows of a pair][D], of two row tiles [..][D][rows of a pair]
  float* o_sum;    // [CTAs][2 units][128][D], kLong only
  int64_t q_stride;
  int heads, group, row_pairs, pair_rows;  // pair_rows: 128 or 256
  float scale_log2;
  int* status;
};

// A CTA's place in the list of tiles.
struct Cursor {
  int b, kr;       // sequence; KV head x row pairs
  int pre;         // cached positions of the sequence as given
  int n;           // tiles of the sequence
  int t0, t1;      // this piece's tiles
  int left;        // tiles of the run from t0 on
};

__device__ __forceinline__ int tiles_of(const TreeView& t, int pre) {
  int64_t len = pre < 0 ? 0 : static_cast<int64_t>(pre) + t.tokens;
  if (len > t.capacity) len = t.capacity;
  const int n = static_cast<int>((len + kStep - 1) / kStep);
  return n < 1 ? 1 : n;
}
// The first tile that reaches behind the cached positions.
__device__ __forceinline__ int tail_of(int pre) { return pre < 0 ? 0 : pre / kStep; }
__device__ __forceinline__ void next_piece(const TreeAttnParams& p, Cursor& c) {
  c.left -= c.t1 - c.t0;
  c.t0 = 0;
  if (++c.kr == p.tree.kv_heads * p.row_pairs) {
    c.kr = 0;
    ++c.b;
    if (c.left > 0) {
      c.pre = p.tree.prefix[c.b];
      c.n = tiles_of(p.tree, c.pre);
    }
  }
  c.t1 = min(c.n, c.left);
}

// The lanes of a warp hold the tree of a sequence: lane i tokens i and i + 32.
struct LaneTree {
  uint64_t seen0, seen1;
  int root0, root1;  // -1 where the token is there, -2 where not
};
__device__ __forceinline__ LaneTree load_tree(const TreeView& t, int b, int pre, int lane, bool report, int* status) {
  LaneTree w;
  bool bad = false;
  w.root0 = lane < t.tokens ? tree_parent(t, b, lane, &bad) : -2;
  w.root1 = lane + 32 < t.tokens ? tree_parent(t, b, lane + 32, &bad) : -2;
  w.seen0 = 1ull << lane;
  w.seen1 = 1ull << (lane + 32);
  // the walk's length doubles: six rounds at most, as parents lie below their children
  while (__any_sync(0xffffffffu, w.root0 >= 0 || w.root1 >= 0)) {
    // a token's entries through its current ancestor
    auto ask = [&](int at, uint64_t& seen, int& root) {
      const int src = at < 0 ? 0 : at;
      const uint64_t s0 = __shfl_sync(0xffffffffu, w.seen0, src & 31), s1 = __shfl_sync(0xffffffffu, w.seen1, src & 31);
      const int r0 = __shfl_sync(0xffffffffu, w.root0, src & 31), r1 = __shfl_sync(0xffffffffu, w.root1, src & 31);
      seen = src < 32 ? s0 : s1;
      root = src < 32 ? r0 : r1;
    };
    uint64_t a_seen, b_seen;
    int a_root, b_root;
    ask(w.root0, a_seen, a_root);
    ask(w.root1, b_seen, b_root);
    if (w.root0 >= 0) {
      w.seen0 |= a_seen;
      w.root0 = a_root;
    }
    if (w.root1 >= 0) {
      w.seen1 |= b_seen;
      w.root1 = b_root;
    }
  }
  // tokens without a slot
  const int64_t room = pre < 0 ? 0 : t.capacity - pre;
  if (w.root0 == -1 && lane >= room) {
    w.root0 = -2;
    bad = true;
  }
  if (w.root1 == -1 && lane + 32 >= room) {
    w.root1 = -2;
    bad = true;
  }
  if (report && bad) report_device_error(status, FITQ_ERR_ARG);
  return w;
}
// Token `tok` (any lane's own) of the tree; every lane of the warp asks.
__device__ __forceinline__ bool tree_token(const LaneTree& w, int tok, uint64_t& seen) {
  const int src = tok & 31;
  const uint64_t s0 = __shfl_sync(0xffffffffu, w.seen0, src), s1 = __shfl_sync(0xffffffffu, w.seen1, src);
  const int r0 = __shfl_sync(0xffffffffu, w.root0, src), r1 = __shfl_sync(0xffffffffu, w.root1, src);
  seen = tok < 32 ? s0 : s1;
  return (tok < 32 ? r0 : r1) == -1;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// MN-major 128-byte-swizzled operand: `lbo` bytes between 64-element atoms, 1,024 between
// groups of eight positions.
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr, uint32_t lbo) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((1024u >> 4) & 0x3FFFu) << 32 | 1ull << 46 | 2ull << 61;
}

template <typename T>
struct Mma16;  // operand type bits of the instruction descriptor; the exponent of what is not finite
template <>
struct Mma16<__nv_bfloat16> {
  static constexpr uint32_t kType = (1u << 7) | (1u << 10), kExp = 0x7f80u;
};
template <>
struct Mma16<__half> {
  static constexpr uint32_t kType = 0, kExp = 0x7c00u;
};

extern __shared__ uint8_t g_tree_smem[];

template <typename T, int D, bool kTwo, bool kLong>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const TreeAttnParams p) {
  using L = TreeSmem<D, kTwo>;
  constexpr int kStages = L::kStages;
  constexpr int kWindow = window_steps<T>();
  __shared__ uint64_t b_full[kStages], b_free[kStages], b_tail[kStages], b_qready, b_sfull[2][2], b_pready[2][2], b_odone[2][2], b_alldone,
      b_segdone, b_fixed, b_done;
  __shared__ uint32_t sh_tmem;
  __shared__ int sh_abort;
  __shared__ Cursor sh_start;
  __shared__ int sh_share;
  __shared__ uint64_t sh_bad[2];  // tokens with elements that are not finite, by piece
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(g_tree_smem) + 1023u) & ~1023u;
  const uint32_t s_q = base, s_ring = base + L::kOffRing;

  pdl_launch_dependents();
  pdl_wait();
  const TreeView& tr = p.tree;
  const int krs = tr.kv_heads * p.row_pairs;
  if (warp == 0) {  // where this CTA's run begins
    int total = 0;
    for (int b0 = 0; b0 < tr.batch; b0 += 32) total += b0 + lane < tr.batch ? tiles_of(tr, tr.prefix[b0 + lane]) : 0;
    total = __reduce_add_sync(0xffffffffu, total) * krs;
    const int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * share;
    Cursor c{0, 0, 0, 1, 0, 0, 0};
    int before = 0;
    for (int b0 = 0; first < total && b0 < tr.batch; b0 += 32) {
      const int pre = b0 + lane < tr.batch ? tr.prefix[b0 + lane] : 0;
      const int n = b0 + lane < tr.batch ? tiles_of(tr, pre) * krs : 0;
      int upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > first);
      if (hit) {
        const int at = __ffs(hit) - 1;
        c.b = b0 + at;
        c.pre = __shfl_sync(0xffffffffu, pre, at);
        c.n = __shfl_sync(0xffffffffu, n, at) / krs;
        const int in = static_cast<int>(first) - before - __shfl_sync(0xffffffffu, upto - n, at);
        c.kr = in / c.n;
        c.t0 = in % c.n;
        c.left = static_cast<int>(total - first < share ? total - first : share);
        c.t1 = c.n - c.t0 < c.left ? c.n : c.t0 + c.left;
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) {
      sh_start = c;
      sh_share = share;
      sh_abort = 0;
    }
  } else if (warp == 1 && lane == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&b_full[i], 1);
      mbar_init(&b_free[i], 2);  // both units', or the one's that takes the tile
      mbar_init(&b_tail[i], 1);
    }
    mbar_init(&b_qready, 8);  // an arrival per softmax warp
    mbar_init(&b_alldone, 8);
    mbar_init(&b_segdone, 8);
    for (int i = 0; i < 2; ++i) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&b_sfull[i][h], 1);
        mbar_init(&b_pready[i][h], 4);
        mbar_init(&b_odone[i][h], 1);
      }
    }
    mbar_init(&b_fixed, 1);
    mbar_init(&b_done, 2);
    fence_mbar_init();
  } else if (warp == 9) {
    tmem_alloc(&sh_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh_tmem;  // S_0, S_1 (128 columns each), O_0, O_1 (D each, 128 apart)
  Cursor c = sh_start;
  const int rows_all = tr.tokens * p.group;

  auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool { return mbar_wait_warp(bar, parity, &sh_abort, p.status); };
  auto arrive_warp = [&](uint64_t* bar) {  // behind every lane's stores and fences
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };
  // rows of a piece, and whether its tiles are dealt to the units in turn
  auto rows_of = [&](int kr) { return min(rows_all - kr % p.row_pairs * p.pair_rows, p.pair_rows); };
  // steps of unit r in a piece of nt tiles
  auto steps_of = [](bool par, int rows, int nt, int r) {
    return par ? (nt + 1 - r) / 2 : r == 0 || rows > kRows ? nt : 0;
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax: a row per thread
    const int r = warp >> 2, lr = tid & 127;
    const uint32_t t_lane = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t t_s = tmem + t_lane + r * 128, t_o = tmem + t_lane + 256;
    struct Row {
      int64_t token;   // of all sequences' tokens
      int hd;
      bool has, here, live;  // live: the warp has a row
      uint64_t seen;
    };
    LaneTree tree;
    int tree_b = -1;
    // The thread's row's queries (both units share a row where one row tile is enough), on their
    // way while the piece before ends: 215 -> 201 us for 64 sequences of 100 to 8,191.  Twice as
    // many registers of them, for two row tiles, spill and cost 6%.
    uint4 queries[D / 16];
    const uint4* source = nullptr;
    auto fetch = [&](const Cursor& c) -> Row {
      Row w;
      const int kvh = c.kr / p.row_pairs, rows = rows_of(c.kr);
      const bool par = rows <= kRows;
      const int in_piece = par ? lr : r * kRows + lr;
      w.has = in_piece < rows;
      w.live = __any_sync(0xffffffffu, w.has);
      const int row = c.kr % p.row_pairs * p.pair_rows + (w.has ? in_piece : 0);
      const int tok = row / p.group;
      w.hd = kvh * p.group + row % p.group;
      w.token = static_cast<int64_t>(c.b) * tr.tokens + tok;
      source = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + w.token * p.q_stride + static_cast<int64_t>(w.hd) * D) +
               (par ? r * (D / 16) : 0);
      if (!kTwo) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) queries[i] = w.has ? source[i] : make_uint4(0, 0, 0, 0);
      }
      return w;
    };
    auto look = [&](const Cursor& c, Row& w) {  // the row's token in the tree
      if (c.b != tree_b) {
        tree = load_tree(tr, c.b, c.pre, lane, warp == 0 && c.kr == 0 && c.t0 == 0, p.status);
        tree_b = c.b;
      }
      const int row = c.kr % p.row_pairs * p.pair_rows + (w.has ? (rows_of(c.kr) <= kRows ? lr : r * kRows + lr) : 0);
      w.here = tree_token(tree, row / p.group, w.seen) && w.has;
    };
    auto put = [&](const Cursor& c, bool has) {  // the queries to shared memory
      const bool par = rows_of(c.kr) <= kRows;
      const uint32_t dst = s_q + (par ? 0 : r * L::kQ) + lr * 128;
      const int i0 = par ? r * (D / 16) : 0;
#pragma unroll 1
      for (int part = 0; part < (kTwo && !par ? 2 : 1); ++part) {
        if (kTwo) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) queries[i] = has ? source[part * (D / 16) + i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int x = i0 + part * (D / 16) + i;
          sts128(dst + (x >> 3) * L::kQPanel + (((x & 7) ^ (lr & 7)) << 4), queries[i].x, queries[i].y, queries[i].z, queries[i].w);
        }
      }
      fence_async_proxy();
      arrive_warp(&b_qready);
    };
    int u = 0;  // steps of this unit before the piece
    int piece = 0;
    bool ok = c.left > 0;
    Row w{};
    if (ok) {
      w = fetch(c);
      // two row tiles load their queries in put: the scores need them first
      if (kTwo) put(c, w.has);
      look(c, w);
      if (!kTwo) put(c, w.has);
    }
    const float cn = p.scale_log2;
    const uint64_t cn2 = pack2(cn, cn);
    while (ok) {
      const int rows = rows_of(c.kr);
      const bool par = rows <= kRows;
      const int steps = steps_of(par, rows, c.t1 - c.t0, r);
      float m = kFloor, l = 0.f, m_kept = kFloor;
      float4* sum_row = reinterpret_cast<float4*>(p.o_sum + ((static_cast<int64_t>(blockIdx.x) * 2 + r) * kRows + lr) * D);
      if (piece > 0) ok = wait_all(&b_segdone, (piece - 1) & 1);  // O has been read by both units
      for (int t = 0; ok && t < steps; ++t) {
        const int h = (u + t) & 1;
        const int pos0 = (c.t0 + (par ? 2 * t + r : t)) * kStep;
        const bool begins = kLong ? t % kWindow == 0 : t == 0;  // O begins anew with this step
        if (kLong && begins && t > 0) {  // O joins the row's sums, whose columns are its own
          ok = wait_all(&b_odone[r][h ^ 1], ((u + t - 1) >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          const float k = exp2_approx(m_kept - m);
#pragma unroll 1
          for (int cc = 0; cc < D / 16; ++cc) {
            uint32_t x[16];
            tmem_ld_x16(t_o + r * 128 + 16 * cc, x);
            tmem_ld_wait();
            if (w.has) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float4 v = t > kWindow ? sum_row[4 * cc + i] : make_float4(0.f, 0.f, 0.f, 0.f);
                v.x = fmaf(k, v.x, __uint_as_float(x[4 * i]));
                v.y = fmaf(k, v.y, __uint_as_float(x[4 * i + 1]));
                v.z = fmaf(k, v.z, __uint_as_float(x[4 * i + 2]));
                v.w = fmaf(k, v.w, __uint_as_float(x[4 * i + 3]));
                sum_row[4 * cc + i] = v;
              }
            }
            __syncwarp();
          }
          m_kept = m;
        }
        ok = wait_all(&b_sfull[r][h], ((u + t) >> 1) & 1);
        if (!ok) break;
        if (w.live) {
          tc_fence_after();
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(t_s + h * kStep, v[0]);
          tmem_ld_32x32b_x32(t_s + h * kStep + 32, v[1]);
          tmem_ld_wait();
          if (pos0 + kStep > c.pre) {  // behind the cached positions: the tree's word, shifted to the tile
            const int shift = c.pre - pos0;
            const uint64_t vis = shift >= 0 ? (shift > 63 ? ~0ull : (w.seen << shift) | ((1ull << shift) - 1))
                                 : shift > -64 ? w.seen >> -shift : 0ull;
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              const uint32_t word = static_cast<uint32_t>(vis >> (32 * cc));
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((word >> i) & 1u)) v[cc][i] = 0xff800000u;
            }
          }
          float top[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) top[x] = -INFINITY;
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int i = 0; i < 32; i += 8)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                top[x] = fmaxf(top[x], fmaxf(__uint_as_float(v[cc][i + 2 * x]), __uint_as_float(v[cc][i + 2 * x + 1])));
          const float raw = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * cn;
          if (__any_sync(0xffffffffu, raw > m + kRoom)) {
            const float m_new = fmaxf(m, raw - (kRoom - kSlack));
            const float al = exp2_approx(m - m_new);
            m = m_new;
            l *= al;
            if (!begins) {
              ok = wait_all(&b_odone[r][h ^ 1], ((u + t - 1) >> 1) & 1);  // the step before has been added
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int cc = 0; cc < D / 16; ++cc) {
                uint32_t x[16];
                tmem_ld_x16(t_o + r * 128 + 16 * cc, x);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * al);
                tmem_st_x16(t_o + r * 128 + 16 * cc, x);
              }
            }
          }
          // ---- weights, written over the scores
          const uint64_t m2 = pack2(-m, -m);
          uint64_t s2[2] = {0, 0};
          uint32_t pk[32];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float x0, x1;
              unpack2(fma2(pack2(__uint_as_float(v[cc][i]), __uint_as_float(v[cc][i + 1])), cn2, m2), x0, x1);
              const float w0 = exp2_approx(x0), w1 = exp2_approx(x1);
              s2[(i >> 1) & 1] = add2(s2[(i >> 1) & 1], pack2(w0, w1));
              pk[16 * cc + i / 2] = Half16<T>::pack(w0, w1);
            }
          tmem_st_x32(t_s + h * kStep, pk);
          float a, c2;
          unpack2(add2(s2[0], s2[1]), a, c2);
          l += a + c2;
          tmem_st_done();
          tc_fence_before();
        }
        arrive_warp(&b_pready[r][h]);
      }
      const Cursor old = c;
      const Row row = w;
      if (!ok) break;
      next_piece(p, c);
      if (c.left > 0) {
        w = fetch(c);
        look(c, w);
      }
      // the last step's products (and those before them), and the cleaned values' notes
      if (ok && steps > 0) ok = wait_all(&b_odone[r][(u + steps - 1) & 1], ((u + steps - 1) >> 1) & 1);
      if (ok) ok = wait_all(&b_fixed, piece & 1);
      if (!ok) break;
      u += steps;
      const float kept = steps > kWindow && kLong ? exp2_approx(m_kept - m) : 0.f;
      // m, l and the factor of the sums meet the other unit's in the unit's columns of scores
      const uint32_t mine[4] = {__float_as_uint(m), __float_as_uint(l), __float_as_uint(kept),
                                kLong && steps > kWindow ? 1u : 0u};
      tmem_st_x4(t_s, mine);
      tmem_st_done();
      tc_fence_before();
      arrive_warp(&b_alldone);
      ok = wait_all(&b_alldone, piece & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t ml_a[4], ml_b[4];
      tmem_ld_x4(par ? tmem + t_lane : t_s, ml_a);
      tmem_ld_x4(tmem + t_lane + 128, ml_b);
      tmem_ld_wait();
      tc_fence_before();
      const uint64_t bad = sh_bad[piece & 1] & row.seen;
      if (c.left > 0) put(c, w.has);  // the next piece's scores begin while this one's rows are written
      // ---- the piece's rows
      if (row.live) {
        const float4 ma = make_float4(__uint_as_float(ml_a[0]), __uint_as_float(ml_a[1]), __uint_as_float(ml_a[2]),
                                      ml_a[3] ? 1.f : 0.f);
        const float4 mb = make_float4(__uint_as_float(ml_b[0]), par ? __uint_as_float(ml_b[1]) : 0.f,
                                      __uint_as_float(ml_b[2]), ml_b[3] ? 1.f : 0.f);
        // a unit that saw nothing weighs 0, whatever its sums hold
        const bool use_a = row.here && ma.y != 0.f, use_b = row.here && mb.y != 0.f;
        const float mm = fmaxf(use_a ? ma.x : kFloor, use_b ? mb.x : kFloor);
        const float ka = use_a ? exp2_approx(ma.x - mm) : 0.f, kb = use_b ? exp2_approx(mb.x - mm) : 0.f;
        const float ll = (use_a ? ka * ma.y : 0.f) + (use_b ? kb * mb.y : 0.f);
        const bool whole = old.t0 == 0 && old.t1 == old.n;
        const float inv = ll == 0.f ? 0.f : whole ? 1.f / ll : 1.f;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (old.t0 > 0 ? 0 : 1);
        const int in_pair = par ? lr : r * kRows + lr;
        const int kvh = old.kr / p.row_pairs;
        if (!whole && row.has && (!par || r == 0)) p.ml_part[slot * p.pair_rows + in_pair] = make_float2(mm, ll);
        const int c0 = par ? r * (D / 2) : 0, c1 = par ? c0 + D / 2 : D;
        const uint32_t o_a = t_o + (par ? 0 : r * 128), o_b = t_o + 128;
        const float4* sum_a = reinterpret_cast<const float4*>(p.o_sum + ((static_cast<int64_t>(blockIdx.x) * 2 + (par ? 0 : r)) * kRows + lr) * D);
        const float4* sum_b = reinterpret_cast<const float4*>(p.o_sum + ((static_cast<int64_t>(blockIdx.x) * 2 + 1) * kRows + lr) * D);
        T* dst = static_cast<T*>(p.out) + (row.token * p.heads + row.hd) * D;
#pragma unroll 1
        for (int cc = c0; cc < c1; cc += 32) {
          uint32_t x[32];
          float f[32];
          tmem_ld_32x32b_x32(o_a + cc, x);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = use_a ? ka * __uint_as_float(x[i]) : 0.f;
          if (kLong && use_a && ma.w != 0.f) {
            const float k = ka * ma.z;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 y = sum_a[cc / 4 + i];
              f[4 * i] = fmaf(k, y.x, f[4 * i]);
              f[4 * i + 1] = fmaf(k, y.y, f[4 * i + 1]);
              f[4 * i + 2] = fmaf(k, y.z, f[4 * i + 2]);
              f[4 * i + 3] = fmaf(k, y.w, f[4 * i + 3]);
            }
          }
          if (par) {
            __syncwarp();
            tmem_ld_32x32b_x32(o_b + cc, x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (use_b) f[i] = fmaf(kb, __uint_as_float(x[i]), f[i]);
            if (kLong && use_b && mb.w != 0.f) {
              const float k = kb * mb.z;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 y = sum_b[cc / 4 + i];
                f[4 * i] = fmaf(k, y.x, f[4 * i]);
                f[4 * i + 1] = fmaf(k, y.y, f[4 * i + 1]);
                f[4 * i + 2] = fmaf(k, y.z, f[4 * i + 2]);
                f[4 * i + 3] = fmaf(k, y.w, f[4 * i + 3]);
              }
            }
          }
          if (bad != 0 && row.here) {  // what was zeroed because it is not finite
            for (uint64_t rest = bad; rest != 0; rest &= rest - 1) {
              const int64_t slot = static_cast<int64_t>(old.pre) + __ffsll(static_cast<long long>(rest)) - 1;
              const T* vs = static_cast<const T*>(p.v_cache) + old.b * tr.stride_b + kvh * tr.stride_h + slot * tr.stride_p + cc;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float y = static_cast<float>(vs[i]);
                if (!(fabsf(y) <= 3.4e38f)) f[i] += y;
              }
            }
          }
          if (row.has) {
            if (whole) {
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                float g[8];
#pragma unroll
                for (int y = 0; y < 8; ++y) g[y] = f[i + y] * inv;
                *reinterpret_cast<uint4*>(dst + cc + i) = pack8<T>(g);
              }
            } else {
              // Two row tiles: column by column, a warp's rows side by side (row by row a piece of 160 rows took
              // 3.7 us).  One: row by row, whose pieces a warp joins with its lanes on them (25 rows of 17
              // pieces took 18.2 us instead of 13.6 otherwise).
              float* po = kTwo ? p.o_part + (slot * D + cc) * p.pair_rows + in_pair : p.o_part + (slot * p.pair_rows + in_pair) * D + cc;
              if (kTwo) {
#pragma unroll
                for (int i = 0; i < 32; ++i) po[static_cast<int64_t>(i) * p.pair_rows] = f[i];
              } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                  reinterpret_cast<float4*>(po)[i] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
              }
            }
          }
          __syncwarp();
        }
        tc_fence_before();
      }
      arrive_warp(&b_segdone);
      ++piece;
      if (c.left <= 0) break;
    }
  } else if (warp == 8) {
    if (lane == 0) {
      // ---------------------------------------------------------- K and V tiles, in turn, into the ring
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int slot = 0, loads = 0;
      uint32_t on_tail = 0, tails = 0;  // by slot: the last load completes on b_tail; the parity of its next phase
      uint32_t phase = 1;  // of the slot's release
      bool ok = true;
      int4 cut = make_int4(-1, 0, 0, 0);
      while (ok && c.left > 0) {
        const int kvh = c.kr / p.row_pairs;
        const int tail = tail_of(c.pre);
        if (c.t0 == 0 && c.t1 < c.n) cut = make_int4(c.b, c.kr, 1 + (c.n - c.t1 + sh_share - 1) / sh_share, 0);
        for (int j = c.t0; ok && j < c.t1; ++j) {
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            if (loads >= kStages) ok = mbar_wait(&b_free[slot], phase, &sh_abort, p.status);
            if (!ok) break;
            uint64_t* bar = kv && j >= tail ? &b_tail[slot] : &b_full[slot];
            mbar_arrive_expect_tx(bar, L::kTile);
            on_tail = (on_tail & ~(1u << slot)) | (bar == &b_tail[slot] ? 1u << slot : 0u);
            if (bar == &b_tail[slot]) tails ^= 1u << slot;
#pragma unroll
            for (int g = 0; g < D / 64; ++g)
              tma_load_4d(s_ring + slot * L::kTile + g * L::kPanel, kv ? &tm_v : &tm_k, bar, 64 * g, j * kStep, kvh, c.b);
            ++loads;
            if (++slot == kStages) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
        next_piece(p, c);
      }
      p.desc[blockIdx.x] = cut;
      if (!ok) {  // the copies in flight land before the CTA ends
        int never = 0;
        for (int i = loads > kStages ? loads - kStages : 0; i < loads; ++i) {
          const int at = i % kStages;
          if ((on_tail >> at) & 1u)
            mbar_wait(&b_tail[at], ((tails >> at) & 1u) ^ 1u, &never, p.status);
          else
            mbar_wait(&b_full[at], (i / kStages) & 1, &never, p.status);
        }
      }
    }
    __syncwarp();
  } else if (warp != 10) {
    // ------------------------------------------------------------ MMA issuers
    const int r = warp == 9 ? 0 : 1;
    const uint32_t idesc_s = (1u << 4) | Mma16<T>::kType | (kStep >> 3 << 17) | (kRows >> 4 << 24);
    const uint32_t idesc_o = (1u << 4) | Mma16<T>::kType | (1u << 16) | (D >> 3 << 17) | (kRows >> 4 << 24);
    const uint64_t dq = umma_smem_desc_sw128(s_q), dk = umma_smem_desc_sw128(s_ring), dv = desc_mn(s_ring, L::kPanel);
    int piece = 0, u = 0;
    uint32_t lb = 0;  // loads before the piece
    bool ok = true;
    while (ok && c.left > 0) {
      const int rows = rows_of(c.kr), nt = c.t1 - c.t0;
      const bool par = rows <= kRows;
      const int steps = steps_of(par, rows, nt, r);
      auto release = [&](uint32_t slot) {
        commit_warp(&b_free[slot]);
        if (par) commit_warp(&b_free[slot]);
      };
      auto issue_s = [&](int t) {
        const int h = (u + t) & 1, j = par ? 2 * t + r : t;
        const uint32_t slot = (lb + 2 * j) % kStages;
        const uint64_t qa = dq + ((!kTwo || par ? 0 : r * L::kQ) >> 4), kb = dk + (slot * L::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16_ss(tmem + r * 128 + h * kStep, qa + (((kk >> 2) * L::kQPanel + (kk & 3) * 32) >> 4),
                      kb + (((kk >> 2) * L::kPanel + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
        commit_warp(&b_sfull[r][h]);
        release(slot);
      };
      auto issue_o = [&](int t) {
        const int h = (u + t) & 1, j = par ? 2 * t + r : t;
        const uint32_t slot = (lb + 2 * j + 1) % kStages;
        const uint64_t vb = dv + (slot * L::kTile >> 4);
#pragma unroll
        for (int kk = 0; kk < kStep / 16; ++kk)
          umma_f16_ts(tmem + 256 + r * 128, tmem + r * 128 + h * kStep + kk * 8, vb + (kk * 2048 >> 4), idesc_o,
                      (kLong ? t % kWindow : t) != 0 || kk > 0 ? 1u : 0u);
        commit_warp(&b_odone[r][h]);
        release(slot);
      };
      ok = wait_all(&b_qready, piece & 1);
      auto loaded = [&](int t, int values) -> bool {  // step t's keys or values
        const uint32_t at = lb + 2 * (par ? 2 * t + r : t) + values;
        return wait_all(&b_full[at % kStages], (at / kStages) & 1);
      };
      for (int t = 0; ok && t < 2 && t < steps; ++t) {
        ok = loaded(t, 0);
        if (!ok) break;
        tc_fence_after();
        issue_s(t);
      }
      for (int t = 0; ok && t < steps; ++t) {
        ok = loaded(t, 1) && wait_all(&b_pready[r][(u + t) & 1], ((u + t) >> 1) & 1);
        if (!ok) break;
        tc_fence_after();
        issue_o(t);
        if (t + 2 < steps) {
          ok = loaded(t + 2, 0);
          if (!ok) break;
          tc_fence_after();
          issue_s(t + 2);
        }
      }
      u += steps;
      lb += 2 * nt;
      ++piece;
      next_piece(p, c);
    }
    // every MMA has retired before tensor memory is given back
    commit_warp(&b_done);
    int never = 0;
    mbar_wait(&b_done, 0, &never, p.status);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ cleaning: two rows of values per lane
    LaneTree tree;
    int tree_b = -1, piece = 0;
    uint32_t lb = 0, used = 0;  // used: parity of each slot's b_tail
    bool ok = true;
    while (ok && c.left > 0) {
      if (piece > 0) ok = wait_all(&b_segdone, (piece - 1) & 1);  // the notes of the piece before have been read
      if (!ok) break;
      const int pre = c.pre < 0 ? 0 : c.pre, tail = tail_of(c.pre);
      if (c.b != tree_b) {
        tree = load_tree(tr, c.b, c.pre, lane, false, p.status);
        tree_b = c.b;
      }
      uint64_t bad = 0;
      for (int j = max(tail, c.t0); ok && j < c.t1; ++j) {
        const uint32_t at = lb + 2 * (j - c.t0) + 1, slot = at % kStages;
        ok = wait_all(&b_tail[slot], (used >> slot) & 1u);
        if (!ok) break;
        used ^= 1u << slot;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int in = half * 32 + lane, rel = j * kStep + in - pre;
          uint64_t seen;
          const bool there = tree_token(tree, rel < 0 ? 0 : rel & 63, seen) && rel < 64;
          bool odd = false;
          if (rel >= 0) {
            const uint32_t row = s_ring + slot * L::kTile + in * 128;
#pragma unroll
            for (int g = 0; g < D / 64; ++g)
#pragma unroll
              for (int x = 0; x < 8; ++x) {
                const uint32_t a = row + g * L::kPanel + ((x ^ (in & 7)) << 4);
                if (!there) {
                  sts128(a, 0u, 0u, 0u, 0u);
                  continue;
                }
                uint32_t v[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
                // an exponent of all ones carries into the sign's place
                constexpr uint32_t kE2 = Mma16<T>::kExp * 0x10001u, kOne2 = (0x8000u - Mma16<T>::kExp) * 0x10001u;
                if (((((v[0] & kE2) + kOne2) | ((v[1] & kE2) + kOne2) | ((v[2] & kE2) + kOne2) | ((v[3] & kE2) + kOne2)) & 0x80008000u) == 0)
                  continue;
                odd = true;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  if ((v[y] & Mma16<T>::kExp) == Mma16<T>::kExp) v[y] &= 0xffff0000u;
                  if ((v[y] & (Mma16<T>::kExp << 16)) == (Mma16<T>::kExp << 16)) v[y] &= 0x0000ffffu;
                }
                sts128(a, v[0], v[1], v[2], v[3]);
              }
          }
          const uint32_t odds = __ballot_sync(0xffffffffu, odd);
          const int bit0 = j * kStep + half * 32 - pre;  // token of lane 0
          if (odds) bad |= bit0 >= 0 ? static_cast<uint64_t>(odds) << bit0 : static_cast<uint64_t>(odds) >> -bit0;
        }
        fence_async_proxy();
        arrive_warp(&b_full[slot]);
      }
      if (!ok) break;
      if (lane == 0) sh_bad[piece & 1] = bad;
      arrive_warp(&b_fixed);
      lb += 2 * (c.t1 - c.t0);
      ++piece;
      next_piece(p, c);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of the pairs that the runs' ends cut: CTA (c, y) takes eight rows of the
// pair that begins in run c and ends in a later one, a warp each.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_attn_combine_kernel(const TreeAttnParams p) {
  constexpr int kE = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();  // the pieces
  const int cta = blockIdx.x;
  const int4 cut = p.desc[cta];
  if (cut.x < 0) return;
  const int parts = cut.z, in = static_cast<int>(blockIdx.y) * 8 + warp;
  const int row = cut.y % p.row_pairs * p.pair_rows + in;
  if (row >= p.tree.tokens * p.group || in >= p.pair_rows) return;
  // piece i: the run's later slot, then the first slots of the runs behind it
  auto at = [&](int i) { return (static_cast<int64_t>(cta + i) * 2 + (i == 0 ? 1 : 0)) * p.pair_rows + in; };
  float mx = kFloor;
  for (int i = lane; i < parts; i += 32) {
    const float2 ml = p.ml_part[at(i)];
    if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
  }
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
  float l = 0.f, f[kE];
#pragma unroll
  for (int x = 0; x < kE; ++x) f[x] = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 32) {
    float2 ml = make_float2(kFloor, 0.f);
    if (i0 + lane < parts) ml = p.ml_part[at(i0 + lane)];
    const float w = ml.y == 0.f ? 0.f : exp2_approx(ml.x - mx);
    const uint32_t live = __ballot_sync(0xffffffffu, ml.y != 0.f);
    float wl = ml.y == 0.f ? 0.f : w * ml.y;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) wl += __shfl_xor_sync(0xffffffffu, wl, x);
    l += wl;
    const int here = min(32, parts - i0);
#pragma unroll 4
    for (int i = 0; i < here; ++i) {
      const float k = __shfl_sync(0xffffffffu, w, i);
      if (!((live >> i) & 1u)) continue;  // a piece that saw nothing weighs 0, whatever its rows hold
      const float* src = p.o_part + at(i0 + i) * D + lane * kE;
      float v[kE];
      if (kE == 4)
        *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      else
        *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
      for (int x = 0; x < kE; ++x) f[x] = fmaf(k, v[x], f[x]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int kvh = cut.y / p.row_pairs;
  const int64_t token = static_cast<int64_t>(cut.x) * p.tree.tokens + row / p.group;
  T* dst = static_cast<T*>(p.out) + (token * p.heads + kvh * p.group + row % p.group) * D + lane * kE;
  if (kE == 4)
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(Half16<T>::pack(f[0] * inv, f[1] * inv), Half16<T>::pack(f[kE - 2] * inv, f[kE - 1] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = Half16<T>::pack(f[0] * inv, f[1] * inv);
}

// The same of two row tiles, whose pieces lie column by column: CTA (c, y) takes 32 rows, a lane per row
// and D / 8 columns per warp.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_attn_combine_cols_kernel(const TreeAttnParams p) {
  constexpr int kCols = D / 8, kPitch = 2 * D + 16, kPieces = 4;
  __shared__ __align__(16) uint8_t tile[32 * kPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();  // the pieces
  const int cta = blockIdx.x;
  const int4 cut = p.desc[cta];
  if (cut.x < 0) return;
  const int parts = cut.z, in = static_cast<int>(blockIdx.y) * 32 + lane, row0 = cut.y % p.row_pairs * p.pair_rows;
  const bool has = in < p.pair_rows && row0 + in < p.tree.tokens * p.group;
  // piece i: the run's later slot, then the first slots of the runs behind it
  auto slot = [&](int i) { return static_cast<int64_t>(cta + i) * 2 + (i == 0 ? 1 : 0); };
  const int at = has ? in : 0;
  float mx = kFloor;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float2 ml = p.ml_part[slot(i) * p.pair_rows + at];
    if (ml.y != 0.f) mx = fmaxf(mx, ml.x);
  }
  float l = 0.f, f[kCols];
#pragma unroll
  for (int x = 0; x < kCols; ++x) f[x] = 0.f;
  for (int i0 = 0; i0 < parts; i0 += kPieces) {  // several pieces' loads at once
    float2 ml[kPieces];
    float v[kPieces][kCols];
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int64_t from = slot(i0 + k < parts ? i0 + k : 0);
      ml[k] = p.ml_part[from * p.pair_rows + at];
      if (i0 + k >= parts) ml[k].y = 0.f;
#pragma unroll
      for (int x = 0; x < kCols; ++x) v[k][x] = p.o_part[(from * D + warp * kCols + x) * p.pair_rows + at];
    }
#pragma unroll
    for (int k = 0; k < kPieces; ++k)
      if (ml[k].y != 0.f) {  // a piece that saw nothing weighs 0, whatever its rows hold
        const float w = exp2_approx(ml[k].x - mx);
        l = fmaf(w, ml[k].y, l);
#pragma unroll
        for (int x = 0; x < kCols; ++x) f[x] = fmaf(w, v[k][x], f[x]);
      }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int x = 0; x < kCols; x += 8) {
    float g[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) g[y] = f[x + y] * inv;
    *reinterpret_cast<uint4*>(tile + lane * kPitch + (warp * kCols + x) * 2) = pack8<T>(g);
  }
  __syncthreads();
  const int kvh = cut.y / p.row_pairs;
  for (int e = threadIdx.x; e < 32 * (D / 8); e += 256) {
    const int mine = static_cast<int>(blockIdx.y) * 32 + e / (D / 8), row = row0 + mine;
    if (mine >= p.pair_rows || row >= p.tree.tokens * p.group) continue;
    const int64_t token = static_cast<int64_t>(cut.x) * p.tree.tokens + row / p.group;
    T* dst = static_cast<T*>(p.out) + (token * p.heads + kvh * p.group + row % p.group) * D;
    reinterpret_cast<uint4*>(dst)[e % (D / 8)] = *reinterpret_cast<const uint4*>(tile + e / (D / 8) * kPitch + e % (D / 8) * 16);
  }
}

struct Plan {
  int ctas, row_pairs, pair_rows;
  size_t ml_off, o_off, sum_off, bytes;
};

Plan plan_of(const TreeView& t, int heads, int dim, int num_sms) {
  Plan a;
  const int64_t rows = static_cast<int64_t>(heads / t.kv_heads) * t.tokens;
  a.pair_rows = rows <= kRows ? kRows : 2 * kRows;
  a.row_pairs = static_cast<int>((rows + a.pair_rows - 1) / a.pair_rows);
  const int64_t tiles = (t.capacity + kStep - 1) / kStep * t.batch * t.kv_heads * a.row_pairs;  // at most
  a.ctas = static_cast<int>(tiles < num_sms ? tiles : num_sms);
  auto up = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t slots = static_cast<size_t>(a.ctas) * 2 * a.pair_rows;
  a.ml_off = up(static_cast<size_t>(a.ctas) * sizeof(int4));
  a.o_off = a.ml_off + up(slots * sizeof(float2));
  a.sum_off = a.o_off + up(slots * dim * sizeof(float));
  a.bytes = a.sum_off;
  // sums of the units' rows, where a unit may take more steps than a window of either type
  if ((t.capacity + kStep - 1) / kStep > window_steps<__half>())
    a.bytes += static_cast<size_t>(a.ctas) * 2 * kRows * dim * sizeof(float);
  return a;
}

template <typename T, int D, bool kTwo>
int attn_t(const TreeAttnParams& p, const Plan& a, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  constexpr int smem = TreeSmem<D, kTwo>::kBytes;
  const int64_t tiles = (p.tree.capacity + kStep - 1) / kStep;
  auto* kernel = tiles > window_steps<T>() ? tree_attn_kernel<T, D, kTwo, true> : tree_attn_kernel<T, D, kTwo, false>;
  if (!set_smem_limit(kernel, smem)) return FITQ_ERR_CUDA;
  cudaError_t e = launch_pdl(kernel, dim3(a.ctas), dim3(kThreads), smem, st, tk, tv, p);
  note_launch();
  if (e != cudaSuccess) return FITQ_ERR_CUDA;
  if (a.ctas > 1) {
    const int rows = p.tree.tokens * p.group < a.pair_rows ? p.tree.tokens * p.group : a.pair_rows;
    e = kTwo ? launch_pdl(tree_attn_combine_cols_kernel<T, D>, dim3(a.ctas, (rows + 31) / 32), dim3(256), 0, st, p)
             : launch_pdl(tree_attn_combine_kernel<T, D>, dim3(a.ctas, (rows + 7) / 8), dim3(256), 0, st, p);
    note_launch();
    if (e != cudaSuccess) return FITQ_ERR_CUDA;
  }
  return launch_result();
}

template <typename T>
int attn_sized(const TreeAttnParams& p, const Plan& a, int dim, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  if (dim == 128) return a.pair_rows > kRows ? attn_t<T, 128, true>(p, a, tk, tv, st) : attn_t<T, 128, false>(p, a, tk, tv, st);
  return a.pair_rows > kRows ? attn_t<T, 64, true>(p, a, tk, tv, st) : attn_t<T, 64, false>(p, a, tk, tv, st);
}

}  // namespace

size_t tree_attention_workspace(const TreeView& tree, int heads, int dim, int num_sms) {
  return plan_of(tree, heads, dim, num_sms).bytes;
}

int launch_tree_attention(const TreeView& tree, const void* q, int64_t q_stride, const void* k_cache,
                          const void* v_cache, void* out, int heads, int dim, int dtype, void* workspace, int* status,
                          cudaStream_t st, int num_sms) {
  const Plan a = plan_of(tree, heads, dim, num_sms);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const TreeAttnParams p{tree, q, v_cache, out, reinterpret_cast<int4*>(ws), reinterpret_cast<float2*>(ws + a.ml_off),
                         reinterpret_cast<float*>(ws + a.o_off), reinterpret_cast<float*>(ws + a.sum_off), q_stride, heads,
                         heads / tree.kv_heads, a.row_pairs, a.pair_rows,
                         1.4426950408889634f / sqrtf(static_cast<float>(dim)), status};
  // a dimension of one entry may come with any stride: the map gets one it takes
  auto bytes = [&](int64_t stride, int64_t n) { return static_cast<uint64_t>((n > 1 ? stride : dim) * 2); };
  const uint64_t dims[4] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(tree.capacity),
                            static_cast<uint64_t>(tree.kv_heads), static_cast<uint64_t>(tree.batch)};
  const uint64_t strides[3] = {bytes(tree.stride_p, tree.capacity), bytes(tree.stride_h, tree.kv_heads),
                               bytes(tree.stride_b, tree.batch)};
  const uint32_t box[4] = {64, kStep, 1, 1};
  const CUtensorMapDataType type = dtype == FITQ_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tk, tv;
  if (!encode_tmap_4d(&tk, type, k_cache, dims, strides, box) || !encode_tmap_4d(&tv, type, v_cache, dims, strides, box))
    return FITQ_ERR_CUDA;
  return dtype == FITQ_DTYPE_BF16 ? attn_sized<__nv_bfloat16>(p, a, dim, tk, tv, st)
                                  : attn_sized<__half>(p, a, dim, tk, tv, st);
}

}  // namespace fitq
