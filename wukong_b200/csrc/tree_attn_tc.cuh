// Tree attention on the 5th-generation tensor cores, for pages of 8 tokens and more.
//
// Work.  A unit is (tree, KV head, 128 of the tree's query rows, node-major with the heads of the group inside); its
// keys are cut into blocks of 128.  All blocks of all units form one list that is dealt out in equal contiguous shares to
// as many CTAs as the SMs hold, whatever the lengths: a share may hold several units, or a piece of one.  A unit that a
// single share covers is written at once; the pieces of the others go to scratch as (maximum, sum, unnormalised output) and
// are joined by tree_attn_join_kernel in key order, so results are run-to-run identical.  When the arguments say that there
// are no more units than CTAs and that they are short, units stay whole and nothing is joined.
//
// A CTA has two TMA warps (pages of K and of V into a ring each), an MMA warp and one or two teams of four softmax warps.
//   S = Q K^T (128 x 128) -> P = exp2(S - m), bf16 -> O += P V (128 x head_dim)      (P over S, or beside it where there is room)
// Two teams take alternate key blocks with tensor-memory columns of their own, so one team's exponentials run while the
// other's products do; a single team leaves that to the SM's other CTA.  The running maximum m of a row moves only when a
// block exceeds it by 2^8; the accumulator is rescaled then and not at every block.  f32 queries are two bf16 parts (hi +
// lo, two products); for f32 results P is two parts as well: 16 bits of each, 3e-6 of the result in the mean for unit-normal
// queries (2e-6 for bf16 ones), 5e-6 for queries half as large again.  bf16 results keep P in one part: 2.1e-3 in the mean,
// of which the result's own rounding is 1.7e-3; the second part would leave that alone, for 10 to 21 % of the time (tree of 64
// nodes over 32749 tokens 57.7 -> 69.8 us, Llama-shape batch 137 -> 161 us called).
//
// Bound.  K and V are read once from HBM (569.9 MB for 571.6 MB of work in the Llama-shape batch of 64 trees; once for each
// 128 query rows where a head has more and its K and V do not fit L2) and stream at the copy rate inside a unit: 1.41 us a block of head_dim 128 on all SMs together, 0.72 us of head_dim 64.  The batch takes 111
// to 117 us from card to card (137 in a loop of seconds, where the board's power cap lowers the clock to 1.53 GHz) against 87 us of its bytes; the rest is the beginnings and ends of units (8 k cycles each, partly under the rings'
// prefetch), the first trip to memory and the join (4 us).  With 128 rows a unit it is the chain S -> softmax -> P V of
// the teams, 2200 cycles a block against 1330 of the tensor pipe and the shared-memory port.
//
// With 64 (32) query rows or fewer the operand's 128 rows hold 2 (4) copies of them, and each copy takes its own half
// (quarter) of a block's keys, with zeros for the others': a team's warps share the exponentials of a small tree that
// would otherwise all fall to one of them.  The copies are added up like the pieces of a unit.
//
// V and 0 x NaN: a probability of zero does not silence a NaN or an infinity in the product.  In the blocks with tree
// nodes and behind the last key, where rows see different keys, V elements that are not finite are set to zero in shared
// memory before the product.  In the committed context, which every row sees, one makes the result something that is not
// finite, but not always the right thing: a weight below f32, a copy's zero or a negative lo part of P makes NaN of an
// infinity.  Either way the elements' own sum over the keys that a row sees is put in the result's place.
#pragma once
#include "common.cuh"
#include "tc_common.cuh"
#include <type_traits>

namespace wkb {
int* gemm_status_word();

namespace tree {

constexpr int KBLK = 128, QROWS = 128, SUB = 128 * 128;

// Header of the scratch: where share c begins, for the join.  Then (m, l) and O of two pieces a share.
struct ShareStart {
  int unit_start, unit_len, share, total, row0, live, head, rowblk;      // unit_len 0: it begins in none; total -1: a wait ran out
};
struct Scratch {
  ShareStart* start;
  float2* ml;
  float* o;
  int rows;      // rows a piece has room for
};
__host__ __device__ inline int piece_rows(i64 max_nodes, i64 group) {
  const i64 r = max_nodes * group;
  return (int)(r < QROWS ? r : QROWS);
}
inline i64 scratch_bytes(i64 max_nodes, i64 group, i64 hd, i64 shares) {
  const i64 rows = 2 * shares * (i64)piece_rows(max_nodes, group);
  return (i64)sizeof(ShareStart) * shares + rows * 8 + rows * hd * 4;
}
inline Scratch carve(void* p, i64 max_nodes, i64 group, i64 shares) {
  const int r = piece_rows(max_nodes, group);
  uint8_t* b = static_cast<uint8_t*>(p);
  Scratch s;
  s.start = reinterpret_cast<ShareStart*>(b);
  s.ml = reinterpret_cast<float2*>(b + sizeof(ShareStart) * shares);
  s.o = reinterpret_cast<float*>(b + sizeof(ShareStart) * shares + 2 * shares * r * 8);
  s.rows = r;
  return s;
}
static_assert(sizeof(ShareStart) % 16 == 0, "the planes behind the header stay 16-byte aligned");

// How a key block lies in shared memory: boxes of whole rows of a page, the 64-dim halves of a box behind one another (one
// copy a box; copies of half rows were twice as many, and their issue was the limit).  With two halves a box is 8 tokens,
// so that the block's 8-key groups are evenly spaced and one instruction multiplies all 128 keys; boxes of 16 tokens need
// two of 64 keys each, and reading the query operand twice cost more (1.53 against 1.41 us a block) than it saved.
template <int HD>
struct Layout {
  static constexpr int HALVES = HD / 64, GROUP = 1024 * HALVES, HALF = 1024;      // distance of the 8-key groups, of the halves
  static __host__ __device__ int box_rows(int page_tokens) { return HALVES == 2 ? 8 : page_tokens < KBLK ? page_tokens : KBLK; }
};

// head_dim 128: one CTA per SM with two teams, which take alternate blocks.  head_dim 64: everything is half as large, so
// two CTAs of one team fit an SM; they work on different units, and one's beginnings and ends run under the other's
// products (33 us with two teams, 30 with two CTAs, for 32 trees of a GPT-2 shape).
template <int HD>
struct Shape {
  static constexpr int TEAMS = HD == 64 ? 1 : 2, CTAS = 2 / TEAMS, THREADS = TEAMS == 2 ? 384 : 256, SHARES = WKB_SM_COUNT * CTAS;
  static constexpr int SMEM = TEAMS == 2 ? 232448 : 115712;                       // a CTA's part of 228 KB, 1 KB of each CTA reserved
  static constexpr int TM_COLS = 256 * TEAMS, O_COL = 128 * TEAMS;                // tensor memory: the teams' S (128 columns each), then their O
};
inline int shares_of(i64 hd) { return hd == 64 ? Shape<64>::SHARES : Shape<128>::SHARES; }

template <int HD, int QS>
struct TcSmem {
  static constexpr int NSUB = HD / 64, BLK = NSUB * SUB;                 // bytes of 128 rows of an operand
  static constexpr int HEADER = 3 * 1024;                                  // barriers, (m, l) of the teams, flags
  // the stage (the copies' sums, and the next query's raw rows): of its own beside two teams; a single team's lies over the
  // query, which is not needed when a result is written
  static constexpr int TEAMS = Shape<HD>::TEAMS, STAGE = QROWS * 64 * 4, STAGE_BYTES = TEAMS == 2 ? STAGE : 0;
  static constexpr int Q_BYTES = TEAMS == 1 && QS * BLK < STAGE ? STAGE : QS * BLK;
  static constexpr int SLOTS = (Shape<HD>::SMEM - HEADER - Q_BYTES - STAGE_BYTES) / BLK;
  static constexpr int NK = (SLOTS + 1) / 2, NV = SLOTS / 2;
  static constexpr int BYTES = HEADER + Q_BYTES + STAGE_BYTES + SLOTS * BLK;
  static_assert(NV >= 2 && BYTES <= Shape<HD>::SMEM, "at least two blocks of each operand in flight");
};

__host__ __device__ constexpr uint32_t tc_idesc(int n, bool b_mn) {      // kind::f16: D f32, A = B = bf16, M = 128
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(QROWS >> 4) << 24);
}
// Shared-memory operand with 128-byte swizzle, atoms of 8 rows of 128 bytes.  K-major (Q, K): sbo = distance of 8-row
// groups, lbo not used.  MN-major (V as it lies in the cache, 64 dims a row): sbo = distance of 8-key groups, lbo of the halves.
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// One box of the cache, box_rows tokens x all dims of one head, as [64-dim half][token][128 bytes].
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
               "r"(bar), "r"(0), "r"(row), "r"(0)
               : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(id),
               "r"(accumulate)
               : "memory");
}
#define WKB_R8(a, i) "=r"(a[i]), "=r"(a[i + 1]), "=r"(a[i + 2]), "=r"(a[i + 3]), "=r"(a[i + 4]), "=r"(a[i + 5]), "=r"(a[i + 6]), "=r"(a[i + 7])
#define WKB_I8(a, i) "r"(a[i]), "r"(a[i + 1]), "r"(a[i + 2]), "r"(a[i + 3]), "r"(a[i + 4]), "r"(a[i + 5]), "r"(a[i + 6]), "r"(a[i + 7])
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* r) {      // 32 columns of this thread's lane; wait with tm_ld_wait
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : WKB_R8(r, 0), WKB_R8(r, 8), WKB_R8(r, 16), WKB_R8(r, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tm_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      WKB_I8(r, 0), WKB_I8(r, 8)
      : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      WKB_I8(r, 0), WKB_I8(r, 8), WKB_I8(r, 16), WKB_I8(r, 24)
      : "memory");
}
#undef WKB_R8
#undef WKB_I8
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 at a time
__device__ __forceinline__ uint64_t two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void of_two(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Parity wait of at most about a second; each try may park the thread until the phase completes.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((it & 255u) == 255u) {
      uint64_t t;
      asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
      if (t0 == 0) t0 = t;
      else if (t - t0 > 1000000000ull) return false;
    }
  }
}
// non-zero when one of a word's two bf16 has an exponent of all ones
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) { return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }
// What 8 bf16 hold that is not finite, a nibble for each: 1 infinity, 2 minus infinity, 4 NaN.  Or-ing nibbles adds elements
// up, in any order: the sum is what kind_sum gives (none, an infinity, or NaN for a NaN or both infinities).
__device__ __forceinline__ uint32_t kinds_of(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t kinds = 0u;
  if (!(not_finite2(w[0]) | not_finite2(w[1]) | not_finite2(w[2]) | not_finite2(w[3]))) return kinds;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = (w[e >> 1] >> (16 * (e & 1))) & 0xffffu;
    if ((b & 0x7f80u) == 0x7f80u) kinds |= ((b & 0x7fu) ? 4u : (b >> 15) ? 2u : 1u) << (4 * e);
  }
  return kinds;
}
__device__ __forceinline__ float kind_sum(uint32_t kind) { return kind == 1u ? INFINITY : kind == 2u ? -INFINITY : NAN; }
__device__ __forceinline__ uint32_t low_bits(i64 n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// A tree's share of the work list.
struct TreeWork {
  TreeRef t;
  int keys, blocks, rowblks;
};
__device__ __forceinline__ TreeWork tree_work(const Geo& g, const int* slot, const int* ctx, const int* row0, int t) {
  TreeWork w;
  w.t = tree_ref(g, slot, ctx, row0, t);
  const i64 keys = (i64)w.t.ctx + w.t.nodes, cover = (i64)g.mbps * g.page_tokens;
  w.keys = (int)(keys < cover ? keys : cover);
  w.t.ctx = min(w.t.ctx, w.keys);
  w.blocks = (w.keys + KBLK - 1) / KBLK;
  w.rowblks = (w.t.nodes * (g.q_heads / g.kv_heads) + QROWS - 1) / QROWS;      // 0 for a tree without rows
  return w;
}
// A unit counts as its blocks and UNIT_COST more: what beginning and ending one takes, in blocks (0: 161 us, 2: 118, 3: 116,
// 4: 114, 7: 118, 10: 123 on one card, for the 64 trees of a Llama-shape batch).
constexpr int UNIT_COST = 4;
__device__ __forceinline__ int unit_items(const Geo& g, const TreeWork& w) { return g.split ? w.blocks + UNIT_COST : 1; }
__device__ __forceinline__ int tree_items(const Geo& g, const TreeWork& w) { return unit_items(g, w) * w.rowblks * g.kv_heads; }

// One piece of a unit: blocks [b0, b1) of `unit_len`.
struct Piece {
  TreeWork w;
  int head, rowblk, unit_start, b0, b1;
};
// Walks a share: item is its position in the list, tree_start that of tree `tree`.
struct Walk {
  int item, end, tree, tree_start;
  __device__ __forceinline__ bool next(const Geo& g, const int* slot, const int* ctx, const int* row0, Piece& p) {
    while (item < end) {
      for (;;) {
        p.w = tree_work(g, slot, ctx, row0, tree);
        const int items = tree_items(g, p.w);
        if (item < tree_start + items) break;
        tree_start += items;
        if (++tree >= g.n_trees) return false;
      }
      const int size = unit_items(g, p.w), unit = (item - tree_start) / size;
      p.head = unit / p.w.rowblks;
      p.rowblk = unit - p.head * p.w.rowblks;
      p.unit_start = tree_start + unit * size;
      p.b0 = item - p.unit_start;
      p.b1 = g.split ? min(p.w.blocks, p.b0 + end - item) : p.w.blocks;
      item = p.unit_start + size;
      if (p.b0 < p.b1) return true;      // else the share begins behind the unit's last block
    }
    return false;
  }
};

template <int HD, int QS, int PS>
__global__ void __launch_bounds__(Shape<HD>::THREADS, Shape<HD>::CTAS)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const void* __restrict__ q,
                    const u16* __restrict__ vcache, const uint32_t* __restrict__ block_table, const int* __restrict__ slot,
                    const int* __restrict__ ctxs, const int* __restrict__ row0s, const uint32_t* __restrict__ mask, void* __restrict__ out, int out_dtype,
                    Geo g, float scale, Scratch scr, int* __restrict__ status) {
  using SM = TcSmem<HD, QS>;
  // Tensor memory: with one team and one part of P there is room for P beside S, so that the next block's scores need not wait
  // for this block's P V; else P lies over S, 32 columns (16 of each part) for 32 keys.
  constexpr bool BESIDE = Shape<HD>::TEAMS == 1 && PS == 1;
  constexpr int P_BASE = BESIDE ? Shape<HD>::O_COL + HD : 0, P_CHUNK = BESIDE ? 16 : 32;
  static_assert(!BESIDE || P_BASE + 64 <= Shape<HD>::TM_COLS, "P fits behind O");
  constexpr int NK = SM::NK, NV = SM::NV, NSUB = SM::NSUB, BLK = SM::BLK, TEAMS = Shape<HD>::TEAMS, THREADS = Shape<HD>::THREADS, CREW = 128 * TEAMS;      // crew: the softmax threads
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  // header: barriers at 0, flags at 256, (m, l) at 512 .. 2560; the operands behind it on a 1024-byte boundary
  const uint32_t q_base = (raw + 2560 + 1023u) & ~1023u, stage_base = TEAMS == 2 ? q_base + SM::Q_BYTES : q_base, k_ring = q_base + SM::Q_BYTES + SM::STAGE_BYTES, v_ring = k_ring + NK * BLK;
  auto kfull = [&](int s) { return raw + 8u * s; };
  auto kempty = [&](int s) { return raw + 8u * (NK + s); };
  auto vfull = [&](int s) { return raw + 8u * (2 * NK + s); };
  auto vempty = [&](int s) { return raw + 8u * (2 * NK + NV + s); };
  const uint32_t more = raw + 8u * (2 * NK + 2 * NV);
  auto s_full = [&](int t) { return more + 8u * t; };
  auto p_full = [&](int t) { return more + 8u * (2 + t); };
  auto o_done = [&](int t) { return more + 8u * (4 + t); };
  const uint32_t q_full = more + 8u * 6, q_first = more + 8u * 7;      // the first piece's query is everybody's work
  static_assert(8 * (2 * NK + 2 * NV + 8) <= 256, "barriers fit the header");
  volatile int* flags = reinterpret_cast<volatile int*>(smem_raw + 256);      // 0 tensor memory, 1 failed, 3 and 4 the share's first tree and its start
  // of the (up to three) blocks from that with the context's end on: which keys have a V that is not finite, a bit each
  volatile uint32_t* bad_keys = reinterpret_cast<volatile uint32_t*>(smem_raw + 288);
  float2* ml_s = reinterpret_cast<float2*>(smem_raw + 512);
  float* stage = reinterpret_cast<float*>(smem_raw + (stage_base - raw));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (q_base - raw > (uint32_t)SM::HEADER) {      // the operands would not fit behind the header: never, as the base is 1024-byte aligned
    if (threadIdx.x == 0) atomicExch(status, WKB_STATUS_ATTN_WAIT);
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < NK; ++s) { mbar_init(kfull(s), 1); mbar_init(kempty(s), 1); }
    for (int s = 0; s < NV; ++s) { mbar_init(vfull(s), 1); mbar_init(vempty(s), 1); }
    for (int t = 0; t < 2; ++t) { mbar_init(s_full(t), 1); mbar_init(p_full(t), 4); mbar_init(o_done(t), 1); }
    mbar_init(q_full, 4); mbar_init(q_first, 4 * TEAMS);
    flags[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(raw + 256), "r"((uint32_t)Shape<HD>::TM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = (uint32_t)flags[0];
  pdl_wait();
  pdl_trigger();
  // ---- this CTA's share: prefix sums of the trees' items.  Up to 32 trees every warp for itself, which saves the barriers;
  // more over all threads, a contiguous run of trees each
  int share, total;
  Walk walk;
  if (g.n_trees <= 32) {
    const int mine = lane < g.n_trees ? tree_items(g, tree_work(g, slot, ctxs, row0s, lane)) : 0;
    int scan = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    total = __shfl_sync(0xffffffffu, scan, 31);
    share = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    walk.item = min((int)blockIdx.x * share, total);
    walk.end = min(walk.item + share, total);
    const int t = __ffs(__ballot_sync(0xffffffffu, walk.item < scan)) - 1;      // -1: nothing to do
    walk.tree = max(t, 0);
    walk.tree_start = __shfl_sync(0xffffffffu, scan - mine, walk.tree);
  } else {
    int* sums = reinterpret_cast<int*>(ml_s);
    const int per = (g.n_trees + THREADS - 1) / THREADS, t0 = threadIdx.x * per, t1 = min(t0 + per, g.n_trees);
    int mine = 0;
    for (int t = t0; t < t1; ++t) mine += tree_items(g, tree_work(g, slot, ctxs, row0s, t));
    int scan = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) before += sums[w]; total += sums[w]; }
    share = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int first = (int)blockIdx.x * share;
    int at = before + scan - mine;
    if (first < total && first >= at && first < at + mine) {
      int t = t0;
      for (;; ++t) {
        const int n = tree_items(g, tree_work(g, slot, ctxs, row0s, t));
        if (first < at + n) break;
        at += n;
      }
      flags[3] = t; flags[4] = at;
    }
    __syncthreads();
    walk = Walk{min(first, total), min(first + share, total), flags[3], flags[4]};
  }
  const int group = g.q_heads / g.kv_heads, gshift = 31 - __clz(group);      // a power of two
  const bool none = walk.item >= walk.end;
  if (threadIdx.x == THREADS - 64) {      // (of the warp without a part) what the join has to know about the unit that this share begins in
    ShareStart st{0, 0, share, total, 0, 0, 0, 0};
    if (!none) {
      Walk w = walk;
      Piece p;
      if (w.next(g, slot, ctxs, row0s, p)) {
        st.unit_start = p.unit_start; st.unit_len = p.w.blocks; st.row0 = p.w.t.row0; st.head = p.head; st.rowblk = p.rowblk;
        st.live = min(QROWS, p.w.t.nodes * group - p.rowblk * QROWS);
      }
    }
    scr.start[blockIdx.x] = st;
  }
  if (none) {
    // nothing to do
  } else if (warp == 0 || warp == THREADS / 32 - 1) {
    // ---------------- TMA: one warp for K, one for V; lane i brings the i-th box of a block ----------------
    const bool is_v = warp != 0;
    const uint32_t ring = is_v ? v_ring : k_ring;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    const int slots = is_v ? NV : NK, box_rows = Layout<HD>::box_rows(g.page_tokens), boxes = KBLK / box_rows, per = 32 / boxes;
    const uint32_t box_bytes = (uint32_t)box_rows * HD * 2;
    Piece p;
    int n = 0;      // blocks so far, over all pieces of the share
    bool ok = true;
    while (ok && walk.next(g, slot, ctxs, row0s, p)) {
      const uint32_t* bt = block_table + (i64)p.w.t.slot * g.mbps;
      const i64 oob = g.num_pages * g.kv_heads * g.page_tokens;
      // The warp holds the cache rows of 32 boxes (32 / boxes blocks), lane by lane, and the next 32 are on their way: a
      // look-up a block, used at once, cost more than the copies.  Boxes behind the last key repeat the last page (their
      // keys are not seen).
      const int len = p.b1 - p.b0;
      auto cache_rows = [&](int batch) -> int {
        const i64 at = (i64)(p.b0 + batch * per) * KBLK + (i64)lane * box_rows;
        const int last = (p.w.keys - 1) / box_rows * box_rows, pos = at < last ? (int)at : last;
        const uint32_t page = bt[pos >> g.page_shift];
        return page < (uint64_t)g.num_pages ? (int)(((i64)page * g.kv_heads + p.head) * g.page_tokens + (pos & (g.page_tokens - 1))) : (int)oob;
      };
      int rows_now = cache_rows(0), rows_next = per < len ? cache_rows(1) : 0, in_batch = 0, batch = 0;
      for (int j = 0; j < len; ++j) {
        if (in_batch == per) {
          in_batch = 0;
          ++batch;
          rows_now = rows_next;
          if ((batch + 1) * per < len) rows_next = cache_rows(batch + 1);
        }
        const int row = __shfl_sync(0xffffffffu, rows_now, in_batch * boxes + (lane & (boxes - 1)));
        ++in_batch;
        const int s = n % slots;
        const uint32_t fb = is_v ? vfull(s) : kfull(s), eb = is_v ? vempty(s) : kempty(s);
        if (!__all_sync(0xffffffffu, bar_wait(eb, ((n / slots) & 1) ^ 1))) { ok = false; break; }
        if (lane == 0) mbar_expect_tx(fb, BLK);
        __syncwarp();
        if (lane < boxes) tma_box(ring + s * BLK + (uint32_t)lane * box_bytes, map, fb, row);
        ++n;
      }
    }
    if (!ok && lane == 0) {
      atomicExch(status, WKB_STATUS_ATTN_WAIT);
      flags[1] = 1;
      for (int i = max(0, n - slots); i < n; ++i) bar_wait(is_v ? vfull(i % slots) : kfull(i % slots), (i / slots) & 1);      // copies in flight
    }
  } else if (warp == 1) {
    // ---------------- MMA: S a block ahead for each team, each P V as its team delivers P ----------------
    if (lane == 0) {
      constexpr uint32_t ID_S = tc_idesc(KBLK, false), ID_O = tc_idesc(HD, true);
      using LY = Layout<HD>;
      Piece p;
      int n = 0, pieces = 0;
      int uses[2] = {0, 0};      // P V products of each team so far
      bool ok = true;
      while (ok && walk.next(g, slot, ctxs, row0s, p)) {
        const int len = p.b1 - p.b0;
        auto scores = [&](int j) {
          const int i = n + j, s = i % NK, t = j % TEAMS;
          if (!bar_wait(kfull(s), (i / NK) & 1)) return false;
          tc_fence_after();
          const uint32_t kaddr = k_ring + s * BLK;
#pragma unroll
          for (int part = 0; part < QS; ++part)
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              umma_bf16(tmem + t * 128, sdesc(q_base + part * BLK + (uint32_t)(k >> 2) * SUB + (uint32_t)(k & 3) * 32u, 16, 1024),
                        sdesc(kaddr + (uint32_t)(k >> 2) * LY::HALF + (uint32_t)(k & 3) * 32u, 16, LY::GROUP), ID_S, (part > 0 || k > 0) ? 1u : 0u);
          umma_commit(s_full(t));
          umma_commit(kempty(s));
          return true;
        };
        ok = pieces == 0 ? bar_wait(q_first, 0) : bar_wait(q_full, (pieces - 1) & 1);
        ++pieces;
        ok = ok && scores(0);
        if (TEAMS == 2 && len > 1) ok = ok && scores(1);
        for (int j = 0; j < len && ok; ++j) {
          const int t = j % TEAMS, i = n + j, s = i % NV;
          ok = bar_wait(p_full(t), uses[t] & 1);
          if (BESIDE && j + 1 < len) ok = ok && scores(j + 1);
          ok = ok && bar_wait(vfull(s), (i / NV) & 1);
          if (!ok) break;
          ++uses[t];
          tc_fence_after();
          const uint32_t vaddr = v_ring + s * BLK, o_col = tmem + Shape<HD>::O_COL + t * HD;
          // 32 keys take 32 columns of P: 16 of the hi part (two keys a column), 16 of the lo part
#pragma unroll
          for (int k = 0; k < KBLK / 16; ++k)
#pragma unroll
            for (int part = 0; part < PS; ++part)
              mma_ts(o_col, tmem + t * 128 + P_BASE + (k >> 1) * P_CHUNK + part * 16 + (k & 1) * 8, sdesc(vaddr + (uint32_t)k * 2u * LY::GROUP, LY::HALF, LY::GROUP), ID_O,
                     (j >= TEAMS || k > 0 || part > 0) ? 1u : 0u);
          umma_commit(vempty(s));
          umma_commit(o_done(t));
          if (!BESIDE && j + TEAMS < len) ok = scores(j + TEAMS);
        }
        n += len;
      }
      if (!ok) { atomicExch(status, WKB_STATUS_ATTN_WAIT); flags[1] = 1; }
    }
  } else if (warp < 2 + 4 * TEAMS) {      // (one more warp has no part: it makes the V warp another scheduler's)
    // ---------------- softmax teams ----------------
    const int team = (warp - 2) >> 2, quarter = warp & 3, a = quarter * 32 + lane, tid = threadIdx.x - 64;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16), s_col = lane_base + team * 128, p_col = s_col + P_BASE, o_col = lane_base + Shape<HD>::O_COL + team * HD;
    // scores in base 2; the sign of `scale` goes into the query; never 0, which would make NaN of a hidden key's -inf
    const float sc = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-37f);
    const bool negate = scale < 0.0f;
    bool ok = true;
    int n = 0, uses = 0, done[2] = {0, 0};      // blocks of the share, this team's blocks, either team's
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (ok && !__all_sync(0xffffffffu, bar_wait(bar, parity))) {
        ok = false;
        if (lane == 0) { atomicExch(status, WKB_STATUS_ATTN_WAIT); flags[1] = 1; }
      }
    };
    auto teams_sync = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(CREW) : "memory"); };      // every softmax thread passes every one of these
    auto teams_any = [&](bool mine) {      // the same barrier, and whether any thread says so
      uint32_t any;
      asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(any) : "r"((uint32_t)mine), "n"(CREW) : "memory");
      return any != 0u;
    };
    // The query operand (K-major, 128-byte swizzle).  The raw rows of the next piece come to the stage while this piece's
    // blocks are worked on (q_fetch), and the team that is not at work on the last block turns them into the operand's parts
    // and copies (q_put) as soon as that block's scores have been multiplied.  A thread reads back what it fetched itself.
    // Rows beyond the stage (f32, head_dim 128, rows 64 and up) come when the first ones have left it.  A single team reads
    // the rows where they lie, after its result is written.
    constexpr int CH = HD / 8, RAW = 16 * (QS == 1 ? 1 : 2), KEPT = SM::STAGE / RAW;      // chunks of 8 values a row, their bytes, chunks staged
    auto live_of = [&](const Piece& p) { return min(QROWS, p.w.t.nodes * group - p.rowblk * QROWS); };
    auto copies_of = [&](int live) { return live <= 32 ? 4 : live <= 64 ? 2 : 1; };
    auto q_at = [&](const Piece& p, int idx) {
      const int qr = idx / CH, c = idx % CH, ur = p.rowblk * QROWS + qr;
      return static_cast<const uint8_t*>(q) +
             ((i64)(p.w.t.row0 + (ur >> gshift)) * g.q_row_stride + ((i64)p.head * group + (ur & (group - 1))) * HD + c * 8) * (QS == 1 ? 2 : 4);
    };
    auto q_fetch = [&](const Piece& p, int from, int self, int threads) {
      const int n = min(live_of(p) * CH, from + KEPT);
#pragma unroll 1
      for (int idx = from + self; idx < n; idx += threads) {
        const uint8_t* src = q_at(p, idx);
#pragma unroll
        for (int k = 0; k < RAW; k += 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage_base + (uint32_t)(idx - from) * RAW + k), "l"(src + k) : "memory");
      }
    };
    auto q_put = [&](const Piece& p, int self, int threads, uint32_t bar) {
      const int live = live_of(p), copies = copies_of(live), crows = QROWS / copies;
      const uint32_t flip = negate ? 0x80008000u : 0u;
      for (int from = 0; from < crows * CH; from += KEPT) {
        if (TEAMS == 2 && from > 0) q_fetch(p, from, self, threads);
        asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 2
        for (int idx = from + self; idx < min(crows * CH, from + KEPT); idx += threads) {
          const int qr = idx / CH, c = idx % CH;
          float4 x[2] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
          if (qr < live) {
            const float4* raw_q = reinterpret_cast<const float4*>(TEAMS == 2 ? reinterpret_cast<const uint8_t*>(stage) + (idx - from) * RAW : q_at(p, idx));
            x[0] = raw_q[0];
            if (QS > 1) x[1] = raw_q[1];
          }
          uint32_t w[QS][4];
          if (QS == 1) { w[0][0] = f2u(x[0].x); w[0][1] = f2u(x[0].y); w[0][2] = f2u(x[0].z); w[0][3] = f2u(x[0].w); }
          else {
            float f[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
#pragma unroll
            for (int k = 0; k < QS; ++k)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                w[k][e] = pack_bf16(f[2 * e], f[2 * e + 1]);
                f[2 * e] -= u2f(w[k][e] << 16);
                f[2 * e + 1] -= u2f(w[k][e] & 0xffff0000u);
              }
          }
          const uint32_t dst = q_base + (uint32_t)(c >> 3) * SUB + (uint32_t)qr * 128u + (uint32_t)(((c & 7) ^ (qr & 7)) << 4);
#pragma unroll 1
          for (int cp = 0; cp < copies; ++cp)
#pragma unroll
            for (int k = 0; k < QS; ++k)
              asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + k * BLK + (uint32_t)(cp * crows) * 128u), "r"(w[k][0] ^ flip), "r"(w[k][1] ^ flip),
                           "r"(w[k][2] ^ flip), "r"(w[k][3] ^ flip)
                           : "memory");
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    Piece p, following;
    bool more = walk.next(g, slot, ctxs, row0s, following);
    if (more) {
      if (TEAMS == 2) q_fetch(following, 0, tid, CREW);
      q_put(following, tid, CREW, q_first);
      if (TEAMS == 2) teams_sync();      // the stage is free for the next piece's rows
    }
    while (more) {
      p = following;
      more = walk.next(g, slot, ctxs, row0s, following);
      const int len = p.b1 - p.b0;
      const int live = live_of(p), copies = copies_of(live), crows = QROWS / copies;
      const int copy = a / crows, r = a % crows;
      const bool puts = TEAMS == 2 && more && team == (len & 1);      // the team without the last block
      if (puts) q_fetch(following, 0, tid & 127, 128);
      // ---- the team's key blocks
      auto mask_of = [&](int row) { return mask + (i64)(p.w.t.row0 + ((p.rowblk * QROWS + row) >> gshift)) * g.mask_words; };
      const uint32_t* own_mask = mask_of(min(r, live - 1));
      const int words = (p.w.t.nodes + 31) >> 5;
      // which of the keys pos .. pos + 31 the row with this mask sees
      auto visible = [&](const uint32_t* mrow, int pos) -> uint32_t {
        uint32_t bits = low_bits((i64)p.w.t.ctx - pos);
        const i64 j = (i64)pos - p.w.t.ctx;
        if (j > -32) {
          if (j < 0) bits |= mrow[0] << (int)-j;
          else {
            const int w = (int)(j >> 5);
            const uint32_t lo = w < words ? mrow[w] : 0u, hi = w + 1 < words ? mrow[w + 1] : 0u;
            bits |= __funnelshift_r(lo, hi, (int)(j & 31));
          }
        }
        return bits & low_bits((i64)p.w.keys - pos);
      };
      float m = -INFINITY, l = 0.0f;      // m in base 2, the maximum in use
      // One block, 32 columns at a time in rolled loops: the kernel is short enough that first executions of unrolled code
      // (instruction fetches) took longer than the work.  The last columns of the first pass stay in registers.
      bool mend = false;      // results of this piece need mending: V holds something that is not finite
      const int chunks = 4 / copies, col0 = copy * chunks * 32;
      auto block = [&](auto masked_c, int j) {
        constexpr bool masked = decltype(masked_c)::value;      // some row does not see some key
        const int pos0 = (p.b0 + j) * KBLK + col0;
        float s[32];
        auto load = [&](int c) {
          tm_ld32(s_col + col0 + c * 32, reinterpret_cast<uint32_t*>(s));
          tm_ld_wait();
          if (masked) {
            const uint32_t bits = visible(own_mask, pos0 + c * 32);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[e] = (bits >> e) & 1u ? s[e] : -INFINITY;
          }
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          load(c);
          float b4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int e = 4; e < 28; e += 8)
#pragma unroll
            for (int k = 0; k < 4; ++k) b4[k] = fmaxf(fmaxf(b4[k], s[e + k]), s[e + 4 + k]);
          top = fmaxf(fmaxf(top, b4[0]), b4[1]);
          top = fmaxf(fmaxf(top, b4[2]), b4[3]);
          top = fmaxf(fmaxf(top, s[28]), s[29]);
          top = fmaxf(fmaxf(top, s[30]), s[31]);
        }
        top *= sc;
        const bool move = top > m + 8.0f || (m == -INFINITY && top > -INFINITY);
        if (__any_sync(0xffffffffu, move)) {
          const float next = move ? top : m;
          const float corr = move ? ex2(m - next) : 1.0f;      // 0 when nothing had been seen
          if (j >= TEAMS) {      // the accumulator holds this team's earlier blocks
            wait(o_done(team), (uses - 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tm_ld32(o_col + c, o);
              tm_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = f2u(u2f(o[e]) * corr);
              tm_st32(o_col + c, o);
            }
          }
          l *= corr;
          m = next;
        }
        const float m_use = m == -INFINITY ? 0.0f : m;
        if (BESIDE && j > 0) {      // the last block's P V has read P
          wait(o_done(team), (uses - 1) & 1);
          tc_fence_after();
        }
#pragma unroll 1
        for (int c = chunks - 1;; ) {
          uint64_t l2[2] = {two(0.0f, 0.0f), two(0.0f, 0.0f)};
          uint32_t pk[32];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float p0, p1;
            of_two(fma_two(two(s[e], s[e + 1]), two(sc, sc), two(-m_use, -m_use)), p0, p1);
            p0 = ex2(p0);
            p1 = ex2(p1);
            l2[(e >> 1) & 1] = add_two(l2[(e >> 1) & 1], two(p0, p1));
            pk[e >> 1] = pack_bf16(p0, p1);
            if (PS == 2) pk[16 + (e >> 1)] = pack_bf16(p0 - u2f(pk[e >> 1] << 16), p1 - u2f(pk[e >> 1] & 0xffff0000u));
          }
          if (PS == 2) tm_st32(p_col + (copy * chunks + c) * P_CHUNK, pk);
          else tm_st16(p_col + (copy * chunks + c) * P_CHUNK, pk);
          float la, lb;
          of_two(add_two(l2[0], l2[1]), la, lb);
          l += la + lb;
          if (--c < 0) break;
          load(c);
        }
        if (copies > 1 && (!BESIDE || j == 0)) {      // zeros for the other copies' keys; beside S they stay
          uint32_t zero[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) zero[e] = 0u;
#pragma unroll 1
          for (int c = 0; c < 4; ++c)
            if (c / chunks != copy) {
              if (PS == 2) tm_st32(p_col + c * P_CHUNK, zero);
              else tm_st16(p_col + c * P_CHUNK, zero);
            }
        }
      };
      for (int j = team; j < len; j += TEAMS) {
        wait(s_full(team), uses & 1);
        tc_fence_after();
        const bool masked = (p.b0 + j + 1) * KBLK > p.w.t.ctx;
        if (masked) block(std::true_type(), j);
        else block(std::false_type(), j);
        // V of keys that some row does not see
        if (masked) {
          const int i = n + j, sl = i % NV, row = quarter * 32 + lane;
          wait(vfull(sl), (i / NV) & 1);
          const uint32_t vrow = v_ring + sl * BLK + (uint32_t)(row >> 3) * Layout<HD>::GROUP + (uint32_t)(row & 7) * 128u;
          auto piece_at = [&](int k) { return vrow + (uint32_t)(k >> 3) * Layout<HD>::HALF + (uint32_t)(((k & 7) ^ (row & 7)) << 4); };
          uint32_t bad = 0u;
#pragma unroll 1
          for (int k = 0; k < 8 * NSUB; k += 8) {
            uint32_t w[8][4];
#pragma unroll
            for (int c = 0; c < 8; ++c)
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[c][0]), "=r"(w[c][1]), "=r"(w[c][2]), "=r"(w[c][3]) : "r"(piece_at(k + c)));
#pragma unroll
            for (int c = 0; c < 8; ++c) bad |= not_finite2(w[c][0]) | not_finite2(w[c][1]) | not_finite2(w[c][2]) | not_finite2(w[c][3]);
          }
          if (bad) {
#pragma unroll 1
            for (int k = 0; k < 32 * NSUB; ++k) {
              const uint32_t at = piece_at(k >> 2) + (uint32_t)(k & 3) * 4u;
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
              const uint32_t b = not_finite2(w);
              w &= ((b & 0x8000u) ? 0u : 0xffffu) | ((b & 0x80000000u) ? 0u : 0xffff0000u);
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          const uint32_t which = __ballot_sync(0xffffffffu, bad != 0u && (p.b0 + j) * KBLK + row < p.w.keys);
          if (lane == 0) bad_keys[(p.b0 + j - p.w.t.ctx / KBLK) * 4 + quarter] = which;
          mend |= which != 0u;
        }
        tm_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(team));
        ++uses;
      }
      n += len;

      // ---- the result: the teams' accumulators lie in the same lanes and are added in registers; the copies lie in other
      // lanes and are added through shared memory, 64 columns at a time
      done[0] += TEAMS == 2 ? (len + 1) >> 1 : len;
      done[1] += TEAMS == 2 ? len >> 1 : 0;
      if (puts) {
        wait(s_full(team ^ 1), (done[team ^ 1] - 1) & 1);      // the last product with this piece's query is done
        q_put(following, tid & 127, 128, q_full);
      }
      ml_s[team * QROWS + a] = make_float2(team < len ? m : -INFINITY, team < len ? l : 0.0f);
      teams_sync();
      const bool both = TEAMS == 2 && len > 1;      // team 1 had a block
      wait(o_done(0), (done[0] - 1) & 1);
      if (both) wait(o_done(1), (done[1] - 1) & 1);
      tc_fence_after();
      float m_all = -INFINITY, l_all = 0.0f;
#pragma unroll 4
      for (int i = r; i < (both ? 2 : 1) * QROWS; i += crows) m_all = fmaxf(m_all, ml_s[i].x);      // copies of team 0, then of team 1
      const float m_use = m_all == -INFINITY ? 0.0f : m_all;
#pragma unroll 4
      for (int i = r; i < (both ? 2 : 1) * QROWS; i += crows) {
        const float2 v = ml_s[i];
        l_all += v.y * ex2(v.x - m_use);
      }
      const bool whole = len == p.w.blocks, fine = flags[1] == 0;
      const float inv = !whole ? 1.0f : l_all != 0.0f ? 1.0f / l_all : 0.0f;      // a unit in one piece is normalised here
      const float w0 = ex2(ml_s[a].x - m_use) * inv, w1 = both ? ex2(ml_s[QROWS + a].x - m_use) * inv : 0.0f;
      // a share's piece that begins the share is its even one; a later one that it does not finish is its odd one
      const int piece = p.unit_start + p.b0 == (int)blockIdx.x * share ? 2 * blockIdx.x : 2 * blockIdx.x + 1;
      if (!whole && fine && team == 0 && copy == 0 && r < live) scr.ml[(i64)piece * scr.rows + r] = make_float2(m_all, l_all);
      const bool staged = copies > 1;
      auto out_at = [&](int row) {      // of column 0
        const int ur = p.rowblk * QROWS + row;
        return whole ? (i64)(p.w.t.row0 + (ur >> gshift)) * g.out_row_stride + ((i64)p.head * group + (ur & (group - 1))) * HD
                     : ((i64)piece * scr.rows + row) * HD;
      };
      auto put = [&](i64 at, const float4& v) {
        if (!whole) *reinterpret_cast<float4*>(scr.o + at) = v;
        else if (out_dtype == 0) *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
        else *reinterpret_cast<uint2*>(static_cast<u16*>(out) + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      };
#pragma unroll 1
      for (int c0 = 0; c0 < HD; c0 += 64) {
#pragma unroll 1
        for (int half = team; half < 2; half += TEAMS) {
          const int col = c0 + half * 32;
          uint32_t o[32];
          tm_ld32(lane_base + Shape<HD>::O_COL + col, o);
          if (both) {
            uint32_t o1[32];
            tm_ld32(lane_base + Shape<HD>::O_COL + HD + col, o1);
            tm_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = f2u(ffma(u2f(o1[e]), w1, u2f(o[e]) * w0));
          } else {
            tm_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = f2u(u2f(o[e]) * w0);
          }
          uint64_t zero = two(0.0f, 0.0f);      // stays 0 unless an element is not finite
#pragma unroll
          for (int e = 0; e < 32; e += 2) zero = fma_two(two(u2f(o[e]), u2f(o[e + 1])), two(0.0f, 0.0f), zero);
          float zero_a, zero_b;
          of_two(zero, zero_a, zero_b);
          mend |= !(zero_a + zero_b == 0.0f);
          if (staged) {
            float4* d = reinterpret_cast<float4*>(stage + a * 64 + half * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e ^ (a & 7)] = make_float4(u2f(o[4 * e]), u2f(o[4 * e + 1]), u2f(o[4 * e + 2]), u2f(o[4 * e + 3]));
          } else if (r < live && fine) {
            const i64 at = out_at(r) + col;
            if (whole && out_dtype == 1) {
              uint4* d = reinterpret_cast<uint4*>(static_cast<u16*>(out) + at);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                d[e] = make_uint4(pack_bf16(u2f(o[8 * e]), u2f(o[8 * e + 1])), pack_bf16(u2f(o[8 * e + 2]), u2f(o[8 * e + 3])),
                                  pack_bf16(u2f(o[8 * e + 4]), u2f(o[8 * e + 5])), pack_bf16(u2f(o[8 * e + 6]), u2f(o[8 * e + 7])));
            } else {
              float4* d = reinterpret_cast<float4*>((whole ? static_cast<float*>(out) : scr.o) + at);
#pragma unroll
              for (int e = 0; e < 8; ++e) d[e] = make_float4(u2f(o[4 * e]), u2f(o[4 * e + 1]), u2f(o[4 * e + 2]), u2f(o[4 * e + 3]));
            }
          }
        }
        if (!staged) continue;
        teams_sync();
        // a thread keeps its four columns and goes down the rows, STEP at a time (a multiple of the group)
        constexpr int STEP = CREW / 16;
        const int c4 = tid & 15, first = tid >> 4;
        const i64 down = whole ? (i64)(STEP >> gshift) * g.out_row_stride : (i64)STEP * HD;
        i64 at = out_at(first) + c0 + c4 * 4;
        auto part = [&](int x) { return *reinterpret_cast<const float4*>(stage + x * 64 + ((c4 ^ (x & 7)) << 2)); };
        auto add = [](float4& a, const float4& b) { a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; };
#pragma unroll 2
        for (int row = first; row < live; row += STEP, at += down) {
          float4 v = part(row);
          if (copies > 1) add(v, part(row + crows));
          if (copies > 2) { add(v, part(row + 2 * crows)); add(v, part(row + 3 * crows)); }
          if (fine) put(at, v);
        }
        if (c0 + 64 < HD) teams_sync();
      }
      tc_fence_before();
      if (teams_any(mend)) {
        // Rare: V holds a NaN or an infinity.  The sum of those elements over the keys that a row sees is then its result
        // (a row with a NaN score stays NaN).  The whole blocks of the context are everybody's: their columns' kinds are
        // gathered once, 16 keys at a time, and the keys of the other blocks are known: 2.5 ms for 150 000 keys in one
        // piece (which the products take 1.7 to 3.6 ms for), so the other warps' waits of a second do not run out.
        constexpr int CH8 = HD / 8;
        uint32_t* kinds_s = reinterpret_cast<uint32_t*>(stage);      // [HD / 8]
        if (tid < CH8) kinds_s[tid] = 0u;
        teams_sync();
        auto kinds_at = [&](int pos, int c) {
          const uint32_t page = block_table[(i64)p.w.t.slot * g.mbps + (pos >> g.page_shift)];
          if (page >= (uint64_t)g.num_pages) return 0u;
          return kinds_of(*reinterpret_cast<const uint4*>(vcache + (((i64)page * g.kv_heads + p.head) * g.page_tokens + (pos & (g.page_tokens - 1))) * HD + c * 8));
        };
        const int shared_end = min(p.b1, p.w.t.ctx / KBLK) * KBLK;
        uint32_t kinds = 0u;
#pragma unroll 4
        for (int pos = p.b0 * KBLK + tid / CH8; pos < shared_end; pos += CREW / CH8) kinds |= kinds_at(pos, tid % CH8);
        if (kinds) atomicOr(&kinds_s[tid % CH8], kinds);
        teams_sync();
#pragma unroll 1
        for (int it = tid; it < live * CH8; it += CREW) {
          const int row = it / CH8, c = it % CH8;
          bool nan = false;
#pragma unroll 1
          for (int i = row; i < (both ? 2 : 1) * QROWS; i += crows) nan |= ml_s[i].y != ml_s[i].y;
          kinds = kinds_s[c];
#pragma unroll 1
          for (int w = 0; w < 12; ++w) {
            const int blk = p.w.t.ctx / KBLK + (w >> 2);
            if (blk < p.b0 || blk >= p.b1) continue;
            const int pos = blk * KBLK + (w & 3) * 32;
            uint32_t bits = bad_keys[w];
            if (bits) bits &= visible(mask_of(row), pos);
            for (; bits; bits &= bits - 1) kinds |= kinds_at(pos + __ffs(bits) - 1, c);
          }
          if (nan || !fine) continue;
          const i64 at = out_at(row) + c * 8;
#pragma unroll 1
          for (int e = 0; e < 8; ++e) {
            const uint32_t kind = (kinds >> (4 * e)) & 7u;
            if (!kind) continue;
            if (!whole) scr.o[at + e] = kind_sum(kind);
            else if (out_dtype == 0) static_cast<float*>(out)[at + e] = kind_sum(kind);
            else static_cast<u16*>(out)[at + e] = f32_to_bf16_bits(kind_sum(kind));
          }
        }
        teams_sync();
      }
      // the accumulators, the stage and ml_s are free
      if (TEAMS == 1 && more) q_put(following, tid, CREW, q_full);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && flags[1]) scr.start[blockIdx.x].total = -1;
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape<HD>::TM_COLS) : "memory");
  }
}

// Block (c, rows): if the boundary before share c falls inside a unit, and is the first one that does, join the unit's
// pieces (in key order) for these rows and write the result.  A row is HD / 4 lanes, which first share the pieces' (m, l)
// out among them, so that the trips to L2 do not add up with the number of pieces.
template <int HD>
__global__ void __launch_bounds__(256) tree_attn_join_kernel(void* __restrict__ out, int out_dtype, Geo g, Scratch scr) {
  pdl_wait();
  pdl_trigger();
  const int c = blockIdx.x + 1;
  const ShareStart st = scr.start[c];
  const int x = c * st.share;
  if (x >= st.total || st.unit_len == 0 || x <= st.unit_start || x - st.share > st.unit_start) return;
  const int last = (st.unit_start + st.unit_len - 1) / st.share, group = g.q_heads / g.kv_heads;
  constexpr int LANES = HD / 4;
  const int lane = threadIdx.x % LANES, row = blockIdx.y * (256 / LANES) + threadIdx.x / LANES, col = lane * 4;
  const unsigned team = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
  if (row >= st.live) return;      // (all lanes of a row)
  auto piece = [&](int k) { return (i64)(k * st.share >= st.unit_start ? 2 * k : 2 * k + 1) * scr.rows + row; };
  float m = -INFINITY;
  bool failed = false;
  for (int k = c - 1 + lane; k <= last; k += LANES) {
    m = fmaxf(m, scr.ml[piece(k)].x);
    failed |= scr.start[k].total < 0;
  }
  if (__any_sync(team, failed)) return;      // not all pieces were written
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(team, m, o, LANES));
  const float use = m == -INFINITY ? 0.0f : m;
  float l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k0 = c - 1; k0 <= last; k0 += LANES) {
    const int n = min(LANES, last + 1 - k0);
    const float2 ml = lane < n ? scr.ml[piece(k0 + lane)] : make_float2(-INFINITY, 0.0f);
    const float w = ex2(ml.x - use);
    l += ml.y * w;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float wk = __shfl_sync(team, w, k, LANES);
      const float4 v = *reinterpret_cast<const float4*>(scr.o + piece(k0 + k) * HD + col);
      // what is not finite counts as it is: its piece's weight may be 0 in f32, and 0 x inf is NaN
      auto add = [&](float& to, float x) { to = ffma(x, fabsf(x) <= 3.402823466e+38f ? wk : 1.0f, to); };
      add(o.x, v.x); add(o.y, v.y); add(o.z, v.z); add(o.w, v.w);
    }
  }
  for (int k = LANES / 2; k > 0; k >>= 1) l += __shfl_xor_sync(team, l, k, LANES);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  o.x *= inv; o.y *= inv; o.z *= inv; o.w *= inv;
  const int ur = st.rowblk * QROWS + row;
  const i64 at = (i64)(st.row0 + ur / group) * g.out_row_stride + ((i64)st.head * group + ur % group) * HD + col;
  if (out_dtype == 0) *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = o;
  else *reinterpret_cast<uint2*>(static_cast<u16*>(out) + at) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
}

// One layer's cache as [64-dim half][num_pages * kv_heads * page_tokens][64] of bf16; box = all halves of box_rows tokens
// of one head, 128-byte swizzle.  Rows past the cache read as zeros.
inline int cache_map(CUtensorMap* map, const void* cache, i64 rows, i64 head_dim, int box_rows) {
  EncodeTiledFn enc = get_encode();
  if (!enc) return (int)cudaErrorNotSupported;
  cuuint64_t dims[3] = {64, (cuuint64_t)rows, (cuuint64_t)(head_dim / 64)};
  cuuint64_t strides[2] = {(cuuint64_t)head_dim * 2, 128};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, (cuuint32_t)(head_dim / 64)};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <int HD, int QS, int PS>
int launch_tc(const void* q, const void* kc, const void* vc, const uint32_t* bt, const int* slot, const int* ctx, const int* row0, const uint32_t* mask,
              void* out, int out_dtype, const Geo& g, float scale, void* scratch, cudaStream_t st) {
  const int box_rows = Layout<HD>::box_rows(g.page_tokens);
  const i64 cache_rows = g.num_pages * g.kv_heads * g.page_tokens;
  CUtensorMap mk, mv;
  int rc = cache_map(&mk, kc, cache_rows, HD, box_rows);
  if (rc) return rc;
  rc = cache_map(&mv, vc, cache_rows, HD, box_rows);
  if (rc) return rc;
  int* status = gemm_status_word();
  if (!status) return (int)cudaErrorMemoryAllocation;
  auto kern = tree_attn_tc_kernel<HD, QS, PS>;
  using SH = Shape<HD>;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<HD, QS>::BYTES);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev & 63] = true;
  }
  const int group = g.q_heads / g.kv_heads;
  const Scratch scr = carve(scratch, g.max_nodes, group, SH::SHARES);
  cudaError_t e = launch_pdl(kern, SH::SHARES, SH::THREADS, (size_t)TcSmem<HD, QS>::BYTES, st, mk, mv, q, (const u16*)vc, bt, slot, ctx, row0, mask, out,
                             out_dtype, g, scale, scr, status);
  if (e != cudaSuccess || !g.split) return (int)e;
  const int rows_per = 256 / (HD / 4);
  return (int)launch_pdl(tree_attn_join_kernel<HD>, dim3(SH::SHARES - 1, (unsigned)((scr.rows + rows_per - 1) / rows_per)), 256, 0, st, out, out_dtype, g, scr);
}

}  // namespace tree
}  // namespace wkb
