// Attention of draft trees over the paged cache.  A tree hangs off a sequence of `ctx` committed tokens; its nodes' K / V
// lie at positions ctx, ctx + 1, ... of the sequence's pages, in node order, and a node sees the committed tokens and the
// nodes that its mask names (itself and its ancestors, in a tree):
//
//   out_r = sum_p softmax_p(scale * q_r . k_p) v_p   over  p < ctx  and  p = ctx + j, j < nodes, bit j of mask_r
//
// No counterpart in the reference, whose decode attention takes one token a sequence
// (crates/wukong_codegen_gpu/src/paged_attention.rs:395-534).
#include "common.cuh"
#include "wkb_device.h"

namespace wkb {
namespace tree {

constexpr int MAX_NODES = 256, MAX_TREES = 4096;

struct Geo {
  int rows, n_trees, max_nodes, mask_words, q_heads, kv_heads, page_tokens, page_shift, mbps;
  i64 num_pages, q_row_stride, out_row_stride;
  int split;      // units may be cut into pieces (tensor-core kernel)
};
struct TreeRef {
  int row0, nodes, ctx, slot;
};
// The tree's extents, clamped to what the arguments cover; nodes 0 for a tree that is switched off (slot or ctx < 0).
__device__ __forceinline__ TreeRef tree_ref(const Geo& g, const int* __restrict__ slot, const int* __restrict__ ctx, const int* __restrict__ row0, int t) {
  TreeRef r;
  r.slot = slot[t];
  r.ctx = ctx[t];
  const int a = min(max(row0[t], 0), g.rows), b = min(max(row0[t + 1], a), g.rows);
  r.row0 = a;
  r.nodes = r.slot < 0 || r.ctx < 0 ? 0 : min(b - a, g.max_nodes);
  return r;
}

// For pages of 4 tokens, which fill no swizzle atom of the tensor-core kernel's operands.  One warp per (row, query head),
// bound by the latency of its loads (5.7 ms where the tensor-core kernel takes 0.12, 64 Llama-shape trees).  32 keys at a time: a lane scores one key, then the lanes turn to the head's
// dimensions and add the visible keys' values one after the other.  A key that a row does not see is skipped, so
// whatever its V holds stays out of the sum.
template <int HD>
__global__ void __launch_bounds__(256) tree_attn_rows_kernel(const void* __restrict__ q, int q_dtype, const u16* __restrict__ kc, const u16* __restrict__ vc,
                                                             const uint32_t* __restrict__ block_table, const int* __restrict__ slot,
                                                             const int* __restrict__ ctxs, const int* __restrict__ row0,
                                                             const uint32_t* __restrict__ mask, void* __restrict__ out, int out_dtype, Geo g,
                                                             float scale_log2e) {
  pdl_wait();
  pdl_trigger();
  __shared__ float q_s[8][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const i64 items = (i64)g.rows * g.q_heads;
  for (i64 it = (i64)blockIdx.x * 8 + warp; it < items; it += (i64)gridDim.x * 8) {
    const int row = (int)(it / g.q_heads), h = (int)(it % g.q_heads), kvh = h / (g.q_heads / g.kv_heads);
    int lo = 0, hi = g.n_trees;                  // the last tree that starts at or before this row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (row0[mid] <= row) lo = mid; else hi = mid;
    }
    const TreeRef t = tree_ref(g, slot, ctxs, row0, lo);
    if (row < t.row0 || row >= t.row0 + t.nodes) continue;
    __syncwarp();
    for (int d = lane; d < HD; d += 32) {
      const i64 at = (i64)row * g.q_row_stride + (i64)h * HD + d;
      q_s[warp][d] = (q_dtype == 0 ? static_cast<const float*>(q)[at] : bf16_bits_to_f32(static_cast<const u16*>(q)[at])) * scale_log2e;
    }
    __syncwarp();
    const uint32_t* bt = block_table + (i64)t.slot * g.mbps;
    const uint32_t* mrow = mask + (i64)row * g.mask_words;
    const i64 keys = min((i64)t.ctx + t.nodes, (i64)g.mbps * g.page_tokens);
    float m = -INFINITY, l = 0.0f, acc[HD / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) acc[e] = 0.0f;
    for (i64 p0 = 0; p0 < keys; p0 += 32) {
      const i64 p = p0 + lane;
      bool seen = p < keys;
      if (seen && p >= t.ctx) {
        const int j = (int)(p - t.ctx);
        seen = (mrow[j >> 5] >> (j & 31)) & 1u;
      }
      i64 off = -1;
      float s = -INFINITY;
      if (seen) {
        const uint32_t page = bt[p >> g.page_shift];
        s = 0.0f;
        if (page < (uint64_t)g.num_pages) {      // an entry past the cache reads as a page of zeros
          off = (((i64)page * g.kv_heads + kvh) * g.page_tokens + (p & (g.page_tokens - 1))) * HD;
          const uint4* k4 = reinterpret_cast<const uint4*>(kc + off);
#pragma unroll 4
          for (int c = 0; c < HD / 8; ++c) {
            const uint4 w = k4[c];
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s = ffma(q_s[warp][c * 8 + 2 * e], u2f(ws[e] << 16), s);
              s = ffma(q_s[warp][c * 8 + 2 * e + 1], u2f(ws[e] & 0xffff0000u), s);
            }
          }
        }
      }
      unsigned todo = __ballot_sync(0xffffffffu, seen);
      if (!todo) continue;
      const float m_new = fmaxf(m, warp_max(s)), m_use = m_new == -INFINITY ? 0.0f : m_new;
      const float corr = exp2f(m - m_use), pr = seen ? exp2f(s - m_use) : 0.0f;
      l = l * corr + warp_sum(pr);
      m = m_new;
#pragma unroll
      for (int e = 0; e < HD / 32; ++e) acc[e] *= fabsf(acc[e]) <= 3.402823466e+38f ? corr : 1.0f;      // an infinity of V stays one where corr is 0 ...
      while (todo) {
        const int b = __ffs(todo) - 1;
        todo &= todo - 1;
        const float pb = __shfl_sync(0xffffffffu, pr, b);
        const i64 ob = __shfl_sync(0xffffffffu, off, b);
        if (ob < 0) continue;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) {
          const float x = bf16_bits_to_f32(vc[ob + e * 32 + lane]);
          acc[e] = ffma(fabsf(x) <= 3.402823466e+38f ? pb : 1.0f, x, acc[e]);      // ... or the weight
        }
      }
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;      // a row that sees nothing: zeros
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) {
      const i64 at = (i64)row * g.out_row_stride + (i64)h * HD + e * 32 + lane;
      if (out_dtype == 0) static_cast<float*>(out)[at] = acc[e] * inv;
      else static_cast<u16*>(out)[at] = f32_to_bf16_bits(acc[e] * inv);
    }
  }
}

}  // namespace tree
}  // namespace wkb

#include "tree_attn_tc.cuh"

using namespace wkb;

extern "C" {

i64 wkb_paged_attn_tree_scratch_bytes(i64 max_nodes, i64 q_heads, i64 kv_heads, i64 head_dim) {
  if (max_nodes <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0) return 0;
  if (max_nodes > 0x7fffffff || q_heads > 0x7fffffff || head_dim > 0x7fffffff) return 0;
  return tree::scratch_bytes(max_nodes, q_heads / kv_heads, head_dim, tree::shares_of(head_dim));
}

int wkb_paged_attn_tree(const void* q, int q_dtype, i64 q_row_stride, const void* kcache, const void* vcache, i64 num_pages, const uint32_t* block_table,
                        const int* tree_slot, const int* tree_ctx, const int* tree_row0, const uint32_t* tree_mask, i64 mask_words, void* out,
                        int out_dtype, i64 out_row_stride, i64 rows, i64 n_trees, i64 max_nodes, i64 q_heads, i64 kv_heads, i64 head_dim,
                        i64 page_tokens, i64 max_blocks_per_seq, float scale, void* scratch, i64 scratch_bytes, void* stream) {
  if (rows <= 0 || n_trees <= 0) return 0;
  // every extent first, so that no product below wraps around (and no row's address in the kernels)
  if (rows > 0x7fffffff || q_heads > 0x7fffffff || max_blocks_per_seq > 0x7fffffff || mask_words > 0x7fffffff || q_row_stride > (i64)1 << 31 ||
      out_row_stride > (i64)1 << 31)
    return (int)cudaErrorInvalidValue;
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0) return (int)cudaErrorInvalidValue;
  const i64 group = q_heads / kv_heads;
  if ((group != 1 && group != 2 && group != 4 && group != 8) || (head_dim != 64 && head_dim != 128)) return (int)cudaErrorInvalidValue;
  if (page_tokens < 4 || page_tokens > 65536 || (page_tokens & (page_tokens - 1)) != 0) return (int)cudaErrorInvalidValue;   // power of two, >= 4
  if (max_nodes < 1 || max_nodes > tree::MAX_NODES || n_trees > tree::MAX_TREES || mask_words * 32 < max_nodes) return (int)cudaErrorInvalidValue;
  if (max_blocks_per_seq < 1 || max_blocks_per_seq * page_tokens > 0x7fffff00 || num_pages < 1 || rows * q_heads > 0x7fffffffff)
    return (int)cudaErrorInvalidValue;
  if (num_pages > 0x7fffff00 / (kv_heads * page_tokens)) return (int)cudaErrorInvalidValue;
  if ((q_dtype != 0 && q_dtype != 1) || (out_dtype != 0 && out_dtype != 1)) return (int)cudaErrorInvalidValue;
  if (!(fabsf(scale) <= 1e38f)) return (int)cudaErrorInvalidValue;      // (NaN; in base 2 it has to be finite)
  if (q_row_stride < 0 || out_row_stride < 0 || (rows > 1 && out_row_stride < q_heads * head_dim)) return (int)cudaErrorInvalidValue;      // result rows do not overlap
  if (q_row_stride % 8 != 0 || out_row_stride % 8 != 0) return (int)cudaErrorMisalignedAddress;
  if (((((uintptr_t)q) | ((uintptr_t)kcache) | ((uintptr_t)vcache) | ((uintptr_t)out) | ((uintptr_t)scratch)) & 15) != 0) return (int)cudaErrorMisalignedAddress;
  if (!scratch || scratch_bytes < wkb_paged_attn_tree_scratch_bytes(max_nodes, q_heads, kv_heads, head_dim)) return (int)cudaErrorInvalidValue;
  int page_shift = 0;
  while ((1 << page_shift) < page_tokens) ++page_shift;
  tree::Geo g{(int)rows, (int)n_trees, (int)max_nodes, (int)mask_words, (int)q_heads, (int)kv_heads, (int)page_tokens, page_shift, (int)max_blocks_per_seq,
              num_pages, q_row_stride, out_row_stride, 1};
  cudaStream_t st = as_stream(stream);
  if (page_tokens >= 8) {      // a page of 8 tokens fills whole swizzle atoms of the operand
    const i64 row_blocks = (max_nodes * group + tree::QROWS - 1) / tree::QROWS, key_blocks = (max_blocks_per_seq * page_tokens + tree::KBLK - 1) / tree::KBLK + tree::UNIT_COST;
    if ((double)n_trees * (double)kv_heads * (double)row_blocks * (double)key_blocks > 2147000000.0) return (int)cudaErrorInvalidValue;
    // Up to one unit a CTA and 6 blocks a unit: 5 more blocks in a row take 3.5 (head_dim 64) to 5 us, a second kernel 3.3 us
    // and its launch.
    if (n_trees * kv_heads * row_blocks <= tree::shares_of(head_dim) && key_blocks - tree::UNIT_COST <= 6) g.split = 0;
#define WKB_TREE_CASE(HD_, QS_, PS_)                                   \
  if (head_dim == HD_ && (q_dtype == 0 ? 2 : 1) == QS_ && (out_dtype == 0 ? 2 : 1) == PS_) \
    return tree::launch_tc<HD_, QS_, PS_>(q, kcache, vcache, block_table, tree_slot, tree_ctx, tree_row0, tree_mask, out, out_dtype, g, scale, scratch, st);
    WKB_TREE_CASE(64, 1, 1) WKB_TREE_CASE(64, 1, 2) WKB_TREE_CASE(64, 2, 1) WKB_TREE_CASE(64, 2, 2)
    WKB_TREE_CASE(128, 1, 1) WKB_TREE_CASE(128, 1, 2) WKB_TREE_CASE(128, 2, 1) WKB_TREE_CASE(128, 2, 2)
#undef WKB_TREE_CASE
  }
  const i64 blocks = (rows * q_heads + 7) / 8;
  const unsigned grid = (unsigned)(blocks < (i64)WKB_SM_COUNT * 64 ? blocks : (i64)WKB_SM_COUNT * 64);
  auto kern = head_dim == 64 ? tree::tree_attn_rows_kernel<64> : tree::tree_attn_rows_kernel<128>;
  return (int)launch_pdl(kern, grid, 256, 0, st, q, q_dtype, (const u16*)kcache, (const u16*)vcache, block_table, tree_slot, tree_ctx,
                         tree_row0, tree_mask, out, out_dtype, g, scale * 1.4426950408889634f);
}

}  // extern "C"
