// What follows the target model's logits in a speculative decoding step: temperature softmax of the vocabulary rows,
// verification of the drafted tokens against the target's probabilities, and the commit of the accepted nodes' K / V.
// Selection and sampling share the conventions of the reference's categorical draw (crates/wukong_runtime/src/topk.rs:1-136):
// weights that are not positive and finite count as zero, masses are summed in f64, a random number is clamped to [0, 1].
#include "common.cuh"
#include "wkb_device.h"

namespace wkb {
namespace verify {

constexpr int MAX_NODES = 256;

// ---- temperature softmax --------------------------------------------------------------------------------------------
__device__ __forceinline__ float load_logit(const void* x, int dtype, i64 at) {
  return dtype == 0 ? static_cast<const float*>(x)[at] : bf16_bits_to_f32(static_cast<const u16*>(x)[at]);
}
// One CTA per row: maximum (and its lowest column), sum, write.
__global__ void __launch_bounds__(512) token_probs_kernel(const void* __restrict__ x, int dtype, i64 ld, const float* __restrict__ temperature,
                                                          float* __restrict__ out, i64 ld_out, i64 cols) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red_v[16];
  __shared__ int red_i[16];
  const i64 row = blockIdx.x;
  const float temp = temperature ? temperature[row] : 1.0f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float best = -INFINITY;
  int at = 0x7fffffff;
  bool nan = false;
  for (i64 i = threadIdx.x; i < cols; i += 512) {
    const float v = load_logit(x, dtype, row * ld + i);
    nan |= v != v;
    if (v > best || (v == best && (int)i < at)) { best = v; at = (int)i; }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (v > best || (v == best && i < at)) { best = v; at = i; }
  }
  if (lane == 0) { red_v[warp] = best; red_i[warp] = at; }
  nan = __syncthreads_or(nan);
  best = red_v[0]; at = red_i[0];
  for (int w = 1; w < 16; ++w)
    if (red_v[w] > best || (red_v[w] == best && red_i[w] < at)) { best = red_v[w]; at = red_i[w]; }
  __syncthreads();
  const float scale = fminf(1.4426950408889634f / temp, 3.402823466e+38f);      // finite, so that the maximum keeps weight 1
  float sum = 0.0f;
  if (temp > 0.0f) {
    for (i64 i = threadIdx.x; i < cols; i += 512) sum += exp2f((load_logit(x, dtype, row * ld + i) - best) * scale);
    sum = warp_sum(sum);
    if (lane == 0) red_v[warp] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < 16; ++w) sum += red_v[w];
  }
  for (i64 i = threadIdx.x; i < cols; i += 512) {
    float p;
    if (nan || temp != temp) p = NAN;
    else if (best == -INFINITY) p = 0.0f;                 // every token is ruled out
    else if (temp > 0.0f) p = exp2f((load_logit(x, dtype, row * ld + i) - best) * scale) / sum;
    else p = (int)i == at ? 1.0f : 0.0f;
    out[row * ld_out + i] = p;
  }
}

// ---- verification ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ double weight(float v) { return v > 0.0f && v <= 3.402823466e+38f ? (double)v : 0.0; }

// One CTA per tree.  Thread 0 walks the tree; a pass over the vocabulary sums the mass that is left.
__global__ void __launch_bounds__(512) tree_verify_kernel(const float* __restrict__ probs, i64 ld_p, const float* __restrict__ draft, i64 ld_q,
                                                          const int* __restrict__ token, const int* __restrict__ parent, const int* __restrict__ row0,
                                                          int rows, int cols, int max_nodes, const float* __restrict__ u_node,
                                                          const float* __restrict__ u_final, int* __restrict__ path, int* __restrict__ tokens,
                                                          int* __restrict__ n_path, int max_path) {
  pdl_wait();
  pdl_trigger();
  __shared__ int tok_s[MAX_NODES], par_s[MAX_NODES], tried[MAX_NODES], path_s[MAX_NODES];
  __shared__ double z_s[MAX_NODES + 1], part[16];
  __shared__ int cur, tries, len, more;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int a = min(max(row0[t], 0), rows), nodes = min(min(max(row0[t + 1], a), rows) - a, max_nodes);
  for (int i = threadIdx.x; i < max_path; i += 512) { path[(i64)t * max_path + i] = -1; tokens[(i64)t * max_path + i] = -1; }
  if (nodes <= 0) {
    if (threadIdx.x == 0) n_path[t] = 0;
    return;
  }
  for (int i = threadIdx.x; i < nodes; i += 512) { tok_s[i] = token[a + i]; par_s[i] = parent[a + i]; }
  if (threadIdx.x == 0) { cur = 0; tries = 0; len = 1; path_s[0] = 0; z_s[0] = 1.0; }
  __syncthreads();
  // what is left of column i's weight after the `tries` rejections below node cur
  auto left = [&](int i) -> double {
    double r = weight(probs[(i64)(a + cur) * ld_p + i]);
    if (draft) {
      const double q = tries ? weight(draft[(i64)(a + cur) * ld_q + i]) : 0.0;
      for (int k = 0; k < tries; ++k) r = fmax(r - z_s[k] * q, 0.0);
    } else {
      for (int k = 0; k < tries; ++k)
        if (tried[k] == i) r = 0.0;
    }
    return r;
  };
  const int seg = ((cols + 15) / 16 + 31) / 32 * 32;      // a warp's columns
  auto sums = [&]() {
    double s = 0.0;
    for (int i = warp * seg + lane; i < min(cols, (warp + 1) * seg); i += 32) s += left(i);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) part[warp] = s;
    __syncthreads();
  };
  int next = 1;
  bool summed = false;
  for (;;) {
    if (threadIdx.x == 0) {
      more = 0;
      while (len < max_path) {
        while (next < nodes && par_s[next] != cur) ++next;
        if (next >= nodes) break;
        if (draft && tries && !summed) { more = 1; break; }      // the mass that is left is needed first
        const int x = tok_s[next];
        const bool in = x >= 0 && x < cols;
        const double q = !draft ? 1.0 : in ? weight(draft[(i64)(a + cur) * ld_q + x]) : 0.0;
        const double r = in ? left(x) : 0.0;
        float u = u_node[a + next];
        u = u != u ? 0.0f : fminf(1.0f, fmaxf(0.0f, u));
        if ((double)u * q * z_s[tries] < r) {
          path_s[len++] = next;
          cur = next;
          tries = 0;
        } else {
          if (!draft) z_s[tries + 1] = z_s[tries] - r;
          tried[tries++] = x;
          summed = false;
        }
        ++next;
      }
    }
    __syncthreads();
    if (!more) break;
    sums();
    if (threadIdx.x == 0) {
      double z = 0.0;
      for (int w = 0; w < 16; ++w) z += part[w];
      z_s[tries] = z;
      summed = true;
    }
    __syncthreads();
  }
  sums();
  // inverse CDF over what is left: the lowest column whose running mass exceeds u * mass, the last one with a weight otherwise
  if (warp == 0) {
    double total = 0.0;
    for (int w = 0; w < 16; ++w) total += part[w];
    int pick = -1;
    if (total > 0.0) {
      float u = u_final[t];
      u = u != u ? 0.0f : fminf(1.0f, fmaxf(0.0f, u));
      const double target = (double)u * total;
      double base = 0.0;
      int w = 0, last = 0;
      for (; w < 16; ++w) {
        if (part[w] > 0.0) last = w;
        if (base + part[w] > target) break;
        base += part[w];
      }
      if (w == 16) { w = last; base = 0.0; for (int k = 0; k < last; ++k) base += part[k]; }
      for (int i0 = w * seg; i0 < min(cols, (w + 1) * seg); i0 += 32) {
        const double r = i0 + lane < min(cols, (w + 1) * seg) ? left(i0 + lane) : 0.0;
        double s = r;
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += v;
        }
        const unsigned over = __ballot_sync(0xffffffffu, r > 0.0 && base + s > target), some = __ballot_sync(0xffffffffu, r > 0.0);
        if (over) { pick = i0 + __ffs(over) - 1; break; }
        if (some) pick = i0 + 31 - __clz(some);
        base += __shfl_sync(0xffffffffu, s, 31);
      }
    }
    for (int i = lane; i < len; i += 32) {
      path[(i64)t * max_path + i] = path_s[i];
      tokens[(i64)t * max_path + i] = i + 1 < len ? tok_s[path_s[i + 1]] : pick;
    }
    if (lane == 0) n_path[t] = len;
  }
}

// ---- commit ---------------------------------------------------------------------------------------------------------
// The K / V rows of node path[i] (i >= 1) move from position ctx + path[i] to ctx + i, 16 bytes a thread, in the order of
// the path.  A path ascends, so path[i] >= i and no row is overwritten before it has been read.
__global__ void __launch_bounds__(256) kv_commit_kernel(uint4* __restrict__ kc, uint4* __restrict__ vc, i64 layer_stride, i64 num_pages,
                                                        const uint32_t* __restrict__ block_table, const int* __restrict__ slots,
                                                        const int* __restrict__ ctxs, const int* __restrict__ path, const int* __restrict__ n_path,
                                                        int max_path, int layers, int kv_heads, int chunks, int page_tokens, int mbps,
                                                        int* __restrict__ new_ctx, int* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.y, slot = slots[t], ctx = ctxs[t];
  if (slot < 0 || ctx < 0) return;
  const int n = min(n_path[t], max_path);
  const i64 per = (i64)layers * kv_heads * chunks;
  const i64 at = (i64)blockIdx.x * 256 + threadIdx.x;
  if (at == 0 && new_ctx) new_ctx[t] = ctx + max(n, 0);
  if (at >= 2 * per) return;
  const i64 e = at % per;
  uint4* cache = (at < per ? kc : vc) + e / ((i64)kv_heads * chunks) * layer_stride;
  const int head = (int)(e / chunks % kv_heads), c = (int)(e % chunks);
  int before = 0;
  for (int i = 1; i < n; ++i) {
    const int node = path[(i64)t * max_path + i];
    const i64 src = (i64)ctx + node, dst = (i64)ctx + i;
    const bool ok = node > before && src < (i64)mbps * page_tokens;
    uint32_t ps = 0, pd = 0;
    if (ok) { ps = block_table[(i64)slot * mbps + src / page_tokens]; pd = block_table[(i64)slot * mbps + dst / page_tokens]; }
    if (!ok || ps >= (uint64_t)num_pages || pd >= (uint64_t)num_pages) {      // not a path, or past the table or the cache: stop here
      if (e == 0 && status) atomicExch(status, WKB_STATUS_KV_POS_RANGE);
      return;
    }
    before = node;
    if (node != i) {
      const i64 from = (((i64)ps * kv_heads + head) * page_tokens + src % page_tokens) * chunks + c;
      const i64 to = (((i64)pd * kv_heads + head) * page_tokens + dst % page_tokens) * chunks + c;
      cache[to] = cache[from];
    }
  }
}

}  // namespace verify

int* gemm_status_word();
}  // namespace wkb

using namespace wkb;

extern "C" {

int wkb_token_probs(const void* logits, int in_dtype, i64 ld, const float* temperature_or_null, float* out, i64 ld_out, i64 rows, i64 cols, void* stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((in_dtype != 0 && in_dtype != 1) || ld < cols || ld_out < cols || cols > 0x7fffff00 || rows > 0x7fffffff) return (int)cudaErrorInvalidValue;
  return (int)launch_pdl(verify::token_probs_kernel, (unsigned)rows, 512, 0, as_stream(stream), logits, in_dtype, ld, temperature_or_null, out, ld_out, cols);
}

int wkb_tree_verify(const float* probs, i64 ld_p, const float* draft_or_null, i64 ld_q, const int* token, const int* parent, const int* tree_row0,
                    i64 rows, i64 n_trees, i64 max_nodes, i64 cols, const float* u_node, const float* u_final, int* path, int* tokens, int* n_path,
                    i64 max_path, void* stream) {
  if (n_trees <= 0) return 0;
  if (rows < 0 || rows > 0x7fffffff || n_trees > 0x7fffffff || cols <= 0 || cols > 0x7fffff00 || ld_p < cols || (draft_or_null && ld_q < cols)) return (int)cudaErrorInvalidValue;
  if (max_nodes < 1 || max_nodes > verify::MAX_NODES || max_path < 1 || max_path > max_nodes) return (int)cudaErrorInvalidValue;
  return (int)launch_pdl(verify::tree_verify_kernel, (unsigned)n_trees, 512, 0, as_stream(stream), probs, ld_p, draft_or_null, ld_q, token, parent, tree_row0,
                         (int)rows, (int)cols, (int)max_nodes, u_node, u_final, path, tokens, n_path, (int)max_path);
}

int wkb_paged_kv_commit(void* kcache, void* vcache, i64 layers, i64 layer_stride, i64 num_pages, const uint32_t* block_table, const int* tree_slot,
                        const int* tree_ctx, const int* path, const int* n_path, i64 max_path, i64 n_trees, i64 kv_heads, i64 head_dim,
                        i64 page_tokens, i64 max_blocks_per_seq, int* new_ctx_or_null, void* stream) {
  if (n_trees <= 0 || layers <= 0) return 0;
  if (n_trees > 65535 || max_path < 1 || kv_heads < 1 || head_dim < 8 || head_dim % 8 != 0 || page_tokens < 1 || max_blocks_per_seq < 1 || num_pages < 1 ||
      max_blocks_per_seq * page_tokens > 0x7fffff00 || max_path > 0x7fffffff)
    return (int)cudaErrorInvalidValue;
  if (new_ctx_or_null == tree_ctx) return (int)cudaErrorInvalidValue;      // read by every block of the tree
  if (layers > 1 && layer_stride < num_pages * kv_heads * page_tokens * head_dim) return (int)cudaErrorInvalidValue;
  if (((((uintptr_t)kcache) | ((uintptr_t)vcache)) & 15) != 0 || layer_stride % 8 != 0) return (int)cudaErrorMisalignedAddress;
  const i64 threads = 2 * layers * kv_heads * (head_dim / 8), blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return (int)cudaErrorInvalidValue;
  int* status = gemm_status_word();
  if (!status) return (int)cudaErrorMemoryAllocation;
  return (int)launch_pdl(verify::kv_commit_kernel, dim3((unsigned)blocks, (unsigned)n_trees), 256, 0, as_stream(stream), (uint4*)kcache, (uint4*)vcache,
                         layer_stride / 8, num_pages, block_table, tree_slot, tree_ctx, path, n_path, (int)max_path, (int)layers, (int)kv_heads,
                         (int)(head_dim / 8), (int)page_tokens, (int)max_blocks_per_seq, new_ctx_or_null, status);
}

}  // extern "C"
