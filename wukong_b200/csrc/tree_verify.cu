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
__device__ __forceinline__ float logit(const float* x, int i) { return x[i]; }
__device__ __forceinline__ float logit(const __nv_bfloat16* x, int i) { return bf16_bits_to_f32(reinterpret_cast<const u16*>(x)[i]); }
// 2^x to 2^-22 of the result; 0 below 2^-126
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2(e) / t, finite and not 0, so that the maximum keeps weight 1 and a token that is ruled out weight 0
__device__ __forceinline__ float exponent_scale(float t) { return t != t ? t : fmaxf(fminf(1.4426950408889634f / t, 3.402823466e+38f), 1e-37f); }

// Rows wider than a cluster's registers: one CTA per row, three passes (the second and third mostly from L2).
template <typename T>
__global__ void __launch_bounds__(512) token_probs_wide_kernel(const T* __restrict__ x, i64 ld, const float* __restrict__ temperature, float* __restrict__ out,
                                                               i64 ld_out, int cols) {
  pdl_wait();
  pdl_trigger();
  __shared__ float red_v[16];
  __shared__ int red_i[16];
  const i64 row = blockIdx.x;
  const float temp = temperature ? temperature[row] : 1.0f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float best = -INFINITY;
  int at = 0x7fffffff;
  bool nan = temp != temp;
  for (int i = threadIdx.x; i < cols; i += 512) {
    const float v = logit(x + row * ld, i);
    nan |= v != v;
    if (v > best) { best = v; at = i; }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    if (v > best || (v == best && i < at)) { best = v; at = i; }
  }
  if (lane == 0) { red_v[warp] = best; red_i[warp] = at; }
  nan = __syncthreads_or(nan);
  for (int w = 0; w < 16; ++w)
    if (red_v[w] > best || (red_v[w] == best && red_i[w] < at)) { best = red_v[w]; at = red_i[w]; }
  __syncthreads();
  const float scale = exponent_scale(temp);
  float sum = 0.0f;
  if (temp > 0.0f) {
    for (int i = threadIdx.x; i < cols; i += 512) sum += ex2((logit(x + row * ld, i) - best) * scale);
    sum = warp_sum(sum);
    if (lane == 0) red_v[warp] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < 16; ++w) sum += red_v[w];
  }
  for (int i = threadIdx.x; i < cols; i += 512) {
    float p;
    if (nan) p = NAN;
    else if (best == -INFINITY) p = 0.0f;                 // every token is ruled out
    else if (temp > 0.0f) p = ex2((logit(x + row * ld, i) - best) * scale) / sum;
    else p = i == at ? 1.0f : 0.0f;
    out[row * ld_out + i] = p;
  }
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

constexpr int PT = 512;      // threads of a CTA
// columns of a CTA when `ctas` share a row: whole 128-byte lines of f32
__host__ __device__ __forceinline__ int probs_run(i64 cols, int ctas) { return (int)((cols + ctas - 1) / ctas + 31) / 32 * 32; }

// A row is a cluster's: each CTA keeps up to E * PT columns in registers, so the logits are read once and the probabilities
// written once (HBM is the bound).  Every warp reduces its columns to (maximum, sum relative to it) and puts the pair into
// every CTA's table; one cluster barrier later each warp adds up the whole table, so that nothing else is waited for
// between the last load and the first store (with block-wide reductions and a second barrier 1024 x 32000 took 65 us,
// now 46, 0.86 of the copy rate).  Loads and stores are 4 bytes a thread, coalesced, because the rows of an odd vocabulary are aligned to no more
// than that, and where they are, 16 bytes a thread took longer (54 against 49 us).
template <typename T, int E, int PT>
__global__ void __launch_bounds__(PT, (E > 32 ? 1 : E > 8 ? 2 : 4) * (512 / PT)) token_probs_kernel(const T* __restrict__ x, i64 ld, const float* __restrict__ temperature,
                                                                                                  float* __restrict__ out, i64 ld_out, int cols) {
  pdl_wait();
  pdl_trigger();
  __shared__ float2 table[8 * PT / 32];
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");      // awaited before the first store to another CTA: it has begun
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const i64 row = blockIdx.x / size;
  // The CTAs' columns: equal runs of the row.  Of f32 a thread takes every PT-th one, of bf16 every PT-th pair in an aligned
  // word; where a run begins or ends in the middle of a word, its column is read by itself.
  constexpr int PAIR = sizeof(T) == 2 ? 2 : 1;
  const int run = probs_run(cols, (int)size), start = (int)rank * run, end = min(cols, start + run);
  const T* xr = x + row * ld + start;
  const int shift = PAIR == 2 ? (int)((reinterpret_cast<uintptr_t>(xr) >> 1) & 1) : 0, first = start - shift + PAIR * (int)threadIdx.x;
  const int mine = end - first;      // column at(e) behind `first` is this CTA's below `mine`, and not in front of the run
  auto at = [](int e) { return e / PAIR * PAIR * PT + e % PAIR; };
  auto own = [&](int e) { return at(e) < mine && (e > 0 || first >= start); };
  xr += first - start;
  float* const o = out + row * ld_out + first;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; e += PAIR) {
    if (PAIR == 1) v[e] = own(e) ? logit(xr, at(e)) : -INFINITY;
    else {
      const bool both = own(e) && at(e + PAIR - 1) < mine;
      const uint32_t w = both ? *reinterpret_cast<const uint32_t*>(xr + at(e)) : 0xff80ff80u;
      v[e] = u2f(w << 16);
      v[e + PAIR - 1] = u2f(w & 0xffff0000u);
    }
  }
  if (PAIR == 2) {
    if (first < start && PAIR - 1 < mine) v[PAIR - 1] = logit(xr, PAIR - 1);
    if (mine > 0 && (mine - 1) % (PAIR * PT) == 0 && first + mine - 1 >= start) {      // this thread's last column is a word's first half
      const float last = logit(xr, mine - 1);
#pragma unroll
      for (int e = 0; e < E; e += PAIR)
        if (at(e) == mine - 1) v[e] = last;
    }
  }
  const float temp = temperature ? temperature[row] : 1.0f;
  const bool cold = temp <= 0.0f;      // alike in all CTAs of the row
  const float scale = exponent_scale(temp);
  float m = -INFINITY, second;         // second: the sum, or the column of the maximum
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
  float base;
  if (cold) {
    int col = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
      if (v[e] == m && own(e)) col = first + at(e);
      nan |= v[e] != v[e];
    }
    for (int k = 16; k > 0; k >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m, k);
      const int oc = __shfl_xor_sync(0xffffffffu, col, k);
      if (om > m || (om == m && oc < col)) { m = om; col = oc; }
    }
    if (__any_sync(0xffffffffu, nan)) m = NAN;
    base = 0.0f;
    second = __int_as_float(col);
  } else {
    base = m == -INFINITY ? 0.0f : m;
    second = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = ex2((v[e] - base) * scale);      // a NaN spoils the sum and with it the row
      second += v[e];
    }
    const float mw = warp_max(m);
    second = warp_sum(m == -INFINITY ? second : second * ex2((m - mw) * scale));
    m = mw;
  }
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (lane < (int)size) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_addr(&table[rank * (PT / 32) + warp])), "r"(lane));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(m), "f"(second) : "memory");
  }
  cluster_sync();
  const int entries = (int)size * (PT / 32);
  if (cold) {
    bool nan = false;
    float top = -INFINITY;
    int col = 0x7fffffff;
    for (int k = lane; k < entries; k += 32) {
      const float2 p = table[k];
      nan |= p.x != p.x;
      if (p.x > top || (p.x == top && __float_as_int(p.y) < col)) { top = p.x; col = __float_as_int(p.y); }
    }
    for (int k = 16; k > 0; k >>= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, top, k);
      const int oc = __shfl_xor_sync(0xffffffffu, col, k);
      if (om > top || (om == top && oc < col)) { top = om; col = oc; }
    }
    if (top == -INFINITY) col = -1;      // every token is ruled out
    nan = __any_sync(0xffffffffu, nan);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (own(e)) o[at(e)] = nan ? NAN : first + at(e) == col ? 1.0f : 0.0f;
    return;
  }
  float top = -INFINITY, l = 0.0f;
  for (int k = lane; k < entries; k += 32) top = fmaxf(top, table[k].x);
  top = warp_max(top);
  for (int k = lane; k < entries; k += 32) {
    const float2 p = table[k];
    l += p.x == -INFINITY ? p.y : p.y * ex2((p.x - top) * scale);
  }
  l = warp_sum(l);
  const float behind = (base - top) * scale;      // this thread's exponentials are relative to its own maximum
  const float f = top == -INFINITY ? (l == l ? 0.0f : NAN) : (mine > 0 && base <= top ? ex2(behind) : 1.0f) / l;
  if (PAIR == 2 && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {      // stores of half pairs would be masked sectors, twice as many
#pragma unroll
    for (int e = 0; e < E; e += PAIR) {
      if (own(e) && at(e + 1) < mine) *reinterpret_cast<float2*>(o + at(e)) = make_float2(v[e] * f, v[e + PAIR - 1] * f);
      else {
        if (own(e)) o[at(e)] = v[e] * f;
        if (at(e + PAIR - 1) < mine) o[at(e + PAIR - 1)] = v[e + PAIR - 1] * f;
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (own(e)) o[at(e)] = v[e] * f;
}

// ---- verification ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ double weight(float v) { return v > 0.0f && v <= 3.402823466e+38f ? (double)v : 0.0; }

// 4 bytes of global memory into this thread's cell, or 0 where `have` is 0; complete after cp.async.wait_all
__device__ __forceinline__ void fetch4(float* cell, const float* src, uint32_t have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(cell)), "l"(src), "r"(have) : "memory");
}
// What the leader asks of its cluster: the masses that are left of node `row` after `tries` rejections.
struct alignas(16) Ask {
  int row, tries, last, pad;
};
// One cluster per tree.  The walk needs two numbers of each node, p and q of its token in its parent's rows: the leading
// CTA gathers them for all nodes at once, and its first warp walks in shared memory.  Only the mass that is left after a
// rejection (before the next sibling is tried) and the final draw need a pass over the vocabulary, a contiguous run of
// columns per warp of the cluster; the row is read from HBM once and the run that holds the draw a second time, from L2.
// The leader alone decides, so every CTA takes the same steps.  Sums are in a fixed order.  Bound: the latency of the four
// dependent trips to memory for a few trees (8.1 to 9 us for one chain over 50257 columns, 5 of them a warp's instructions and
// barriers), the longest walk's passes for many (27 us for 64 trees over 32000).
constexpr int HOLD = 16;
template <bool DRAFT>
__global__ void __launch_bounds__(PT, 2) tree_verify_kernel(const float* __restrict__ probs, i64 ld_p, const float* __restrict__ draft, i64 ld_q,
                                                         const int* __restrict__ token, const int* __restrict__ parent, const int* __restrict__ row0,
                                                         int rows, int cols, int max_nodes, const float* __restrict__ u_node,
                                                         const float* __restrict__ u_final, int* __restrict__ path, int* __restrict__ tokens,
                                                         int* __restrict__ n_path, int max_path) {
  pdl_wait();
  pdl_trigger();
  __shared__ int tok_s[MAX_NODES], par_s[MAX_NODES], tried_s[MAX_NODES], path_s[MAX_NODES];
  __shared__ float p_s[MAX_NODES], q_s[MAX_NODES], u_s[MAX_NODES];
  __shared__ double z_s[MAX_NODES + 1], part_s[8 * PT / 32];
  __shared__ Ask ask;
  extern __shared__ float cells[];      // [p, q][HOLD][PT]
  __shared__ int walk_s[3], pick_s[2];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int t = blockIdx.x / size, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = (int)size * (PT / 32);
  const int a = min(max(row0[t], 0), rows), nodes = min(min(max(row0[t + 1], a), rows) - a, max_nodes);
  float u = u_final[t];
  u = u != u ? 0.0f : fminf(1.0f, fmaxf(0.0f, u));
  int* const my_path = path + (i64)t * max_path;
  int* const my_tokens = tokens + (i64)t * max_path;
  if (nodes <= 0) {      // (uniform over the cluster: nobody meets)
    if (rank == 0) {
      for (int i = threadIdx.x; i < max_path; i += PT) { my_path[i] = -1; my_tokens[i] = -1; }
      if (threadIdx.x == 0) n_path[t] = 0;
    }
    return;
  }
  if (rank == 0) {
    for (int i = threadIdx.x; i < nodes; i += PT) {
      const int x = token[a + i], par = parent[a + i];
      const bool known = i > 0 && par >= 0 && par < nodes && x >= 0 && x < cols;
      const float un = u_node[a + i];
      tok_s[i] = x;
      par_s[i] = i > 0 ? par : -1;
      u_s[i] = un != un ? 0.0f : fminf(1.0f, fmaxf(0.0f, un));
      p_s[i] = known ? probs[(i64)(a + par) * ld_p + x] : 0.0f;
      q_s[i] = DRAFT && known ? draft[(i64)(a + par) * ld_q + x] : 0.0f;
    }
    __syncthreads();
  }
  const int run = ((cols + warps - 1) / warps + 31) / 32 * 32;      // columns of a warp
  // what is left of column i's weight p (q the draft's) after the rejections
  auto left = [&](int i, float p, float q, int tries) -> double {
    double r = weight(p);
    if (DRAFT) {
      const double w = weight(q);
      for (int k = 0; k < tries; ++k) r = fmax(r - z_s[k] * w, 0.0);
    } else {
      for (int k = 0; k < tries; ++k)
        if (tried_s[k] == i) r = 0.0;
    }
    return r;
  };
  auto remote = [&](const void* p, uint32_t of) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(of));
    return r;
  };
  // A thread's columns go through its own cells of shared memory, HOLD at a time: all copies in flight together, and
  // rolled loops (unrolled, fetching the instructions took longer than fetching the columns), and a run of no more
  // than that stays there, so that the passes after a node's first read nothing.
  const bool holds = run <= 32 * HOLD;
  float* const cell = cells + threadIdx.x;
  int held = -1;
  int cur = 0, tries = 0, len = 1, next = 1;      // the walk, of the leader's first warp
  bool summed = false;
  if (rank == 0 && warp == 0 && lane == 0) { path_s[0] = 0; z_s[0] = 1.0; }
  for (;;) {
    if (rank == 0 && warp == 0) {
      bool wait = false;
      __syncwarp();
      while (len < max_path && !wait) {
        int c = -1;      // the next node from `next` on whose parent is `cur`
        for (int b = next & ~31; b < nodes && c < 0; b += 32) {
          const unsigned hit = __ballot_sync(0xffffffffu, b + lane < nodes && b + lane >= next && par_s[b + lane] == cur);
          if (hit) c = b + __ffs(hit) - 1;
        }
        if (c < 0) break;
        if (DRAFT && tries && !summed) { wait = true; break; }      // the mass that is left is needed first
        const int x = tok_s[c];
        const bool in = x >= 0 && x < cols;
        const double q = !DRAFT ? 1.0 : in ? weight(q_s[c]) : 0.0, r = in ? left(x, p_s[c], q_s[c], tries) : 0.0;
        __syncwarp();
        if ((double)u_s[c] * q * z_s[tries] < r) {
          if (lane == 0) path_s[len] = c;
          ++len;
          cur = c;
          tries = 0;
        } else {
          if (lane == 0) {
            if (!DRAFT) z_s[tries + 1] = z_s[tries] - r;
            tried_s[tries] = x;
          }
          ++tries;
          summed = false;
        }
        __syncwarp();
        next = c + 1;
      }
      if (lane == 0) { ask.row = a + cur; ask.tries = tries; ask.last = wait ? 0 : 1; }
    }
    cluster_sync();
    Ask now;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(now.row), "=r"(now.tries), "=r"(now.last), "=r"(now.pad) : "r"(remote(&ask, 0)) : "memory");
    if (rank != 0) {
      for (int k = threadIdx.x; k < now.tries; k += PT) {
        if (DRAFT) asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(z_s[k]) : "r"(remote(&z_s[k], 0)) : "memory");
        else asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(tried_s[k]) : "r"(remote(&tried_s[k], 0)) : "memory");
      }
      __syncthreads();
    }
    const float* pr = probs + (i64)now.row * ld_p;
    const float* qr = DRAFT ? draft + (i64)now.row * ld_q : nullptr;
    {
      const int g = (int)rank * (PT / 32) + warp, end = (int)min((i64)cols, (i64)(g + 1) * run);
      double s[4] = {0.0, 0.0, 0.0, 0.0};
      for (i64 i0 = (i64)g * run + lane; i0 - lane < end; i0 += 32 * HOLD) {
        if (!holds || held != now.row) {
#pragma unroll 4
          for (int k = 0; k < HOLD; ++k) {
            const i64 i = i0 + k * 32;
            const uint32_t have = i < end ? 4u : 0u;      // the cell of a column behind the run is filled with 0
            fetch4(cell + k * PT, pr + (have ? i : 0), have);
            if (DRAFT) fetch4(cell + (HOLD + k) * PT, qr + (have ? i : 0), have);
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
        }
        const int n = min(HOLD, (int)((end - (i0 - lane) + 31) >> 5));
        // four sums: an f64 operation's latency is what a column costs
#pragma unroll 1
        for (int k = 0; k < n; k += 4) {
          double r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = weight(cell[(k + e) * PT]);
          if (DRAFT) {
            double w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = weight(cell[(HOLD + k + e) * PT]);
#pragma unroll 1
            for (int j = 0; j < now.tries; ++j) {
              const double z = z_s[j];
#pragma unroll
              for (int e = 0; e < 4; ++e) r[e] = fmax(r[e] - z * w[e], 0.0);
            }
          } else {
#pragma unroll 1
            for (int j = 0; j < now.tries; ++j) {
              const int at = tried_s[j] - (int)i0 - k * 32;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (at == e * 32) r[e] = 0.0;
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] += r[e];
        }
      }
      held = now.row;
      double sum = (s[0] + s[1]) + (s[2] + s[3]);
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote(&part_s[g], 0)), "d"(sum) : "memory");
    }
    cluster_sync();
    if (now.last) break;
    if (rank == 0 && warp == 0) {
      double z = 0.0;
      for (int w = lane; w < warps; w += 32) z += part_s[w];
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (lane == 0) z_s[tries] = z;
      summed = true;
      __syncwarp();
    }
  }
  if (rank != 0) return;
  if (threadIdx.x == 0) { walk_s[0] = cur; walk_s[1] = tries; walk_s[2] = len; pick_s[0] = 0x7fffffff; pick_s[1] = -1; }
  __syncthreads();
  cur = walk_s[0]; tries = walk_s[1]; len = walk_s[2];
  // inverse CDF over what is left: the lowest column whose running mass exceeds u * mass, the last one with a weight otherwise
  const float* pr = probs + (i64)(a + cur) * ld_p;
  const float* qr = DRAFT ? draft + (i64)(a + cur) * ld_q : nullptr;
  // the runs' masses, up to four neighbours a lane: running sums, the whole, and the first run that exceeds the target
  constexpr int PER = 8 * (PT / 32) / 32;
  double v[PER], own = 0.0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    v[k] = lane * PER + k < warps ? part_s[lane * PER + k] : 0.0;
    own += v[k];
  }
  double up_to = own;
  for (int o = 1; o < 32; o <<= 1) {
    const double n = __shfl_up_sync(0xffffffffu, up_to, o);
    if (lane >= o) up_to += n;
  }
  const double total = __shfl_sync(0xffffffffu, up_to, 31);
  int pick = -1;
  if (total > 0.0) {
    double target = (double)u * total, base = up_to - own, before = 0.0;      // before: the mass in front of the run that this lane offers
    int offer = -1, last = -1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (v[k] > 0.0 && offer < 0) {
        last = lane * PER + k;
        before = base;
        if (k + 1 == PER ? up_to > target : base + v[k] > target) offer = last;
      }
      base += v[k];
    }
    const unsigned over = __ballot_sync(0xffffffffu, offer >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
    const int from = over ? __ffs(over) - 1 : 31 - __clz(some);
    const int w0 = __shfl_sync(0xffffffffu, over ? offer : last, from);
    base = __shfl_sync(0xffffffffu, before, from);
    if (!over) target = INFINITY;      // nothing exceeds it: the last weight of all
    // the whole CTA goes over that run, 32 columns a warp at a time
    const i64 end = min((i64)cols, (i64)(w0 + 1) * run);
    for (i64 i0 = (i64)w0 * run; i0 < end; i0 += PT) {
      const i64 i = i0 + threadIdx.x;
      const double r = i < end ? left((int)i, pr[i], DRAFT && tries ? qr[i] : 0.0f, tries) : 0.0;
      double sum = r;
      for (int o = 1; o < 32; o <<= 1) {
        const double n = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += n;
      }
      __syncthreads();
      if (lane == 31) part_s[warp] = sum;
      __syncthreads();
      double sums = lane < PT / 32 ? part_s[lane] : 0.0;      // running sums of the warps, lane w for warp w
      for (int o = 1; o < PT / 32; o <<= 1) {
        const double n = __shfl_up_sync(0xffffffffu, sums, o);
        if (lane >= o) sums += n;
      }
      const double front = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
      sum += warp > 0 ? base + front : base;
      base += __shfl_sync(0xffffffffu, sums, PT / 32 - 1);
      if (r > 0.0) {
        if (sum > target) atomicMin(&pick_s[0], (int)i);
        atomicMax(&pick_s[1], (int)i);
      }
    }
    __syncthreads();
    pick = pick_s[0] != 0x7fffffff ? pick_s[0] : pick_s[1];
  }
  if (warp != 0) return;
  for (int i = lane; i < max_path; i += 32) {
    my_path[i] = i < len ? path_s[i] : -1;
    my_tokens[i] = i + 1 < len ? tok_s[path_s[i + 1]] : i + 1 == len ? pick : -1;
  }
  if (lane == 0) n_path[t] = len;
}

// ---- commit ---------------------------------------------------------------------------------------------------------
// The K / V rows of node path[i] (i >= 1) move from position ctx + path[i] to ctx + i, eight nodes at a time: their
// look-ups, then for each 16 bytes of a token's rows in all layers the loads and the stores.  The grid is bounded, so that
// the four dependent look-ups of a block are paid once for several of its elements.  A path ascends, so path[j] > i for j > i: a row that is
// written was read before, in this batch or an earlier one.  Bound: HBM in 256-byte pieces for many sequences (10 us
// for 64 of 32 layers), dependent trips for one (3.5 us).
__global__ void __launch_bounds__(256, 3) kv_commit_kernel(uint4* __restrict__ kc, uint4* __restrict__ vc, i64 layer_stride, i64 num_pages,
                                                        const uint32_t* __restrict__ block_table, const int* __restrict__ slots,
                                                        const int* __restrict__ ctxs, const int* __restrict__ path, const int* __restrict__ n_path,
                                                        int max_path, int layers, int kv_heads, int chunks, int page_tokens, int mbps,
                                                        int* __restrict__ new_ctx, int* __restrict__ status) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.y, slot = slots[t], ctx = ctxs[t], length = n_path[t], n = min(length, max_path);
  if (slot < 0 || ctx < 0) return;
  const int per = layers * kv_heads * chunks, at0 = (int)blockIdx.x * 256 + threadIdx.x;
  const uint32_t page_stride = (uint32_t)kv_heads * (uint32_t)page_tokens * (uint32_t)chunks;      // a slab is no more than 2^32 units
  const uint32_t* bt = block_table + (i64)slot * mbps;
  const i64 cover = (i64)mbps * page_tokens;
  const uint32_t pt = (uint32_t)page_tokens;
  constexpr int BATCH = 8;
  int before = 0;
  for (int i0 = 1; i0 < n; i0 += BATCH) {
    int node[BATCH];
    uint32_t from[BATCH], to[BATCH];      // in 16-byte units, of the first head
    int good = 0;      // entries of this batch that belong to a path
#pragma unroll
    for (int k = 0; k < BATCH; ++k) node[k] = i0 + k < n ? path[(i64)t * max_path + i0 + k] : -1;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const i64 src = (i64)ctx + node[k], dst = (i64)ctx + i0 + k;
      const bool in = node[k] >= i0 + k && src < cover;
      const uint32_t s32 = in ? (uint32_t)src : 0u, d32 = in ? (uint32_t)dst : 0u;
      const uint32_t ps = in ? bt[s32 / pt] : 0xffffffffu, pd = in ? bt[d32 / pt] : 0xffffffffu;
      const bool ok = ps < (uint64_t)num_pages && pd < (uint64_t)num_pages && node[k] > (k ? node[k ? k - 1 : 0] : before);
      from[k] = ok ? ps * page_stride + (s32 % pt) * (uint32_t)chunks : 0u;
      to[k] = ok ? pd * page_stride + (d32 % pt) * (uint32_t)chunks : 0u;
      if (ok && good == k) good = k + 1;
    }
    for (int at = at0; at < 2 * per; at += (int)gridDim.x * 256) {
      const int e = at < per ? at : at - per, lh = e / chunks, c = e - lh * chunks, layer = lh / kv_heads, head = lh - layer * kv_heads;
      uint4* cache = (at < per ? kc : vc) + layer * layer_stride + (i64)head * page_tokens * chunks + c;
      uint4 v[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < good && from[k] != to[k]) v[k] = cache[from[k]];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (k < good && from[k] != to[k]) cache[to[k]] = v[k];
    }
    if (good < min(BATCH, n - i0)) {      // not a path, or past the table or the cache: the moves end here
      if (at0 == 0) {
        atomicExch(status, WKB_STATUS_KV_POS_RANGE);
        if (new_ctx) new_ctx[t] = ctx + i0 + good;
      }
      return;
    }
    before = node[BATCH - 1];
  }
  if (at0 == 0) {
    if (new_ctx) new_ctx[t] = ctx + max(n, 0);
    if (length > max_path) atomicExch(status, WKB_STATUS_KV_POS_RANGE);
  }
}

// A launch whose blocks form clusters of `ctas`, as a programmatic dependent like launch_pdl's.
template <typename... KArgs, typename... Args>
static cudaError_t launch_cluster(void (*kernel)(KArgs...), unsigned grid, unsigned block, int smem, int ctas, cudaStream_t st, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// A row's columns over the CTAs of a cluster and the registers of their threads: clusters grow until two CTAs per SM are
// at work (small batches) and a thread holds at most 32 columns (large vocabularies), or at 8.  CTAs of 256 threads,
// which leave an SM more of them to overlap, while eight hold a row: 1024 x 7582 f32 in 14.8 us, of 512 threads 17.9;
// 128 x 32000 in 9.1 and 10.9; of bf16 1024 x 7582 in 13.1 and 18.1, 1024 x 32000 in 46.3 and 47.0, 640 x 50257 in 58.7
// and 57.9.
constexpr i64 PROBS_MAX = 8 * (64 * 512 - 32);      // (a run of bf16 may begin with half a pair)
struct ProbsShape {
  int ctas, regs, threads;
};
template <typename T>
static ProbsShape probs_shape(const T* x, i64 ld, i64 rows, i64 cols) {
  constexpr bool PAIRS = sizeof(T) == 2;
  // the column in front of a run: only where a row may begin with half a word (1024 x 32768 bf16: 47.6 us without it, 72 with it)
  const int half = PAIRS && (((reinterpret_cast<uintptr_t>(x) >> 1) | (uintptr_t)ld) & 1);
  const bool small = cols <= 8 * (32 * 256 - 32 * half);
  ProbsShape s{1, 4, small ? 256 : 512};
  auto need = [&] { return probs_run(cols, s.ctas) + half; };
  while (s.ctas < 8 && (need() > 32 * s.threads || (rows * s.ctas < 2 * WKB_SM_COUNT && cols > (i64)s.ctas * 4 * s.threads))) s.ctas *= 2;
  while (s.regs < 64 && s.regs * s.threads < need()) s.regs *= 2;
  return s;
}
template <typename T, int PT>
static int launch_probs(const ProbsShape& s, const T* x, i64 ld, const float* temperature, float* out, i64 ld_out, i64 rows, i64 cols, cudaStream_t st) {
  auto kern = s.regs == 4 ? token_probs_kernel<T, 4, PT> : s.regs == 8 ? token_probs_kernel<T, 8, PT> : s.regs == 16 ? token_probs_kernel<T, 16, PT> : token_probs_kernel<T, 32, PT>;
  if constexpr (PT == 512) {
    if (s.regs == 64) kern = token_probs_kernel<T, 64, PT>;
  }
  return (int)launch_cluster(kern, (unsigned)(rows * s.ctas), PT, 0, s.ctas, st, x, ld, temperature, out, ld_out, (int)cols);
}
template <typename T>
static int launch_probs(const T* x, i64 ld, const float* temperature, float* out, i64 ld_out, i64 rows, i64 cols, cudaStream_t st) {
  if (cols > PROBS_MAX) return (int)launch_pdl(token_probs_wide_kernel<T>, (unsigned)rows, 512, 0, st, x, ld, temperature, out, ld_out, (int)cols);
  const ProbsShape s = probs_shape(x, ld, rows, cols);
  return s.threads == 256 ? launch_probs<T, 256>(s, x, ld, temperature, out, ld_out, rows, cols, st) : launch_probs<T, 512>(s, x, ld, temperature, out, ld_out, rows, cols, st);
}
// CTAs of a tree's cluster: doubled while the trees' CTAs are fewer than two per SM and each has more than 2048 columns, up to 8.
// So the last doubling may pass the 296 CTAs that run at a time (64 trees over 32000 columns: 512 of them, in two waves, 27.5 us).
static int verify_ctas(i64 n_trees, i64 cols) {
  int c = 1;
  while (c < 8 && n_trees * c < 2 * WKB_SM_COUNT && cols > (i64)c * 2048) c *= 2;
  return c;
}

}  // namespace verify

int* gemm_status_word();
}  // namespace wkb

using namespace wkb;

extern "C" {

int wkb_token_probs(const void* logits, int in_dtype, i64 ld, const float* temperature_or_null, float* out, i64 ld_out, i64 rows, i64 cols, void* stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if ((in_dtype != 0 && in_dtype != 1) || ld < cols || ld_out < cols || cols > (1 << 30) || rows > 0x7fffffff / 8) return (int)cudaErrorInvalidValue;
  if (in_dtype == 0) return verify::launch_probs(static_cast<const float*>(logits), ld, temperature_or_null, out, ld_out, rows, cols, as_stream(stream));
  return verify::launch_probs(static_cast<const __nv_bfloat16*>(logits), ld, temperature_or_null, out, ld_out, rows, cols, as_stream(stream));
}

int wkb_tree_verify(const float* probs, i64 ld_p, const float* draft_or_null, i64 ld_q, const int* token, const int* parent, const int* tree_row0,
                    i64 rows, i64 n_trees, i64 max_nodes, i64 cols, const float* u_node, const float* u_final, int* path, int* tokens, int* n_path,
                    i64 max_path, void* stream) {
  if (n_trees <= 0) return 0;
  if (rows < 0 || rows > 0x7fffffff || n_trees > 0x7fffffff || cols <= 0 || cols > 0x7fffff00 || ld_p < cols || (draft_or_null && ld_q < cols)) return (int)cudaErrorInvalidValue;
  if (max_nodes < 1 || max_nodes > verify::MAX_NODES || max_path < 1 || max_path > max_nodes) return (int)cudaErrorInvalidValue;
  const int ctas = verify::verify_ctas(n_trees, cols);
  if (n_trees > 0x7fffffff / ctas) return (int)cudaErrorInvalidValue;
  auto kern = draft_or_null ? verify::tree_verify_kernel<true> : verify::tree_verify_kernel<false>;
  constexpr int SMEM = 2 * verify::HOLD * verify::PT * (int)sizeof(float);
  static bool attr_set[64][2] = {{false}};
  int dev = 0;
  cudaGetDevice(&dev);
  if (!attr_set[dev & 63][draft_or_null != nullptr]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    attr_set[dev & 63][draft_or_null != nullptr] = true;
  }
  return (int)verify::launch_cluster(kern, (unsigned)(n_trees * ctas), verify::PT, SMEM, ctas, as_stream(stream), probs, ld_p, draft_or_null, ld_q, token, parent,
                                     tree_row0, (int)rows, (int)cols, (int)max_nodes, u_node, u_final, path, tokens, n_path, (int)max_path);
}

int wkb_paged_kv_commit(void* kcache, void* vcache, i64 layers, i64 layer_stride, i64 num_pages, const uint32_t* block_table, const int* tree_slot,
                        const int* tree_ctx, const int* path, const int* n_path, i64 max_path, i64 n_trees, i64 kv_heads, i64 head_dim,
                        i64 page_tokens, i64 max_blocks_per_seq, int* new_ctx_or_null, void* stream) {
  if (n_trees <= 0 || layers <= 0) return 0;
  // every extent first, so that no product below wraps around
  if (layers > 0x7fffffff || kv_heads > 0x7fffffff || head_dim > 0x7fffffff || page_tokens > 0x7fffffff || max_blocks_per_seq > 0x7fffffff) return (int)cudaErrorInvalidValue;
  if (n_trees > 65535 || max_path < 1 || kv_heads < 1 || head_dim < 8 || head_dim % 8 != 0 || page_tokens < 1 || max_blocks_per_seq < 1 || num_pages < 1 ||
      max_blocks_per_seq * page_tokens > 0x7fffff00 || max_path > 0x7fffffff ||
      (double)num_pages * (double)kv_heads * (double)page_tokens * (double)(head_dim / 8) > 4294967040.0)      // 64 GB a layer and cache
    return (int)cudaErrorInvalidValue;
  auto meets_new_ctx = [&](const int* a, i64 n) { return new_ctx_or_null && new_ctx_or_null < a + n && a < new_ctx_or_null + n_trees; };
  if (meets_new_ctx(tree_slot, n_trees) || meets_new_ctx(tree_ctx, n_trees) || meets_new_ctx(n_path, n_trees) || meets_new_ctx(path, n_trees * max_path))
    return (int)cudaErrorInvalidValue;      // read by every block of a tree
  if (layers > 1 && layer_stride < num_pages * kv_heads * page_tokens * head_dim) return (int)cudaErrorInvalidValue;
  if (((((uintptr_t)kcache) | ((uintptr_t)vcache)) & 15) != 0 || layer_stride % 8 != 0) return (int)cudaErrorMisalignedAddress;
  if (layers > 0x3fffffff / 2 / (head_dim / 8) / kv_heads) return (int)cudaErrorInvalidValue;
  const i64 threads = 2 * layers * kv_heads * (head_dim / 8), blocks = (threads + 255) / 256;
  const i64 wave = (WKB_SM_COUNT * 3 + n_trees - 1) / n_trees;      // blocks a tree that fill the SMs once
  int* status = gemm_status_word();
  if (!status) return (int)cudaErrorMemoryAllocation;
  return (int)launch_pdl(verify::kv_commit_kernel, dim3((unsigned)(blocks < wave ? blocks : wave), (unsigned)n_trees), 256, 0, as_stream(stream), (uint4*)kcache, (uint4*)vcache,
                         layer_stride / 8, num_pages, block_table, tree_slot, tree_ctx, path, n_path, (int)max_path, (int)layers, (int)kv_heads,
                         (int)(head_dim / 8), (int)page_tokens, (int)max_blocks_per_seq, new_ctx_or_null, status);
}

}  // extern "C"
