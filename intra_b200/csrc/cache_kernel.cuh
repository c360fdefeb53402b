// What happens to a cache between two steps: accepted rows move together (keep_rows_kernel), and the keys that have
// received the least attention leave (evict_select_kernel picks the rows that stay, evict_copy_kernel gathers them).
#pragma once
#include <cooperative_groups.h>
#include <stdint.h>

#include "attn_kernel.cuh"

namespace intra {

// ---- accepted rows ------------------------------------------------------------------------------------------
constexpr int KEEP_THREADS = 256;
constexpr int KEEP_MAX_TOKENS = 64;
constexpr int KEEP_TENSORS = 64;                 // caches one launch takes (a launch's parameters hold 4 KB)

struct KeepParams {
  __nv_bfloat16* cache[KEEP_TENSORS];            // (B, S, Hkv, 128) by strides
  TensorView s[KEEP_TENSORS];
  const int* lengths;                            // (B) keys before the tokens' own
  const int* path;                               // (B, n): tokens to keep, in order; negative: none
  int64_t path_sb;
  int S, Hkv, n;
};

// Row lengths + path[i] -> lengths + i. One CTA per (tensor, batch, head): all rows are read before the first is
// written, so any order of path is right. Entries outside the tokens' rows or the cache move nothing.
__global__ void __launch_bounds__(KEEP_THREADS) keep_rows_kernel(const __grid_constant__ KeepParams p) {
  const int piece = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int hk = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv;
  const TensorView s = p.s[blockIdx.y];
  const int ctx = p.lengths[b];
  uint4* const base = reinterpret_cast<uint4*>(p.cache[blockIdx.y] + b * s.sb + hk * s.sh) + piece;
  constexpr int PER = KEEP_MAX_TOKENS / (KEEP_THREADS / 16);
  uint4 w[PER];
  bool moves[PER];
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    const int i = row + c * (KEEP_THREADS / 16);
    const int from = i < p.n ? p.path[b * p.path_sb + i] : -1;
    moves[c] = from >= 0 && from < p.n && from != i && ctx >= 0 && ctx <= p.S - p.n;
    if (moves[c]) w[c] = base[(int64_t(ctx) + from) * (s.ss / 8)];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < PER; ++c)
    if (moves[c]) base[(int64_t(ctx) + row + c * (KEEP_THREADS / 16)) * (s.ss / 8)] = w[c];
}

// ---- eviction -----------------------------------------------------------------------------------------------
constexpr int EVICT_THREADS = 1024;
constexpr int EVICT_WARPS = EVICT_THREADS / 32;
constexpr int EVICT_MAX_CLUSTER = 8;
constexpr int EVICT_SMEM_KEYS = 48 * 1024;       // order keys one CTA holds in shared memory; longer parts are read again

struct EvictParams {
  const __nv_bfloat16* k;      // (B, S, Hkv, 128) by strides
  const __nv_bfloat16* v;
  const float* weights;        // (B, Hkv, S) by strides, unit stride over keys
  const int* lengths;          // (B) rows in use, null: S
  __nv_bfloat16* k2;           // (B, keep, Hkv, 128) by strides
  __nv_bfloat16* v2;
  float* weights2;             // (B, Hkv, keep) by strides, unit stride over keys
  int* kept;                   // (B, Hkv, keep) contiguous
  TensorView ks, vs, k2s, v2s;
  int64_t weights_sb, weights_sh, weights2_sb, weights2_sh;
  int S, Hkv, keep, recent;
  int cluster, part;           // CTAs per (batch, head), keys per CTA
  int in_smem;                 // a CTA's part fits EVICT_SMEM_KEYS
};

// Weights as unsigned numbers of the same order; both zeros are equal, NaN is above everything.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(w + 0.f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// Picks the rows of one (batch, head) that stay: the last `recent` in use and the heaviest of the others, ties to the
// lowest row, `keep` in all. A cluster holds the weights, a contiguous part per CTA, a contiguous part of that per
// warp. The weight of the last row that stays is found digit by digit, eight bits at a time, from histograms that are
// summed over the cluster; then one pass numbers the rows that stay.
__global__ void __launch_bounds__(EVICT_THREADS) evict_select_kernel(const __grid_constant__ EvictParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ uint32_t evict_keys[];
  __shared__ int hist[256], total[256];
  __shared__ int warp_above[EVICT_WARPS], warp_ties[EVICT_WARPS];
  __shared__ int cta_above, cta_ties;
  __shared__ int digit_s, need_s;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % p.cluster, u = blockIdx.x / p.cluster;
  const int hk = u % p.Hkv, b = u / p.Hkv;
  const int used = p.lengths ? min(max(p.lengths[b], 0), p.S) : p.S;
  const float* const w = p.weights + b * p.weights_sb + hk * p.weights_sh;
  int* const kept = p.kept + int64_t(u) * p.keep;
  float* const w2 = p.weights2 + b * p.weights2_sb + hk * p.weights2_sh;

  if (used <= p.keep) {                                            // all stay
    for (int i = rank * EVICT_THREADS + tid; i < p.keep; i += p.cluster * EVICT_THREADS) {
      kept[i] = i < used ? i : -1;
      w2[i] = i < used ? w[i] : 0.f;
    }
    return;                                                        // the whole cluster
  }
  const int old = used - p.recent;                                 // rows that have to earn their place
  int need = p.keep - p.recent;                                    // how many of them stay; less than old
  const int begin = int(int64_t(rank) * p.part < old ? int64_t(rank) * p.part : old);
  const int end = min(old - begin, p.part) + begin;
  if (p.in_smem)
    for (int i = begin + tid; i < end; i += EVICT_THREADS) evict_keys[i - begin] = order_key(w[i]);
  auto key_at = [&](int i) { return p.in_smem ? evict_keys[i - begin] : order_key(w[i]); };

  uint32_t prefix = 0, mask = 0;                                   // digits of the last kept row's key found so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i0 = begin + warp * 32; i0 < end; i0 += EVICT_THREADS) {
      const int i = i0 + lane;
      const uint32_t key = i < end ? key_at(i) : 0u;
      const bool in = i < end && (key & mask) == prefix;
      const uint32_t digit = in ? (key >> shift) & 255u : 256u;
      const uint32_t same = __match_any_sync(0xffffffffu, digit);  // one addition per digit of a warp
      if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
    }
    cluster.sync();
    if (tid < 256) {
      int sum = 0;
      for (int c = 0; c < p.cluster; ++c) sum += *cluster.map_shared_rank(&hist[tid], c);
      total[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {                                               // the digit at which `need` rows are reached from above
      int mine[8], sum = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) sum += mine[c] = total[255 - (lane * 8 + c)];
      int above = sum;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, above, d);
        if (lane >= d) above += y;
      }
      above -= sum;
      if (above < need && above + sum >= need) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (above < need && above + mine[c] >= need) { digit_s = 255 - (lane * 8 + c); need_s = need - above; }
          above += mine[c];
        }
      }
      if (need == 0 && lane == 0) { digit_s = 255; need_s = 0; }
    }
    cluster.sync();                                                // histograms are free again, digit and need are there
    prefix |= uint32_t(digit_s) << shift;
    mask |= 255u << shift;
    need = need_s;
    __syncthreads();
  }
  // `need` rows of key `prefix` stay, the lowest ones, and all above it (none, where nothing had to be found)
  const bool none = p.keep == p.recent;
  const int warp_part = (p.part + EVICT_WARPS - 1) / EVICT_WARPS;
  const int wb = min(begin + warp * warp_part, end), we = min(wb + warp_part, end);
  int above = 0, ties = 0;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < we ? key_at(i) : 0u;
    above += __popc(__ballot_sync(0xffffffffu, i < we && !none && key > prefix));
    ties += __popc(__ballot_sync(0xffffffffu, i < we && !none && key == prefix));
  }
  if (lane == 0) { warp_above[warp] = above; warp_ties[warp] = ties; }
  __syncthreads();
  if (tid == 0) {
    int a = 0, t = 0;
    for (int c = 0; c < EVICT_WARPS; ++c) { a += warp_above[c]; t += warp_ties[c]; }
    cta_above = a;
    cta_ties = t;
  }
  cluster.sync();
  above = ties = 0;
  for (int c = 0; c < rank; ++c) {
    above += *cluster.map_shared_rank(&cta_above, c);
    ties += *cluster.map_shared_rank(&cta_ties, c);
  }
  for (int c = 0; c < warp; ++c) { above += warp_above[c]; ties += warp_ties[c]; }
  const uint32_t lower = (1u << lane) - 1u;
  for (int i0 = wb; i0 < we; i0 += 32) {
    const int i = i0 + lane;
    const uint32_t key = i < we ? key_at(i) : 0u;
    const bool is_above = i < we && !none && key > prefix, is_tie = i < we && !none && key == prefix;
    const uint32_t va = __ballot_sync(0xffffffffu, is_above), vt = __ballot_sync(0xffffffffu, is_tie);
    const int tie = ties + __popc(vt & lower);
    if (is_above || (is_tie && tie < need)) {
      const int at = above + __popc(va & lower) + min(tie, need);
      kept[at] = i;
      w2[at] = w[i];
    }
    above += __popc(va);
    ties += __popc(vt);
  }
  for (int i = rank * EVICT_THREADS + tid; i < p.recent; i += p.cluster * EVICT_THREADS) {
    kept[p.keep - p.recent + i] = old + i;
    w2[p.keep - p.recent + i] = w[old + i];
  }
  cluster.sync();                                                  // nobody leaves while its counts are read
}

// Rows of K and V into their new places. Sixteen threads a row, EVICT_ROWS rows each; rows that do not exist become zeros.
constexpr int EVICT_COPY_THREADS = 256;
constexpr int EVICT_ROWS = 2;
__global__ void __launch_bounds__(EVICT_COPY_THREADS) evict_copy_kernel(const __grid_constant__ EvictParams p) {
  constexpr int STEP = EVICT_COPY_THREADS / 16;
  const int piece = threadIdx.x & 15;
  const int per_unit = (p.keep + STEP * EVICT_ROWS - 1) / (STEP * EVICT_ROWS);
  const int u = blockIdx.x / per_unit;
  const int first = (blockIdx.x - u * per_unit) * (STEP * EVICT_ROWS) + (threadIdx.x >> 4);
  const int hk = u % p.Hkv, b = u / p.Hkv;
  const uint4* const k = reinterpret_cast<const uint4*>(p.k + b * p.ks.sb + hk * p.ks.sh) + piece;
  const uint4* const v = reinterpret_cast<const uint4*>(p.v + b * p.vs.sb + hk * p.vs.sh) + piece;
  uint4* const k2 = reinterpret_cast<uint4*>(p.k2 + b * p.k2s.sb + hk * p.k2s.sh) + piece;
  uint4* const v2 = reinterpret_cast<uint4*>(p.v2 + b * p.v2s.sb + hk * p.v2s.sh) + piece;
  const int* const kept = p.kept + int64_t(u) * p.keep;
  uint4 kw[EVICT_ROWS], vw[EVICT_ROWS];
#pragma unroll
  for (int c = 0; c < EVICT_ROWS; ++c) {
    const int i = first + c * STEP;
    const int from = i < p.keep ? kept[i] : -1;
    kw[c] = vw[c] = make_uint4(0u, 0u, 0u, 0u);
    if (from >= 0) { kw[c] = k[from * (p.ks.ss / 8)]; vw[c] = v[from * (p.vs.ss / 8)]; }
  }
#pragma unroll
  for (int c = 0; c < EVICT_ROWS; ++c) {
    const int i = first + c * STEP;
    if (i < p.keep) { k2[i * (p.k2s.ss / 8)] = kw[c]; v2[i * (p.v2s.ss / 8)] = vw[c]; }
  }
}

}  // namespace intra
