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
constexpr int EVICT_THREADS = 512;
constexpr int EVICT_WARPS = EVICT_THREADS / 32;
constexpr int EVICT_MAX_CLUSTER = 8;
constexpr int EVICT_SMEM_KEYS = 48 * 1024;       // order keys one CTA holds in shared memory; longer parts are read again
constexpr int EVICT_DIGITS = 3;                  // of 11, 11 and 10 bits: the first one tells weights of one power of two apart
constexpr int EVICT_BINS = 2048;

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
  int cluster;                 // CTAs per (batch, head)
};

// Weights as unsigned numbers of the same order; both zeros are equal, NaN is above everything. Never zero, which pads.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t bits = __float_as_uint(w + 0.f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The weight an order key stands for (minus zero as zero).
__device__ __forceinline__ float weight_of_key(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

// Picks the rows of one (batch, head) that stay: the last `recent` in use and the heaviest of the others, ties to the
// lowest row, `keep` in all. A cluster holds the weights, a contiguous part per CTA, a contiguous part of that per
// warp. The weight of the last row that stays is found digit by digit from histograms that are summed over the cluster
// (one buffer per digit, so that each takes one barrier); then one pass numbers the rows that stay. What bounds it is
// the chain of these steps; adding up one digit for all lanes of a warp is not: with all weights equal, or 99 of 100 zero, calls take what
// they take with weights spread out (8 heads of 16,384 keys 14.6 to 15.0 us, 128 heads 58 to 59, the copy included). 16 x 8 heads of 1600 to 16384 keys: 44 us with digits of 8 bits, warps that add up equal
// digits first (match) and 1024 threads, 17 us so.
template <bool IN_SMEM>
__global__ void __launch_bounds__(EVICT_THREADS, 2) evict_select_kernel(const __grid_constant__ EvictParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint32_t evict_keys[];
  __shared__ int hist[EVICT_DIGITS][EVICT_BINS];
  __shared__ int warp_above[EVICT_WARPS], warp_ties[EVICT_WARPS];
  __shared__ int2 cta_counts;                                      // rows above and ties, read by the cluster
  __shared__ int digit_s, need_s;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % p.cluster, u = blockIdx.x / p.cluster;
  const int hk = u % p.Hkv, b = u / p.Hkv;
  for (int i = tid; i < EVICT_DIGITS * EVICT_BINS; i += EVICT_THREADS) hist[0][i] = 0;
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
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
  const int part = ((old + p.cluster - 1) / p.cluster + 3) & ~3;
  const int begin = int(min(int64_t(rank) * part, int64_t(old))), n = min(part, old - begin);
  const float* const mine_w = w + begin;
  const int n4 = (n + 3) >> 2;
  auto four = [&](int v) {                                         // order keys 4 v .. of this CTA, zeros behind the last
    if constexpr (IN_SMEM) {
      return reinterpret_cast<const uint4*>(evict_keys)[v];
    } else {
      uint32_t k[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k[e] = 4 * v + e < n ? order_key(mine_w[4 * v + e]) : 0u;
      return make_uint4(k[0], k[1], k[2], k[3]);
    }
  };
  auto sync_all = [&] {
    if (p.cluster == 1) __syncthreads();
    else cluster.sync();
  };
  __syncthreads();
  if (IN_SMEM) {                                                   // the first digit on the way
    constexpr int AT_ONCE = 16;                                    // loads under way together, before any is added up
    for (int i0 = tid; i0 < n; i0 += AT_ONCE * EVICT_THREADS) {
      float x[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) x[e] = i0 + e * EVICT_THREADS < n ? mine_w[i0 + e * EVICT_THREADS] : 0.f;
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const int i = i0 + e * EVICT_THREADS;
        if (i >= n) break;
        const uint32_t key = order_key(x[e]);
        evict_keys[i] = key;
        atomicAdd(&hist[0][key >> 21], 1);
      }
    }
    if (tid < 4 * n4 - n) evict_keys[n + tid] = 0u;
  }

  uint32_t prefix = 0, mask = 0;                                   // digits of the last kept row's key found so far
#pragma unroll 1
  for (int d = 0; d < EVICT_DIGITS; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t digits = d == 2 ? 1023u : 2047u;
    if (!IN_SMEM || d > 0) {
#pragma unroll 2
      for (int v = tid; v < n4; v += EVICT_THREADS) {
        const uint4 x = four(v);
        if ((x.x & mask) == prefix && (d > 0 || x.x)) atomicAdd(&hist[d][(x.x >> shift) & digits], 1);
        if ((x.y & mask) == prefix && (d > 0 || x.y)) atomicAdd(&hist[d][(x.y >> shift) & digits], 1);
        if ((x.z & mask) == prefix && (d > 0 || x.z)) atomicAdd(&hist[d][(x.z >> shift) & digits], 1);
        if ((x.w & mask) == prefix && (d > 0 || x.w)) atomicAdd(&hist[d][(x.w >> shift) & digits], 1);
      }
    }
    sync_all();
    // The digit at which `need` rows are reached from above: thread t has the bins 2047 - 4 t and the three below.
    int* const my_bins = &hist[d][EVICT_BINS - 4 - 4 * tid];
    int4 x[EVICT_MAX_CLUSTER];
#pragma unroll
    for (int c = 0; c < EVICT_MAX_CLUSTER; ++c)
      x[c] = c >= p.cluster ? make_int4(0, 0, 0, 0) : p.cluster == 1 ? *reinterpret_cast<const int4*>(my_bins) : *reinterpret_cast<const int4*>(cluster.map_shared_rank(my_bins, c));
    int bins[4] = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < EVICT_MAX_CLUSTER; ++c) { bins[0] += x[c].w; bins[1] += x[c].z; bins[2] += x[c].y; bins[3] += x[c].x; }
    const int mine = bins[0] + bins[1] + bins[2] + bins[3];
    int above = mine;
#pragma unroll
    for (int k = 1; k < 32; k *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, above, k);
      if (lane >= k) above += y;
    }
    if (lane == 31) warp_above[warp] = above;
    if (tid == 0) { digit_s = int(digits); need_s = 0; }           // nothing to find where no row is needed
    __syncthreads();
    above -= mine;
    for (int k = 0; k < warp; ++k) above += warp_above[k];
    if (above < need && above + mine >= need) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (above < need && above + bins[k] >= need) { digit_s = EVICT_BINS - 1 - (4 * tid + k); need_s = need - above; }
        above += bins[k];
      }
    }
    __syncthreads();
    prefix |= uint32_t(digit_s) << shift;
    mask |= digits << shift;
    need = need_s;
    __syncthreads();
  }
  // `need` rows of key `prefix` stay, the lowest ones, and all above it (none, where nothing had to be found)
  const bool none = p.keep == p.recent;
  const int warp_part = (n4 + EVICT_WARPS - 1) / EVICT_WARPS;
  const int wb = min(warp * warp_part, n4), we = min(wb + warp_part, n4);
  // rows above and ties of four keys, in the halves of a word
  auto count = [&](const uint4& x) {
    return (x.x > prefix) + (x.y > prefix) + (x.z > prefix) + (x.w > prefix) +
           (((x.x == prefix) + (x.y == prefix) + (x.z == prefix) + (x.w == prefix)) << 16);
  };
  int above = 0, ties = 0;
  for (int v = wb + lane; v < we; v += 32) {
    const int x = count(four(v));
    above += x & 0xffff;
    ties += x >> 16;
  }
  above = __reduce_add_sync(0xffffffffu, above);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0) { warp_above[warp] = above; warp_ties[warp] = ties; }
  __syncthreads();
  above = lane < warp ? warp_above[lane] : 0;                      // of the warps before this one
  ties = lane < warp ? warp_ties[lane] : 0;
  if (p.cluster > 1) {
    if (warp == 0) {
      const int a = __reduce_add_sync(0xffffffffu, lane < EVICT_WARPS ? warp_above[lane] : 0);
      const int t = __reduce_add_sync(0xffffffffu, lane < EVICT_WARPS ? warp_ties[lane] : 0);
      if (lane == 0) cta_counts = make_int2(a, t);
    }
    cluster.sync();
    if (lane < rank) {                                             // and of the CTAs before
      const int2 x = *cluster.map_shared_rank(&cta_counts, lane);
      above += x.x;
      ties += x.y;
    }
    cluster.barrier_arrive();                                      // the last this CTA reads elsewhere
  }
  above = __reduce_add_sync(0xffffffffu, above);
  ties = __reduce_add_sync(0xffffffffu, ties);
  for (int v0 = wb; v0 < we && !none; v0 += 32) {
    const uint4 x = v0 + lane < we ? four(v0 + lane) : make_uint4(0u, 0u, 0u, 0u);
    const int own = count(x);
    int upto = own;
#pragma unroll
    for (int k = 1; k < 32; k *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, upto, k);
      if (lane >= k) upto += y;
    }
    int a = above + ((upto - own) & 0xffff), t = ties + ((upto - own) >> 16);
    const uint32_t keys[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool is_above = keys[e] > prefix, is_tie = keys[e] == prefix;
      if (is_above || (is_tie && t < need)) {
        const int at = a + min(t, need), i = 4 * (v0 + lane) + e;
        kept[at] = begin + i;
        w2[at] = IN_SMEM ? weight_of_key(keys[e]) : mine_w[i];
      }
      a += is_above;
      t += is_tie;
    }
    upto = __shfl_sync(0xffffffffu, upto, 31);
    above += upto & 0xffff;
    ties += upto >> 16;
  }
  for (int i = rank * EVICT_THREADS + tid; i < p.recent; i += p.cluster * EVICT_THREADS) {
    kept[p.keep - p.recent + i] = old + i;
    w2[p.keep - p.recent + i] = w[old + i];
  }
  if (p.cluster > 1) cluster.barrier_wait();                       // nobody leaves while its counts are read
}

// Rows of K and V into their new places. Sixteen threads a row, EVICT_ROWS rows each; rows that do not exist become zeros.
// It runs at the copy bandwidth: 128 x 2048 rows 42 us, 6.4 TB/s read and written. (Copied by the selection's CTAs, each
// the rows it has numbered, beside other units' selection, the whole call took 61 us instead of 59: too few loads under way.)
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
  cudaGridDependencySynchronize();
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
