// Verification of drafted tokens against the target model's probabilities, from given random numbers.
//
// Node 0 of a sequence's tree is the token sampled last; the walk starts there. A child c of the current node, in
// index order, with token x, is accepted iff u_c q(x) Z < R(x); R is what is left of the current node's target row p and Z
// its weight, R = p and Z = 1 to begin with. A rejection takes the drafts' distribution out,
//
//   R <- max(R - Z q, 0),  Z <- sum R            (both stay where nothing would be left),
//
// so that tokens come out distributed as p whatever q is, if the children of a node were drawn from q independently of one another (R / Z
// is the target's distribution given the rejections; children drawn without replacement follow other distributions). When no child is
// accepted the walk ends, and one more token is drawn from R: the smallest t with R(0) + .. + R(t) > u_0 sum R. Drafts
// without a distribution count as certain: q is one at their token. All of it in 64 bits: an error of 2^-24 in a running
// sum over 10^5 tokens decides the token in one draw of a hundred, 2^-53 in none.
//
// A sequence is a thread-block cluster; each CTA holds a contiguous part of the vocabulary, each warp a contiguous part of
// that. Every CTA walks the tree by itself, from the n probabilities of the drafted tokens, fetched at once; only a
// rejection or the final draw reads a row: one pass, its sums exchanged through distributed shared memory. R is
// not stored: it follows from p, q and the weights of the rejections so far.
//
// What bounds a pass is how much of the rows is under way: every thread copies 16-byte granules VERIFY_AHEAD ahead into slots of
// its own in shared memory (its own copies are all it waits for), and then the arithmetic: 64-bit numbers are made from the bits
// of 32-bit ones by integer multiplications, and compared with zero by their upper words. 32 trees of 26 nodes over 128257 tokens,
// the slowest of which take 4 or 5 passes one after the other: 171 us with a division per rejection and token, 46 without, 42 with
// the granules, 33 so; reading two rows of each once at the copy bandwidth takes 5.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attn_kernel.cuh"
#include "ptx.cuh"

namespace intra {

constexpr int VERIFY_MAX_TOKENS = 64;
constexpr int VERIFY_MAX_VOCABULARY = 1 << 30;   // places in a row, with what a CTA's parts round up, fit 31 bits
constexpr int VERIFY_THREADS = 512;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MAX_CLUSTER = 8;
constexpr int VERIFY_AHEAD = 4;                  // granules of each row a thread has under way
constexpr int VERIFY_SMEM_BYTES = VERIFY_THREADS * VERIFY_AHEAD * 2 * 16;

struct VerifyParams {
  const void* tokens;          // (B, n) by strides, int64 or int32
  const void* target;          // (B, n, V) by strides
  const void* draft;           // (B, n - 1 or n, V) by strides, null: drafts are certain
  const float* uniform;        // (B, n) by strides
  const int* parents;          // n per sequence, null: a chain
  int* accepted;               // (B)
  int* path;                   // (B, n)
  long long* out_tokens;       // (B, n)
  int64_t tokens_sb, target_sb, target_sn, draft_sb, draft_sn, uniform_sb, parents_sb;
  int tokens_wide;             // int64 tokens
  int n, V, cluster;
};

template <typename T> __device__ __forceinline__ double as_double(T x);
template <> __device__ __forceinline__ double as_double(float x) { return x; }
template <> __device__ __forceinline__ double as_double(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ double as_double(__half x) { return __half2float(x); }

// A probability times 2^-896 as a double, from the bits of fp32 by one integer multiplication (the conversion instruction runs at an
// eighth of the rate): the exponent fields differ by that in their bias, and zero and denormals come out right by themselves.
// Negative numbers, minus zero among them, become zero; an infinity or NaN counts as 2^128 or more. Differences are kept to 2^-178 of an unscaled number, so a sum over tokens
// of which none has anything left is zero, and one is positive where some token has.
constexpr double VERIFY_SCALE = 0x1p-896, VERIFY_UNSCALE = 0x1p896;
__device__ __forceinline__ double scaled(float x) { return __longlong_as_double((long long)(max(__float_as_int(x), 0)) * (1 << 29)); }
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }

// The sum over a warp's lanes, the same in all of them.
__device__ __forceinline__ double warp_total(double x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

template <typename T>
__global__ void __launch_bounds__(VERIFY_THREADS, 2) verify_kernel(const __grid_constant__ VerifyParams p) {
  namespace cg = cooperative_groups;
  constexpr int EACH = 16 / sizeof(T);                             // tokens of a granule
  extern __shared__ __align__(16) uint4 verify_smem[];
  __shared__ long long tok[VERIFY_MAX_TOKENS];
  __shared__ int parent[VERIFY_MAX_TOKENS], node[VERIFY_MAX_TOKENS];
  __shared__ double px[VERIFY_MAX_TOKENS], qx[VERIFY_MAX_TOKENS], ux[VERIFY_MAX_TOKENS];
  __shared__ double weight[VERIFY_MAX_TOKENS];                     // Z at each rejection at the current node ...
  __shared__ long long gone[VERIFY_MAX_TOKENS];                    // ... and the token it rejected
  __shared__ double warp_sum[VERIFY_WARPS], scan_sum[VERIFY_WARPS];
  __shared__ double cta_sum[2];                                    // of the last two passes, read by the cluster
  __shared__ int found, found_last;                                // token drawn; the last one with any mass

  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % p.cluster, b = blockIdx.x / p.cluster;
  const int n = p.n, V = p.V;
  const T* const target = static_cast<const T*>(p.target) + b * p.target_sb;
  const T* const draft = p.draft ? static_cast<const T*>(p.draft) + b * p.draft_sb : nullptr;

  if (tid < n) {
    const long long x = p.tokens_wide ? static_cast<const long long*>(p.tokens)[b * p.tokens_sb + tid]
                                      : static_cast<const int*>(p.tokens)[b * p.tokens_sb + tid];
    int up = p.parents ? p.parents[b * p.parents_sb + tid] : tid - 1;
    if (up < 0 || up >= tid) up = -1;                              // no earlier node: never reached
    const bool known = tid > 0 && up >= 0 && x >= 0 && x < V;      // a token outside the vocabulary has no probability
    tok[tid] = x;
    parent[tid] = up;
    px[tid] = known ? as_double(target[up * p.target_sn + x]) : 0.0;
    qx[tid] = draft == nullptr ? 1.0 : known ? as_double(draft[up * p.draft_sn + x]) : 0.0;
    ux[tid] = p.uniform[b * p.uniform_sb + tid];
  }
  __syncthreads();

  int at = 0, accepted = 0, rejections = 0, passes = 0;
  int summed = -1;                                                 // rejections the sums of the last pass stand for
  double Z = 1.0, total = 0.0;
  const T* p_row = target;
  const T* q_row = draft;
  // What is left of the probability p0 of token t after `count` rejections at the current node, q0 being its draft probability.
  auto left = [&](double p0, double q0, long long t, int count) {
    double r = p0;
    for (int c = 0; c < count; ++c) r = fmax(fma(-weight[c], draft != nullptr ? q0 : t == gone[c] ? 1.0 : 0.0, r), 0.0);
    return r;
  };
  auto left_at = [&](int t, int count) {
    return left(as_double(p_row[t]), draft != nullptr && count > 0 ? as_double(q_row[t]) : 0.0, t, count);
  };
  // The current row's granules, the first of which begins `off` tokens before token 0, and those of a warp. They lie on 16-byte
  // boundaries and each holds a token of the row, so none leaves the row's memory page; what else they hold is not used.
  int off = 0, per_warp = 0, granules = 0;
  const uint32_t slots = ptx::smem_u32(verify_smem) + tid * 16;
  constexpr uint32_t SLOT = VERIFY_THREADS * 16;
  // Sum of what is left over the whole row: the same number in every thread of the cluster.
  auto row_sum = [&](int count) {
    const bool drawn = draft != nullptr && count > 0;
    off = int(reinterpret_cast<uintptr_t>(p_row) & 15u) / int(sizeof(T));
    granules = (V + off + EACH - 1) / EACH;
    per_warp = (granules + p.cluster * VERIFY_WARPS - 1) / (p.cluster * VERIFY_WARPS);
    const bool together = drawn && int(reinterpret_cast<uintptr_t>(q_row) & 15u) / int(sizeof(T)) == off;      // else q token by token
    const uint4* const pg = reinterpret_cast<const uint4*>(p_row - off);
    const uint4* const qg = reinterpret_cast<const uint4*>(together ? q_row - off : p_row - off);
    const int g_end = min((rank * VERIFY_WARPS + warp + 1) * per_warp, granules);
    int g = (rank * VERIFY_WARPS + warp) * per_warp + lane;
    auto fetch = [&](int granule, int slot) {                      // always one commit group, possibly empty
      if (granule < g_end) {
        ptx::cp_async_16(slots + slot * 2 * SLOT, pg + granule, 16u);
        if (together) ptx::cp_async_16(slots + (slot * 2 + 1) * SLOT, qg + granule, 16u);
      }
      ptx::cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < VERIFY_AHEAD - 1; ++k) fetch(g + 32 * k, k);
    double part_sum[4] = {0.0, 0.0, 0.0, 0.0};
    for (int slot = 0; g < g_end; g += 32, slot = (slot + 1) % VERIFY_AHEAD) {
      fetch(g + 32 * (VERIFY_AHEAD - 1), (slot + VERIFY_AHEAD - 1) % VERIFY_AHEAD);
      ptx::cp_async_wait<VERIFY_AHEAD - 1>();
      const uint4* const mine = verify_smem + slot * 2 * VERIFY_THREADS + tid;
      const T* const pt = reinterpret_cast<const T*>(mine);
      const T* const qt = reinterpret_cast<const T*>(mine + VERIFY_THREADS);
      const int t0 = g * EACH - off;
      if (t0 < 0 || t0 + EACH > V || (drawn && !together)) {       // the row's ends; rows that lie differently in memory
        for (int e = 0; e < EACH; ++e)
          if (t0 + e >= 0 && t0 + e < V) part_sum[0] += left_at(t0 + e, count) * VERIFY_SCALE;
        continue;
      }
#pragma unroll
      for (int e0 = 0; e0 < EACH; e0 += 4) {
        double r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = scaled(as_float(pt[e0 + e]));
        if (drawn) {
          double q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            q[e] = scaled(as_float(qt[e0 + e]));
            r[e] -= q[e];                                          // the first rejection at a node, whose Z is 1
          }
          for (int c = 1; c < count; ++c) {
            const double w = -weight[c];
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = fma(w, q[e], r[e]);
          }
        } else {
          for (int c = 0; c < count; ++c) {
            const long long x = gone[c] - (t0 + e0);
            if (x < 0 || x > 3) continue;
            const double w = -weight[c];
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = x == e ? fma(w, VERIFY_SCALE, r[e]) : r[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)                                // what has become negative stays so: zero, at the end
          if (__double2hiint(r[e]) >= 0) part_sum[e] += r[e];
      }
    }
    ptx::cp_async_wait<0>();
    double sum = (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
    sum = warp_total(sum) * VERIFY_UNSCALE;
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    const int slot = ++passes & 1;                                 // the pass before may still be read elsewhere
    if (warp == 0) {
      const double all = warp_total(lane < VERIFY_WARPS ? warp_sum[lane] : 0.0);
      if (lane == 0) cta_sum[slot] = all;
    }
    cluster.sync();
    // every warp by itself, a lane for each CTA
    const double all = warp_total(lane < p.cluster ? *cluster.map_shared_rank(&cta_sum[slot], lane) : 0.0);
    summed = count;
    return all;
  };

  if (tid == 0) node[0] = 0;
  const int parent0 = lane < n ? parent[lane] : -1, parent1 = lane + 32 < n ? parent[lane + 32] : -1;
  auto next_child = [&](int after) {                               // of the current node, behind `after`; n: none
    const unsigned long long children = (unsigned long long)(__ballot_sync(0xffffffffu, parent1 == at)) << 32 | __ballot_sync(0xffffffffu, parent0 == at);
    const unsigned long long left_ones = children & ~((2ull << after) - 1ull);
    return left_ones ? __ffsll(left_ones) - 1 : n;
  };
  for (int i = next_child(0); i < n; i = next_child(i)) {
    if (ux[i] * qx[i] * Z < left(px[i], qx[i], tok[i], rejections)) {
      at = i;
      ++accepted;
      if (tid == 0) node[accepted] = i;
      rejections = 0;
      Z = 1.0;
      summed = -1;
      p_row = target + i * p.target_sn;
      if (draft != nullptr) q_row = draft + i * p.draft_sn;
      continue;
    }
    __syncthreads();                                               // everybody is done with the weights so far
    if (tid == 0) { weight[rejections] = Z; gone[rejections] = tok[i]; }
    __syncthreads();
    const double rest = row_sum(rejections + 1);
    if (rest > 0.0) {
      ++rejections;
      Z = total = rest;
    }
  }
  if (summed != rejections) total = row_sum(rejections);

  // ---- the last token: the CTA, the warp's part, the token whose running sum passes the threshold -----------
  const double threshold = ux[0] * total;
  // Which of `count` parts, whose sums the lanes hold, the threshold falls into, and the sum before it. Only a part with any mass is
  // taken, so that a token that has none is not drawn: not by a threshold of zero, and not by the sums' rounding, which differs
  // from lane to lane. Where no part passes the threshold, rounding again, it is the last one with mass.
  auto choose = [&](double sum, int count, double before, int& owner, double& start) {
    double upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += y;
    }
    const bool mass = lane < count && sum > 0.0;
    const uint32_t any = __ballot_sync(0xffffffffu, mass), past = __ballot_sync(0xffffffffu, mass && before + upto > threshold);
    owner = past ? __ffs(past) - 1 : any ? 31 - __clz(any) : 0;
    const double of_others = __shfl_sync(0xffffffffu, upto, owner > 0 ? owner - 1 : 0);
    start = owner > 0 ? before + of_others : before;
  };
  int owner;
  double before;
  choose(lane < p.cluster ? *cluster.map_shared_rank(&cta_sum[passes & 1], lane) : 0.0, p.cluster, 0.0, owner, before);
  if (owner == rank) {
    choose(lane < VERIFY_WARPS ? warp_sum[lane] : 0.0, VERIFY_WARPS, before, owner, before);
    if (tid == 0) { found = 0x7fffffff; found_last = -1; }
    const int g_from = min((rank * VERIFY_WARPS + owner) * per_warp, granules), g_to = min(g_from + per_warp, granules);
    const int to = min(g_to * EACH - off, V), per = (per_warp * EACH + VERIFY_THREADS - 1) / VERIFY_THREADS;
    const int t0 = max(g_from * EACH - off, 0) + tid * per, t1 = min(t0 + per, to);
    double mine = 0.0;
    for (int t = t0; t < t1; ++t) mine += left_at(t, rejections);
    double scan = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= d) scan += y;
    }
    if (lane == 31) scan_sum[warp] = scan;
    __syncthreads();
    double cum = before + (scan - mine);
    for (int w = 0; w < warp; ++w) cum += scan_sum[w];
    for (int t = t0; t < t1; ++t) {
      const double r = left_at(t, rejections);
      cum += r;
      if (r > 0.0) {
        if (cum > threshold) { atomicMin(&found, t); break; }
        atomicMax(&found_last, t);
      }
    }
    __syncthreads();
    if (tid == 0) {
      const int x = found != 0x7fffffff ? found : found_last >= 0 ? found_last : 0;
      p.out_tokens[int64_t(b) * n + accepted] = x;
    }
  }
  if (rank == 0) {
    if (tid == 0) p.accepted[b] = accepted;
    __syncthreads();
    if (tid < n) {
      p.path[int64_t(b) * n + tid] = tid <= accepted ? node[tid] : -1;
      if (tid != accepted) p.out_tokens[int64_t(b) * n + tid] = tid < accepted ? tok[node[tid + 1]] : -1;
    }
  }
  cluster.sync();                                                  // nobody leaves while its sums are read
}

}  // namespace intra
