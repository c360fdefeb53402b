// Verification of drafted tokens against the target model's probabilities, from given random numbers.
//
// Node 0 of a sequence's tree is the token sampled last; the walk starts there. A child c of the current node, in
// index order, with token x, is accepted iff u_c q(x) Z < R(x); R is what is left of the current node's target row p and Z
// its weight, R = p and Z = 1 to begin with. A rejection takes the drafts' distribution out,
//
//   R <- max(R - Z q, 0),  Z <- sum R            (both stay where nothing would be left),
//
// so that tokens come out distributed as p whatever q is (R / Z is the target's distribution given the rejections). When no child is accepted the walk ends, and one more token
// is drawn from R: the smallest t with R(0) + .. + R(t) > u_0 sum R. Drafts without a distribution count as
// certain: q is one at their token. All of it in 64 bits: an error of 2^-24 in a running sum over 10^5 tokens decides
// the token in one draw of a hundred, 2^-53 in none.
//
// A sequence is a thread-block cluster; each CTA holds a contiguous part of the vocabulary, each warp a contiguous part of
// that. Every CTA walks the tree by itself, from the n probabilities of the drafted tokens, fetched at once; only a
// rejection or the final draw reads a row: one pass, its sums exchanged through distributed shared memory. R is
// not stored: it follows from p, q and the weights of the rejections so far.
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attn_kernel.cuh"

namespace intra {

constexpr int VERIFY_MAX_TOKENS = 64;
constexpr int VERIFY_THREADS = 512;
constexpr int VERIFY_WARPS = VERIFY_THREADS / 32;
constexpr int VERIFY_MAX_CLUSTER = 8;

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

template <typename T>
__global__ void __launch_bounds__(VERIFY_THREADS) verify_kernel(const __grid_constant__ VerifyParams p) {
  namespace cg = cooperative_groups;
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

  const int part = (V + p.cluster * VERIFY_WARPS - 1) / (p.cluster * VERIFY_WARPS);      // tokens a warp holds
  const int64_t first = int64_t(rank * VERIFY_WARPS + warp) * part;
  const int begin = int(first < V ? first : V), end = min(V - begin, part) + begin;

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
  // Sum of what is left over the whole row: the same number in every thread of the cluster.
  auto row_sum = [&](int count) {
    double sum = 0.0;
    constexpr int AT_ONCE = 8;                                     // tokens of a lane whose loads are under way together
    int t = begin + lane;
    for (; t + 32 * (AT_ONCE - 1) < end; t += 32 * AT_ONCE) {
      T pt[AT_ONCE], qt[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) pt[e] = p_row[t + 32 * e];
      const bool drawn = draft != nullptr && count > 0;
      if (drawn) {
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) qt[e] = q_row[t + 32 * e];
      }
      double r[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) r[e] = as_double(pt[e]);
      for (int c = 0; c < count; ++c) {
        const double w = -weight[c];
        if (drawn) {
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e) r[e] = fmax(fma(w, as_double(qt[e]), r[e]), 0.0);
        } else {
          const int x = gone[c] >= 0 && gone[c] < V ? int(gone[c]) : -1;
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e) r[e] = t + 32 * e == x ? fmax(w + r[e], 0.0) : r[e];
        }
      }
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) sum += r[e];
    }
    for (; t < end; t += 32) sum += left_at(t, count);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) warp_sum[warp] = sum;
    __syncthreads();
    const int slot = ++passes & 1;                                 // the pass before may still be read elsewhere
    if (tid == 0) {
      double all = 0.0;
      for (int w = 0; w < VERIFY_WARPS; ++w) all += warp_sum[w];
      cta_sum[slot] = all;
    }
    cluster.sync();
    double all = 0.0;
    for (int c = 0; c < p.cluster; ++c) all += *cluster.map_shared_rank(&cta_sum[slot], c);
    summed = count;
    return all;
  };

  if (tid == 0) node[0] = 0;
  for (int i = 1; i < n; ++i) {
    if (parent[i] != at) continue;
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
  double before = 0.0, running = 0.0;
  int owner = -1;
  auto choose = [&](double sum, int who, int& last, double& last_before) {
    if (owner < 0 && running + sum > threshold) { owner = who; before = running; }
    if (sum > 0.0) { last = who; last_before = running; }
    running += sum;
  };
  int last = 0;
  double last_before = 0.0;
  for (int c = 0; c < p.cluster; ++c) choose(*cluster.map_shared_rank(&cta_sum[passes & 1], c), c, last, last_before);
  if (owner < 0) { owner = last; before = last_before; }           // rounding: the last part with any mass
  if (owner == rank) {
    running = last_before = before;
    owner = -1;
    last = 0;
    for (int w = 0; w < VERIFY_WARPS; ++w) choose(warp_sum[w], w, last, last_before);
    if (owner < 0) { owner = last; before = last_before; }
    if (tid == 0) { found = 0x7fffffff; found_last = -1; }
    const int64_t from = int64_t(rank * VERIFY_WARPS + owner) * part;
    const int to = int(from + part < V ? from + part : V), per = (part + VERIFY_THREADS - 1) / VERIFY_THREADS;
    const int t0 = int(from < V ? from : V) + tid * per, t1 = min(t0 + per, to);
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
