// Attention of a few tokens per sequence - drafted tokens that form a tree, or a chain - over the sequence's cache.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j that token i sees: all keys before the tokens' own,
//   its ancestors among them, itself; less the keys a boolean mask hides.
//
// The rows of a KV head are its tokens times its query heads; row r is head r % rep of token r / rep. What bounds
// it: reading K and V once (512 bytes per key and KV head) and, with many rows, the products.
//
// tree_mma_kernel is for up to 32 rows per pass over the keys: the decode kernel's structure (decode_kernel.cuh) with
// full 16-row operands. Each warp streams blocks of 16 keys through a ring of its own and keeps MT tiles of 16 rows in
// registers; probabilities are multiplied as two bf16 numbers each (16 significant bits, two MMAs).
#pragma once
#include <cooperative_groups.h>
#include <math_constants.h>
#include <stdint.h>

#include "attn_kernel.cuh"
#include "warp_mma.cuh"

namespace intra {

constexpr int TREE_MAX_TOKENS = 64;              // ancestors of a token fit a 64-bit word
constexpr int TREE_WARPS = 4;
constexpr int TREE_THREADS = 32 * TREE_WARPS;
constexpr int TREE_CTAS_PER_SM = 2;
constexpr int TREE_STAGES = 3;
constexpr int TREE_BLOCK = 16;                   // keys a warp takes at a time
constexpr int TREE_TILE = TREE_BLOCK * HEAD_DIM * 2;
constexpr int TREE_RING_BYTES = TREE_WARPS * TREE_STAGES * 2 * TREE_TILE;
constexpr int TREE_MAX_BLOCKS = TREE_THREADS;    // key blocks one CTA can be dealt

struct TreeParams {
  const __nv_bfloat16* q;      // (B, H, n, 128) by strides
  const __nv_bfloat16* k;      // (B, S, Hkv, 128) by strides
  const __nv_bfloat16* v;
  const int* parents;          // n per sequence, null: each token follows the one before it
  const int* lengths;          // keys before the tokens' own, per sequence; null: S - n
  const uint8_t* mask;         // (B, n, S) by strides, nonzero = visible; null: no further mask
  __nv_bfloat16* o;            // (B, n, H, 128) contiguous
  float* scratch;              // partial results where one cluster does not hold a unit
  int64_t q_sb, q_sh, q_sn;
  TensorView ks, vs;
  int64_t parents_sb;
  int all_own;                 // tokens see all n own keys: the mask decides alone
  int64_t mask_sb, mask_sn, mask_ss;
  int mask_vec;                // 16 mask bytes of a key block can be loaded at once
  // tree_umma_kernel.cuh: the mask as bits, a word for 32 keys ([sequence][token or 1][word]), the same of the keys any token
  // sees, and a bit for each key tile that holds such keys ([sequence][64-bit word]); null: no mask
  const uint32_t* bits;
  const uint32_t* any;
  const uint8_t* live;
  int bits_tokens, bits_words, live_words;
  int pair;                    // units of 256 rows
  int S, H, Hkv, n;
  int row_groups;              // passes over the keys, each for up to 16 * MT rows
  int cluster, n_clusters;
  float scale_log2;
};

template <int MT>
constexpr int TREE_Q_BYTES = MT * 16 * HEAD_DIM * 2;
template <int MT>
constexpr int TREE_PARTIAL = MT * 16 * (HEAD_DIM + 2);       // floats of one cluster's partial result in the scratch buffer
// Dynamic shared memory: rings (the merge's rows at the end), query tile, with a mask its bits per block and token.
template <int MT>
constexpr int tree_smem_bytes(int mask_tokens) { return TREE_RING_BYTES + TREE_Q_BYTES<MT> + mask_tokens * TREE_MAX_BLOCKS * 2; }

// Keys before the tokens' own. A length that leaves the tokens no room is brought into range, so that no key outside the
// cache is read whatever it says.
__device__ __forceinline__ int tree_context(const TreeParams& p, int b) {
  const int most = p.S - p.n;
  return p.lengths ? min(max(p.lengths[b], 0), most) : most;
}

// Which of the n tokens each token sees, itself included, as bits; called by at least n threads of a CTA of which every
// thread arrives. A parent that is not an earlier token ends the walk. Pointer doubling: six rounds for 64 tokens.
__device__ __forceinline__ void tree_ancestors(const TreeParams& p, int b, int tid, unsigned long long* anc, int8_t* up) {
  if (p.all_own || p.parents == nullptr) {
    if (tid < p.n) anc[tid] = (2ull << (p.all_own ? p.n - 1 : tid)) - 1ull;
    __syncthreads();
    return;
  }
  if (tid < p.n) {
    const int parent = p.parents[b * p.parents_sb + tid];
    up[tid] = int8_t(parent >= 0 && parent < tid ? parent : -1);
    anc[tid] = 1ull << tid;
  }
  __syncthreads();
  for (int reach = 1; reach < p.n; reach *= 2) {
    unsigned long long more = 0;
    int next = -1;
    if (tid < p.n && up[tid] >= 0) {
      more = anc[up[tid]];
      next = up[up[tid]];
    }
    __syncthreads();
    if (tid < p.n) {
      anc[tid] |= more;
      up[tid] = int8_t(next);
    }
    __syncthreads();
  }
}

template <int MT>
__global__ void __launch_bounds__(TREE_THREADS, TREE_CTAS_PER_SM) tree_mma_kernel(const __grid_constant__ TreeParams p) {
  namespace cg = cooperative_groups;
  constexpr int ROWS = 16 * MT;
  extern __shared__ __align__(1024) uint8_t tree_smem[];
  __shared__ float part_m[TREE_WARPS][ROWS], part_l[TREE_WARPS][ROWS];
  __shared__ float cta_m[ROWS], cta_l[ROWS];
  __shared__ unsigned long long anc[TREE_MAX_TOKENS];
  __shared__ int8_t up[TREE_MAX_TOKENS];
  __shared__ int live_key[TREE_MAX_BLOCKS];                        // with a mask: first key of the blocks somebody sees ...
  __shared__ uint16_t live_keys[TREE_MAX_BLOCKS], live_at[TREE_MAX_BLOCKS];   // ... which keys, and the block's place in the bits
  __shared__ int warp_live[TREE_WARPS];
  uint8_t* const q_tile = tree_smem + TREE_RING_BYTES;
  uint16_t* const mask_bits = reinterpret_cast<uint16_t*>(q_tile + TREE_Q_BYTES<MT>);   // [block][token]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, j = lane & 3;
  const int rank = blockIdx.x % p.cluster;
  const int group = blockIdx.x / p.cluster;                        // cluster number
  const int u = group / p.n_clusters;                              // (batch, KV head, row group)
  const int row0 = (u % p.row_groups) * ROWS;
  const int hk = (u / p.row_groups) % p.Hkv;
  const int b = u / (p.row_groups * p.Hkv);
  const int rep = p.H / p.Hkv;
  const int n_rows = min(p.n * rep - row0, ROWS);

  const int ctx = tree_context(p, b);
  const int n_keys = ctx + p.n;
  const int n_dealt = p.cluster * p.n_clusters;
  const int first_blk = (group % p.n_clusters) * p.cluster + rank;
  const int n_blk = (n_keys + TREE_BLOCK - 1) / TREE_BLOCK;
  int n_live = first_blk < n_blk ? (n_blk - 1 - first_blk) / n_dealt + 1 : 0;
  auto block_bits = [&](int key0) { return n_keys - key0 >= TREE_BLOCK ? 0xffffu : (1u << (n_keys - key0)) - 1u; };

  // ---- with a mask: its bits for this CTA's blocks, and which blocks and keys any of the tokens sees ----------
  if (p.mask != nullptr) {
    const int dealt = n_live;
    const int m_tokens = p.mask_sn == 0 ? 1 : p.n;
    for (int e = tid; e < dealt * m_tokens; e += TREE_THREADS) {
      const int t = e / m_tokens, i = e - t * m_tokens;
      const int key0 = (first_blk + t * n_dealt) * TREE_BLOCK;
      const uint32_t there = block_bits(key0);
      const uint8_t* m = p.mask + b * p.mask_sb + i * p.mask_sn + key0 * p.mask_ss;
      uint32_t seen = 0;
      if (p.mask_vec && there == 0xffffu) {
        const uint4 w = *reinterpret_cast<const uint4*>(m);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int c = 0; c < TREE_BLOCK; ++c) seen |= ((ws[c >> 2] >> (8 * (c & 3))) & 0xffu) != 0u ? 1u << c : 0u;
      } else {
        for (int c = 0; c < TREE_BLOCK; ++c)
          if ((there >> c) & 1u) seen |= m[c * p.mask_ss] != 0 ? 1u << c : 0u;
      }
      mask_bits[e] = uint16_t(seen & there);
    }
    __syncthreads();
    uint32_t keys = 0;
    if (tid < dealt)
      for (int i = 0; i < m_tokens; ++i) keys |= mask_bits[tid * m_tokens + i];
    const uint32_t vote = __ballot_sync(0xffffffffu, keys != 0u);
    if (lane == 0) warp_live[warp] = __popc(vote);
    __syncthreads();
    int at = __popc(vote & ((1u << lane) - 1u));
    for (int w = 0; w < warp; ++w) at += warp_live[w];
    if (keys != 0u) {
      live_key[at] = (first_blk + tid * n_dealt) * TREE_BLOCK;
      live_keys[at] = uint16_t(keys);
      live_at[at] = uint16_t(tid * m_tokens);
    }
    __syncthreads();
    n_live = 0;
#pragma unroll
    for (int w = 0; w < TREE_WARPS; ++w) n_live += warp_live[w];
  }
  auto block = [&](int e, uint32_t& seen) {                        // first key of the CTA's e-th block
    if (p.mask != nullptr) { seen = live_keys[e]; return live_key[e]; }
    const int key0 = (first_blk + e * n_dealt) * TREE_BLOCK;
    seen = block_bits(key0);
    return key0;
  };

  // ---- this warp streams blocks warp, warp + TREE_WARPS, ... -----------------------------------------------
  const uint32_t ring = ptx::smem_u32(tree_smem) + warp * (TREE_STAGES * 2 * TREE_TILE);
  const int half = lane >> 4, piece = lane & 15;                   // a copy instruction takes two rows
  const __nv_bfloat16* const kb = p.k + b * p.ks.sb + hk * p.ks.sh + piece * 8;
  const __nv_bfloat16* const vb = p.v + b * p.vs.sb + hk * p.vs.sh + piece * 8;
  auto fetch = [&](int e, int stage) {                             // always one commit group, possibly empty
    if (e < n_live) {
      uint32_t seen;
      const int key0 = block(e, seen);
      const uint32_t dst = ring + stage * (2 * TREE_TILE);
      const __nv_bfloat16* kr = kb + int64_t(key0 + half) * p.ks.ss;
      const __nv_bfloat16* vr = vb + int64_t(key0 + half) * p.vs.ss;
#pragma unroll
      for (int i = 0; i < TREE_BLOCK; i += 2) {                    // keys nobody sees become zeros and are not read
        const uint32_t bytes = (seen >> (i + half)) & 1u ? 16u : 0u;
        const uint32_t off = row_piece(i + half, piece);
        ptx::cp_async_16(dst + off, bytes ? kr + i * p.ks.ss : p.k, bytes);
        ptx::cp_async_16(dst + TREE_TILE + off, bytes ? vr + i * p.vs.ss : p.v, bytes);
      }
    }
    ptx::cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < TREE_STAGES - 1; ++s) fetch(warp + s * TREE_WARPS, s);

  for (int e = tid; e < ROWS * 16; e += TREE_THREADS) {            // query rows; those past the end are zeros
    const int r = e >> 4, c = e & 15;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (r < n_rows) {
      const int token = (row0 + r) / rep, head = hk * rep + (row0 + r) % rep;
      w = *reinterpret_cast<const uint4*>(p.q + b * p.q_sb + head * p.q_sh + token * p.q_sn + c * 8);
    }
    *reinterpret_cast<uint4*>(q_tile + row_piece(r, c)) = w;
  }
  tree_ancestors(p, b, tid, anc, up);                              // its barriers cover the query tile, too

  int token_of[MT][2];                                             // token of rows g and g + 8 of each tile
  float m_run[MT][2], l_run[MT][2];                                // l_run: this lane's keys only
  float o[MT][16][4];                                              // dims 8 t + 2 j, + 1 of rows g, g + 8
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) token_of[mt][h] = min(row0 + mt * 16 + 8 * h + g, p.n * rep - 1) / rep;

  // ldmatrix row addresses: K matrices are (keys 0-7 | 8-15) x (dims 0-7 | 8-15) of a step, V the same transposed, Q
  // (rows 0-7 | 8-15) x (dims 0-7 | 8-15)
  const int mi = lane >> 3, mr = lane & 7;
  const int k_row = (mi >> 1) * 8 + mr, v_row = (mi & 1) * 8 + mr;
  const uint32_t qt = ptx::smem_u32(q_tile);
  const bool masked = p.mask != nullptr;
  // An infinite or NaN value row makes every row's sum NaN, also those of tokens that do not see it (zero times infinity).
  // So a warp whose sums are not finite takes its keys once more, key by key, each only to the rows that see it.
  for (int attempt = 0; attempt < 2; ++attempt) {
    const bool one_by_one = attempt == 1;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      m_run[mt][0] = m_run[mt][1] = -CUDART_INF_F;
      l_run[mt][0] = l_run[mt][1] = 0.f;
#pragma unroll
      for (int t = 0; t < 16; ++t) o[mt][t][0] = o[mt][t][1] = o[mt][t][2] = o[mt][t][3] = 0.f;
    }
    if (one_by_one) {
#pragma unroll
      for (int s = 0; s < TREE_STAGES - 1; ++s) fetch(warp + s * TREE_WARPS, s);
    }
    int stage = 0;
    for (int e = warp; e < n_live; e += TREE_WARPS) {
      ptx::cp_async_wait<TREE_STAGES - 2>();
      __syncwarp();                                                  // every lane's copies of this block have landed, and
      fetch(e + (TREE_STAGES - 1) * TREE_WARPS, (stage + TREE_STAGES - 1) % TREE_STAGES);   // all are done with the last one
      const uint32_t kt = ring + stage * (2 * TREE_TILE), vt = kt + TREE_TILE;
      float s[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][0][i] = s[mt][1][i] = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        uint32_t r[4];
        ldmatrix_x4(kt + row_piece(k_row, 2 * t + (mi & 1)), r);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a[4];
          ldmatrix_x4(qt + row_piece(mt * 16 + v_row, 2 * t + (mi >> 1)), a);
          mma_m16n8k16(s[mt][0], a[0], a[1], a[2], a[3], r[0], r[1]);
          mma_m16n8k16(s[mt][1], a[0], a[1], a[2], a[3], r[2], r[3]);
        }
      }
      uint32_t seen;
      const int key0 = block(e, seen);
      const bool plain = !masked && key0 + TREE_BLOCK <= ctx;        // every token sees the whole block
      bool grow_any = false;
      float alpha[MT][2], x[MT][2][4];
      uint32_t row_bits[MT][2];                                      // keys each row sees
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t bits = seen;
          if (!plain) {
            if (masked) bits = mask_bits[live_at[e] + (p.mask_sn == 0 ? 0 : token_of[mt][h])];
            if (key0 + TREE_BLOCK > ctx) {                           // bits of the tokens' own keys, from key0 on
              const unsigned long long own = anc[token_of[mt][h]];
              const int at = key0 - ctx;
              const uint32_t tree = at >= 0 ? (at < 64 ? uint32_t(own >> at) : 0u) : uint32_t(own << -at) | ((1u << -at) - 1u);
              bits &= tree;
            }
          }
          row_bits[mt][h] = bits;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = 2 * j + (i & 1) + 8 * (i >> 1);
            x[mt][h][i] = (bits >> key) & 1u ? s[mt][i >> 1][2 * h + (i & 1)] * p.scale_log2 : -CUDART_INF_F;
          }
          float m_blk = fmaxf(fmaxf(x[mt][h][0], x[mt][h][1]), fmaxf(x[mt][h][2], x[mt][h][3]));
          m_blk = fmaxf(m_blk, __shfl_xor_sync(0xffffffffu, m_blk, 1));
          m_blk = fmaxf(m_blk, __shfl_xor_sync(0xffffffffu, m_blk, 2));
          // the maximum moves only when the scores outgrow it by 2^8; until then probabilities are merely scaled
          const bool grow = m_blk > m_run[mt][h] + RESCALE_THRESHOLD;
          alpha[mt][h] = grow ? merge_weight(m_run[mt][h], m_blk) : 1.f;
          if (grow) m_run[mt][h] = m_blk;
          grow_any |= grow;
        }
      }
      if (__any_sync(0xffffffffu, grow_any)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            l_run[mt][h] *= alpha[mt][h];
#pragma unroll
            for (int t = 0; t < 16; ++t) {
              o[mt][t][2 * h] *= alpha[mt][h];
              o[mt][t][2 * h + 1] *= alpha[mt][h];
            }
          }
        }
      }
      uint32_t hi[MT][4], lo[MT][4];                                 // A operand: (row half, key half) = (0,0) (1,0) (0,1) (1,1)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float base = m_run[mt][h] == -CUDART_INF_F ? 0.f : m_run[mt][h];
          float pr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) pr[i] = ptx::ex2(x[mt][h][i] - base);
          l_run[mt][h] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
          split_bf16(pr[0], pr[1], hi[mt][h], lo[mt][h]);
          split_bf16(pr[2], pr[3], hi[mt][2 + h], lo[mt][2 + h]);
        }
      }
      if (one_by_one) {
        for (int c = 0; c < TREE_BLOCK; ++c) {
          const int from = (lane & ~3) | ((c & 7) >> 1);             // the lane that has this key's probabilities
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t ph = __shfl_sync(0xffffffffu, c < 8 ? hi[mt][h] : hi[mt][2 + h], from);
              const uint32_t pl = __shfl_sync(0xffffffffu, c < 8 ? lo[mt][h] : lo[mt][2 + h], from);
              const float prob = __uint_as_float(c & 1 ? ph & 0xffff0000u : ph << 16) + __uint_as_float(c & 1 ? pl & 0xffff0000u : pl << 16);
              if ((row_bits[mt][h] >> c) & 1u) {
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                  uint32_t w;
                  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vt + row_piece(c, t) + 4 * j) : "memory");
                  o[mt][t][2 * h] += prob * __uint_as_float(w << 16);
                  o[mt][t][2 * h + 1] += prob * __uint_as_float(w & 0xffff0000u);
                }
              }
            }
          }
        }
      } else
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        uint32_t r[4];
        ldmatrix_x4_trans(vt + row_piece(v_row, 2 * t + (mi >> 1)), r);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_m16n8k16(o[mt][2 * t], hi[mt][0], hi[mt][1], hi[mt][2], hi[mt][3], r[0], r[1]);
          mma_m16n8k16(o[mt][2 * t + 1], hi[mt][0], hi[mt][1], hi[mt][2], hi[mt][3], r[2], r[3]);
          mma_m16n8k16(o[mt][2 * t], lo[mt][0], lo[mt][1], lo[mt][2], lo[mt][3], r[0], r[1]);
          mma_m16n8k16(o[mt][2 * t + 1], lo[mt][0], lo[mt][1], lo[mt][2], lo[mt][3], r[2], r[3]);
        }
      }
      stage = stage + 1 == TREE_STAGES ? 0 : stage + 1;
    }
    ptx::cp_async_wait<0>();
    __syncwarp();
    bool finite = true;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) finite = finite && fabsf(o[mt][t][i]) < CUDART_INF_F;
    if (!__any_sync(0xffffffffu, !finite)) break;
  }

  // ---- merge: lanes of a row, warps, CTAs of the cluster --------------------------------------------------
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = l_run[mt][h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (j == 0) { part_m[warp][mt * 16 + 8 * h + g] = m_run[mt][h]; part_l[warp][mt * 16 + 8 * h + g] = l; }
    }
  __syncthreads();                                                 // the rings are free
  constexpr int ROW = HEAD_DIM + 8;                                // rows start 8 banks apart
  float* const part_o = reinterpret_cast<float*>(tree_smem);       // [warp][row][ROW]
  float* const cta_o = part_o + TREE_WARPS * ROWS * ROW;           // [row][HEAD_DIM], read by the cluster
  static_assert((TREE_WARPS * ROWS * ROW + ROWS * HEAD_DIM) * 4 <= TREE_RING_BYTES, "the merge's rows fit the rings");
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < 16; ++t)
        *reinterpret_cast<float2*>(part_o + (warp * ROWS + mt * 16 + 8 * h + g) * ROW + 8 * t + 2 * j) =
            make_float2(o[mt][t][2 * h], o[mt][t][2 * h + 1]);
  __syncthreads();
  for (int r = 0; r < n_rows; ++r) {                               // thread = dim
    float m_all = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < TREE_WARPS; ++w) m_all = fmaxf(m_all, part_m[w][r]);
    float acc = 0.f, l_all = 0.f;
#pragma unroll
    for (int w = 0; w < TREE_WARPS; ++w) {
      const float f = merge_weight(part_m[w][r], m_all);
      acc += f * part_o[(w * ROWS + r) * ROW + tid];
      l_all += f * part_l[w][r];
    }
    cta_o[r * HEAD_DIM + tid] = acc;
    if (tid == 0) { cta_m[r] = m_all; cta_l[r] = l_all; }
  }
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  for (int r = rank; r < n_rows; r += p.cluster) {
    float m_all = -CUDART_INF_F;
    for (int c = 0; c < p.cluster; ++c) m_all = fmaxf(m_all, *cluster.map_shared_rank(&cta_m[r], c));
    float acc = 0.f, l_all = 0.f;
#pragma unroll 4
    for (int c = 0; c < p.cluster; ++c) {
      const float f = merge_weight(*cluster.map_shared_rank(&cta_m[r], c), m_all);
      acc += f * *cluster.map_shared_rank(cta_o + r * HEAD_DIM + tid, c);
      l_all += f * *cluster.map_shared_rank(&cta_l[r], c);
    }
    if (p.n_clusters == 1) {
      const int token = (row0 + r) / rep, head = hk * rep + (row0 + r) % rep;
      p.o[((int64_t(b) * p.n + token) * p.H + head) * HEAD_DIM + tid] = __float2bfloat16(l_all == 0.f ? 0.f : acc / l_all);
    } else {
      float* part = p.scratch + int64_t(group) * TREE_PARTIAL<MT> + r * (HEAD_DIM + 2);
      part[tid] = acc;
      if (tid == 0) { part[HEAD_DIM] = m_all; part[HEAD_DIM + 1] = l_all; }
    }
  }
  cluster.sync();                                                  // nobody leaves while its shared memory is read
}

// The clusters' partial results of one row -> output row. One CTA per (batch, token, head), thread = dim.
template <int MT>
__global__ void __launch_bounds__(HEAD_DIM) tree_merge_kernel(const __grid_constant__ TreeParams p) {
  const int h = blockIdx.x % p.H;
  const int token = (blockIdx.x / p.H) % p.n, b = blockIdx.x / (p.H * p.n);
  const int rep = p.H / p.Hkv, row = token * rep + h % rep;
  const int u = (b * p.Hkv + h / rep) * p.row_groups + row / (16 * MT);
  const float* part = p.scratch + int64_t(u) * p.n_clusters * TREE_PARTIAL<MT> + row % (16 * MT) * (HEAD_DIM + 2);
  float m_all = -CUDART_INF_F;
  for (int c = 0; c < p.n_clusters; ++c) m_all = fmaxf(m_all, part[int64_t(c) * TREE_PARTIAL<MT> + HEAD_DIM]);
  float acc = 0.f, l_all = 0.f;
#pragma unroll 4
  for (int c = 0; c < p.n_clusters; ++c) {
    const float* pc = part + int64_t(c) * TREE_PARTIAL<MT>;
    const float f = merge_weight(pc[HEAD_DIM], m_all);
    acc += f * pc[threadIdx.x];
    l_all += f * pc[HEAD_DIM + 1];
  }
  p.o[int64_t(blockIdx.x) * HEAD_DIM + threadIdx.x] = __float2bfloat16(l_all == 0.f ? 0.f : acc / l_all);
}

}  // namespace intra
