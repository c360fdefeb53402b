// Attention of a few tokens per sequence - drafted tokens that form a tree, or a chain, or the one token of a decode step
// that accumulates what each key receives - over the sequence's cache.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j that token i sees: all keys before the tokens' own,
//   its ancestors among them, itself; less the keys a boolean mask hides.
//   weights_j += sum of p_ij over the query heads of the KV head (one token).
//
// The rows of a KV head are its tokens times its query heads; row r is head r % rep of token r / rep. What bounds
// it: reading K and V once (512 bytes per key and KV head).
//
// tree_mma_kernel is for up to 16 rows per pass over the keys. Each warp streams blocks of 16 keys through a ring of its
// own with cp.async, TREE_STAGES - 1 blocks ahead, and never waits for another warp until its CTA's piece of a unit ends
// (tree_list.cuh deals the pieces, with 16 keys a tile); the products are warp-level m16n8k16 MMAs; probabilities are multiplied
// as two bf16 numbers each (16 significant bits), the two sums apart: by two MMAs, or, where a unit has no more than 8 rows
// (PACKED), by one whose other 8 rows carry the low parts.
#pragma once
#include <math_constants.h>
#include <stdint.h>

#include "tree_list.cuh"
#include "warp_mma.cuh"

namespace intra {

constexpr int TREE_ROWS = 16;                    // rows of a unit
constexpr int TREE_WARPS = 4;
constexpr int TREE_THREADS = 32 * TREE_WARPS;
constexpr int TREE_CTAS_PER_SM = 2;
constexpr int TREE_STAGES = 3;
constexpr int TREE_BLOCK = 16;                   // keys a warp takes at a time
constexpr int TREE_TILE = TREE_BLOCK * HEAD_DIM * 2;
constexpr int TREE_RING_BYTES = TREE_WARPS * TREE_STAGES * 2 * TREE_TILE;
constexpr int TREE_Q_BYTES = TREE_ROWS * HEAD_DIM * 2;
constexpr int TREE_CHUNK = TREE_THREADS;         // key blocks whose mask is looked at together
constexpr int TREE_MIN_BLOCKS = 4 * TREE_WARPS;  // of a CTA's part: more parts make the merge longer than they make this kernel shorter
// Blocks that partial results and their merge are worth. Equal parts / 8 / 16, us for 16 rows: 8 units of 7 blocks 13.1 / 7.1 / 7.1,
// of 32 blocks 11.7 / 11.7 / 13.6, 240 units of 32 blocks 23.2 / 18.6 / 18.6, 288 of 63 36.9 / 29.8 / 29.9.
constexpr int TREE_SPLIT_COST = 8;
constexpr int TREE_UNIT_COST = 20;               // places a unit has in front of its blocks, at most: the merge of a piece's warps, the rings' start
// Dynamic shared memory: rings (the merge's rows at the end of a piece), query tile, with a mask its bits per block and token.
constexpr int tree_smem_bytes(int mask_tokens) { return TREE_RING_BYTES + TREE_Q_BYTES + mask_tokens * TREE_CHUNK * 2; }
// A partial result: rows of sums, then (maximum in log2 units, weight) per row. CTA c's result of unit u is number c + u: of
// the pairs that occur each has a number of its own, since both grow along the list.
constexpr int TREE_PARTIAL = TREE_ROWS * (HEAD_DIM + 2);

template <bool ACCUMULATE, bool PACKED>
__global__ void __launch_bounds__(TREE_THREADS, TREE_CTAS_PER_SM) tree_mma_kernel(const __grid_constant__ TreeParams p) {
  constexpr int HALVES = PACKED ? 1 : 2;                           // of the 16 rows, that hold rows of the unit
  extern __shared__ __align__(1024) uint8_t tree_smem[];
  __shared__ float part_m[TREE_WARPS][TREE_ROWS], part_l[TREE_WARPS][TREE_ROWS];
  __shared__ int live_key[TREE_CHUNK];                             // with a mask: first key of the blocks somebody sees ...
  __shared__ uint16_t live_keys[TREE_CHUNK], live_at[TREE_CHUNK];  // ... which keys, and the block's place in the bits
  __shared__ int warp_live[TREE_WARPS];
  __shared__ TreeWalk<TREE_BLOCK> walk;
  __shared__ TreePiece piece_s;
  uint8_t* const q_tile = tree_smem + TREE_RING_BYTES;
  uint16_t* const mask_bits = reinterpret_cast<uint16_t*>(q_tile + TREE_Q_BYTES);       // [block][token]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, j = lane & 3;
  const int rep = p.H / p.Hkv, all_rows = p.n * rep;
  cudaGridDependencySynchronize();                                 // the launch may have been set up beside the kernel before it
  cudaTriggerProgrammaticLaunchCompletion();
  if (warp == 0) {
    TreeWalk<TREE_BLOCK> w;
    w.start(p, p.B, blockIdx.x, gridDim.x);
    if (lane == 0) { walk = w; walk.piece(p, piece_s); }
  }
  __syncthreads();
  while (piece_s.count > 0) {
    const TreePiece pc = piece_s;
    const int b = pc.b, hk = pc.hk, row0 = pc.rg * TREE_ROWS, n_rows = min(all_rows - row0, TREE_ROWS);
    const int unit = (b * p.Hkv + hk) * p.row_groups + pc.rg;
    const int first_key = pc.first * TREE_BLOCK;
    auto block_bits = [&](int key0) { return pc.n_keys - key0 >= TREE_BLOCK ? 0xffffu : (1u << (pc.n_keys - key0)) - 1u; };
    const bool masked = p.mask != nullptr;

    const uint32_t ring = ptx::smem_u32(tree_smem) + warp * (TREE_STAGES * 2 * TREE_TILE);
    const int half = lane >> 4, copy_piece = lane & 15;            // a copy instruction takes two rows
    const __nv_bfloat16* const kb = p.k + b * p.ks.sb + hk * p.ks.sh + copy_piece * 8;
    const __nv_bfloat16* const vb = p.v + b * p.vs.sb + hk * p.vs.sh + copy_piece * 8;
    int n_live, chunk_key;                                         // blocks of this chunk, its first key
    auto block = [&](int e, uint32_t& seen) {                      // first key of the chunk's e-th block
      if (masked) { seen = live_keys[e]; return live_key[e]; }
      const int key0 = chunk_key + e * TREE_BLOCK;
      seen = block_bits(key0);
      return key0;
    };
    auto fetch = [&](int e, int stage) {                           // always one commit group, possibly empty
      if (e < n_live) {
        uint32_t seen;
        const int key0 = block(e, seen);
        const uint32_t dst = ring + stage * (2 * TREE_TILE);
        const __nv_bfloat16* kr = kb + int64_t(key0 + half) * p.ks.ss;
        const __nv_bfloat16* vr = vb + int64_t(key0 + half) * p.vs.ss;
#pragma unroll
        for (int i = 0; i < TREE_BLOCK; i += 2) {                  // keys nobody sees become zeros and are not read
          const uint32_t bytes = (seen >> (i + half)) & 1u ? 16u : 0u;
          const uint32_t off = row_piece(i + half, copy_piece);
          ptx::cp_async_16(dst + off, bytes ? kr + i * p.ks.ss : p.k, bytes);
          ptx::cp_async_16(dst + TREE_TILE + off, bytes ? vr + i * p.vs.ss : p.v, bytes);
        }
      }
      ptx::cp_async_commit();
    };

    int token_of[HALVES];                                          // token of rows g and g + 8
#pragma unroll
    for (int h = 0; h < HALVES; ++h) token_of[h] = min(row0 + 8 * h + g, all_rows - 1) / rep;
    unsigned long long own[HALVES] = {};                           // the tokens' own keys they see
    float m_run[HALVES], l_run[HALVES];                            // l_run: this lane's keys only
    // Dims 8 t + 2 j, + 1 of rows g, g + 8. P's low parts go to o_lo or, PACKED, to rows g + 8.
    float o[16][4], o_lo[PACKED ? 1 : 16][4];
    const int mi = lane >> 3, mr = lane & 7;                       // ldmatrix row addresses, see below
    const int k_row = (mi >> 1) * 8 + mr, v_row = (mi & 1) * 8 + mr;
    const uint32_t qt = ptx::smem_u32(q_tile);
    uint32_t qf[PACKED ? 8 : 1][2];                                // A operand of the eight 16-dim steps, rows 0-7
    // An infinite or NaN value row makes every row's sum NaN, also those of tokens that do not see it (zero times infinity).
    // So a CTA whose sums are not finite takes its keys once more, key by key, each only to the rows that see it.
    for (int attempt = 0; attempt < 2; ++attempt) {
      const bool one_by_one = attempt == 1;
#pragma unroll
      for (int h = 0; h < HALVES; ++h) { m_run[h] = -CUDART_INF_F; l_run[h] = 0.f; }
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = o_lo[PACKED ? 0 : t][i] = 0.f;
      const int step = masked ? TREE_CHUNK : pc.count;
      for (int c0 = 0; c0 < pc.count; c0 += step) {
        chunk_key = first_key + c0 * TREE_BLOCK;
        n_live = min(pc.count - c0, step);
        if (masked) {                                              // the chunk's mask bits; blocks and keys that any token sees
          const int dealt = n_live, m_tokens = p.mask_sn == 0 ? 1 : p.n;
          __syncthreads();                                         // everybody is done with the chunk before
          for (int e = tid; e < dealt * m_tokens; e += TREE_THREADS) {
            const int t = e / m_tokens, i = e - t * m_tokens;
            const int key0 = chunk_key + t * TREE_BLOCK;
            const uint32_t there = block_bits(key0);
            const uint8_t* m = p.mask + b * p.mask_sb + i * p.mask_sn + key0 * p.mask_ss;
            uint32_t seen = 0;
            if (p.mask_vec && there == 0xffffu) {
              const uint4 w = *reinterpret_cast<const uint4*>(m);
              const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int c = 0; c < 4; ++c) seen |= ((__vminu4(ws[c], 0x01010101u) * 0x10204080u) >> 28) << (4 * c);
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
            live_key[at] = chunk_key + tid * TREE_BLOCK;
            live_keys[at] = uint16_t(keys);
            live_at[at] = uint16_t(tid * m_tokens);
          }
          __syncthreads();
          n_live = 0;
#pragma unroll
          for (int w = 0; w < TREE_WARPS; ++w) n_live += warp_live[w];
        }
        // this warp streams blocks warp, warp + TREE_WARPS, ...
#pragma unroll
        for (int s = 0; s < TREE_STAGES - 1; ++s) fetch(warp + s * TREE_WARPS, s);
        if (attempt == 0 && c0 == 0) {                             // meanwhile: query rows (zeros past the last), ancestors
          if constexpr (PACKED) {                                  // each warp its own operand
            const int row = row0 + min(g, n_rows - 1), token = token_of[0], head = hk * rep + row - token * rep;
            const uint32_t* const qp = reinterpret_cast<const uint32_t*>(p.q + b * p.q_sb + head * p.q_sh + token * p.q_sn) + j;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              qf[t][0] = g < n_rows ? qp[8 * t] : 0u;
              qf[t][1] = g < n_rows ? qp[8 * t + 4] : 0u;
            }
          }
          for (int e = tid; !PACKED && e < TREE_ROWS * 16; e += TREE_THREADS) {
            const int r = e >> 4, c = e & 15;
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (r < n_rows) {
              const int token = (row0 + r) / rep, head = hk * rep + (row0 + r) - token * rep;
              w = *reinterpret_cast<const uint4*>(p.q + b * p.q_sb + head * p.q_sh + token * p.q_sn + c * 8);
            }
            *reinterpret_cast<uint4*>(q_tile + row_piece(r, c)) = w;
          }
          if ((pc.first + pc.count) * TREE_BLOCK > pc.ctx) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h) own[h] = tree_own_keys(p, b, token_of[h]);
          }
          if (!PACKED) __syncthreads();
        }

        // ldmatrix: K matrices are (keys 0-7 | 8-15) x (dims 0-7 | 8-15) of a step, V the same transposed, Q
        // (rows 0-7 | 8-15) x (dims 0-7 | 8-15)
        int stage = 0;
        for (int e = warp; e < n_live; e += TREE_WARPS) {
          ptx::cp_async_wait<TREE_STAGES - 2>();
          __syncwarp();                                            // every lane's copies of this block have landed, and
          fetch(e + (TREE_STAGES - 1) * TREE_WARPS, (stage + TREE_STAGES - 1) % TREE_STAGES);   // all are done with the last one
          const uint32_t kt = ring + stage * (2 * TREE_TILE), vt = kt + TREE_TILE;
          float s[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) s[0][i] = s[1][i] = 0.f;
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            uint32_t r[4], a[4];
            ldmatrix_x4(kt + row_piece(k_row, 2 * t + (mi & 1)), r);
            if constexpr (PACKED) {
              mma_m16n8k16(s[0], qf[t][0], 0u, qf[t][1], 0u, r[0], r[1]);
              mma_m16n8k16(s[1], qf[t][0], 0u, qf[t][1], 0u, r[2], r[3]);
            } else {
              ldmatrix_x4(qt + row_piece(v_row, 2 * t + (mi >> 1)), a);
              mma_m16n8k16(s[0], a[0], a[1], a[2], a[3], r[0], r[1]);
              mma_m16n8k16(s[1], a[0], a[1], a[2], a[3], r[2], r[3]);
            }
          }
          uint32_t seen;
          const int key0 = block(e, seen);
          const bool plain = !masked && key0 + TREE_BLOCK <= pc.ctx;       // every token sees the whole block
          bool grow_any = false;
          float alpha[HALVES], x[HALVES][4];
          uint32_t row_bits[HALVES];                                  // keys each row sees
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            uint32_t bits = seen;
            if (!plain) {
              if (masked) bits = mask_bits[live_at[e] + (p.mask_sn == 0 ? 0 : token_of[h])];
              if (key0 + TREE_BLOCK > pc.ctx) {                    // bits of the tokens' own keys, from key0 on
                const int at = key0 - pc.ctx;
                bits &= at >= 0 ? (at < 64 ? uint32_t(own[h] >> at) : 0u) : uint32_t(own[h] << -at) | ((1u << -at) - 1u);
              }
            }
            row_bits[h] = bits;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = 2 * j + (i & 1) + 8 * (i >> 1);
              x[h][i] = (bits >> key) & 1u ? s[i >> 1][2 * h + (i & 1)] * p.scale_log2 : -CUDART_INF_F;
            }
            if (ACCUMULATE && 8 * h + g < n_rows) {                // 32 bytes of a row per four lanes
              float* const dst = p.scores + (int64_t(unit) * p.score_rows + 8 * h + g) * p.score_keys + key0 + 2 * j;
              *reinterpret_cast<float2*>(dst) = make_float2(x[h][0], x[h][1]);
              *reinterpret_cast<float2*>(dst + 8) = make_float2(x[h][2], x[h][3]);
            }
            float m_blk = fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3]));
            m_blk = fmaxf(m_blk, __shfl_xor_sync(0xffffffffu, m_blk, 1));
            m_blk = fmaxf(m_blk, __shfl_xor_sync(0xffffffffu, m_blk, 2));
            // the maximum moves only when the scores outgrow it by 2^8; until then probabilities are merely scaled
            const bool grow = m_blk > m_run[h] + RESCALE_THRESHOLD;
            alpha[h] = grow ? merge_weight(m_run[h], m_blk) : 1.f;
            if (grow) m_run[h] = m_blk;
            grow_any |= grow;
          }
          if (__any_sync(0xffffffffu, grow_any)) {
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
              l_run[h] *= alpha[h];
#pragma unroll
              for (int t = 0; t < 16; ++t) {
                o[t][2 * h] *= alpha[h];
                o[t][2 * h + 1] *= alpha[h];
                float* const low = PACKED ? &o[t][2] : &o_lo[PACKED ? 0 : t][2 * h];
                low[0] *= alpha[h];
                low[1] *= alpha[h];
              }
            }
          }
          uint32_t hi[4], lo[4];                                   // A operand: (row half, key half) = (0,0) (1,0) (0,1) (1,1)
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            const float base = m_run[h] == -CUDART_INF_F ? 0.f : m_run[h];
            float pr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[i] = ptx::ex2(x[h][i] - base);
            l_run[h] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
            split_bf16(pr[0], pr[1], hi[h], lo[h]);
            split_bf16(pr[2], pr[3], hi[2 + h], lo[2 + h]);
          }
          if (one_by_one) {
            for (int c = 0; c < TREE_BLOCK; ++c) {
              const int from = (lane & ~3) | ((c & 7) >> 1);       // the lane that has this key's probabilities
#pragma unroll
              for (int h = 0; h < HALVES; ++h) {
                const uint32_t ph = __shfl_sync(0xffffffffu, c < 8 ? hi[h] : hi[2 + h], from);
                const uint32_t pl = __shfl_sync(0xffffffffu, c < 8 ? lo[h] : lo[2 + h], from);
                const float prob = __uint_as_float(c & 1 ? ph & 0xffff0000u : ph << 16) + __uint_as_float(c & 1 ? pl & 0xffff0000u : pl << 16);
                if ((row_bits[h] >> c) & 1u) {
#pragma unroll
                  for (int t = 0; t < 16; ++t) {
                    uint32_t w;
                    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vt + row_piece(c, t) + 4 * j) : "memory");
                    o[t][2 * h] += prob * __uint_as_float(w << 16);
                    o[t][2 * h + 1] += prob * __uint_as_float(w & 0xffff0000u);
                  }
                }
              }
            }
          } else {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
              uint32_t r[4];
              ldmatrix_x4_trans(vt + row_piece(v_row, 2 * t + (mi >> 1)), r);
              if constexpr (PACKED) {
                mma_m16n8k16(o[2 * t], hi[0], lo[0], hi[2], lo[2], r[0], r[1]);
                mma_m16n8k16(o[2 * t + 1], hi[0], lo[0], hi[2], lo[2], r[2], r[3]);
              } else {
                mma_m16n8k16(o[2 * t], hi[0], hi[1], hi[2], hi[3], r[0], r[1]);
                mma_m16n8k16(o[2 * t + 1], hi[0], hi[1], hi[2], hi[3], r[2], r[3]);
                mma_m16n8k16(o_lo[2 * t], lo[0], lo[1], lo[2], lo[3], r[0], r[1]);
                mma_m16n8k16(o_lo[2 * t + 1], lo[0], lo[1], lo[2], lo[3], r[2], r[3]);
              }
            }
          }
          stage = stage + 1 == TREE_STAGES ? 0 : stage + 1;
        }
        ptx::cp_async_wait<0>();
        __syncwarp();
      }
      bool finite = true;
#pragma unroll
      for (int t = 0; t < 16; ++t)
#pragma unroll
        for (int i = 0; i < 2 * HALVES; ++i) {
          o[t][i] += PACKED ? o[t][2 + (i & 1)] : o_lo[PACKED ? 0 : t][i];
          finite = finite && fabsf(o[t][i]) < CUDART_INF_F;
        }
      if (!__syncthreads_or(!finite)) break;
    }

    // ---- the piece's result: lanes of a row, warps; rows of a whole unit to the output, else a partial result ----------
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      float l = l_run[h];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (j == 0) { part_m[warp][8 * h + g] = m_run[h]; part_l[warp][8 * h + g] = l; }
    }
    constexpr int ROW = HEAD_DIM + 8;                              // rows start 8 banks apart
    float* const part_o = reinterpret_cast<float*>(tree_smem);     // [warp][row][ROW]: the rings are free
    static_assert(TREE_WARPS * TREE_ROWS * ROW * 4 <= TREE_RING_BYTES, "the merge's rows fit the rings");
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
#pragma unroll
      for (int t = 0; t < 16; ++t)
        *reinterpret_cast<float2*>(part_o + (warp * TREE_ROWS + 8 * h + g) * ROW + 8 * t + 2 * j) = make_float2(o[t][2 * h], o[t][2 * h + 1]);
    if (tid == 0) walk.piece(p, piece_s);                          // all have taken their copy of this one
    __syncthreads();
    float* const slot = p.scratch + (int64_t(blockIdx.x) + unit) * TREE_PARTIAL;
    const bool whole = pc.count == pc.of;
    for (int r = warp; r < n_rows; r += TREE_WARPS) {              // a warp per row, a lane for four dims
      float m_all = part_m[0][r];
#pragma unroll
      for (int w = 1; w < TREE_WARPS; ++w) m_all = fmaxf(m_all, part_m[w][r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float l_all = 0.f;
#pragma unroll
      for (int w = 0; w < TREE_WARPS; ++w) {
        const float f = merge_weight(part_m[w][r], m_all);
        const float4 y = *reinterpret_cast<const float4*>(part_o + (w * TREE_ROWS + r) * ROW + 4 * lane);
        acc.x += f * y.x; acc.y += f * y.y; acc.z += f * y.z; acc.w += f * y.w;
        l_all += f * part_l[w][r];
      }
      if (!whole || ACCUMULATE) {
        if (lane == 0) reinterpret_cast<float2*>(slot + TREE_ROWS * HEAD_DIM)[r] = make_float2(m_all, l_all);
      }
      if (!whole) {
        reinterpret_cast<float4*>(slot + r * HEAD_DIM)[lane] = acc;
      } else {
        const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
        const int token = (row0 + r) / rep, head = hk * rep + (row0 + r) - token * rep;
        reinterpret_cast<uint2*>(p.o + ((int64_t(b) * p.n + token) * p.H + head) * HEAD_DIM)[lane] =
            make_uint2(ptx::pack_bf16(acc.x * inv, acc.y * inv), ptx::pack_bf16(acc.z * inv, acc.w * inv));
      }
    }
    __syncthreads();                                               // the next piece's copies go where the merge has read
  }
}

// Parts of a unit: the CTAs that had one, and where they left it.
struct TreeParts {
  int first, count;            // first CTA, CTAs
  __device__ __forceinline__ TreeParts(const TreeParams& p, int b, int in_b, uint32_t grid) {
    uint32_t start;
    const TreeList<TREE_BLOCK> list(p, p.B, grid, b, &start);
    const int tiles = tree_tiles<TREE_BLOCK>(p, b);
    start += uint32_t(in_b + 1) * list.places(tiles) - tiles;      // place of the unit's first tile
    first = int(start / list.per);
    count = int((start + tiles - 1) / list.per) - first + 1;
  }
};

// Joins the parts of units that several CTAs had a part of. A warp per row, a lane for four dims.
constexpr int TREE_MERGE_WARPS = 4;
template <int AT_ONCE>                                             // parts whose loads are under way together
__device__ __forceinline__ void tree_merge_row(const TreeParams& p, const TreeParts& parts, int unit, int b, int hk, int row, int at) {
  const int lane = threadIdx.x & 31, rep = p.H / p.Hkv;
  const float* const first = p.scratch + (int64_t(parts.first) + unit) * TREE_PARTIAL;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m_all = -CUDART_INF_F, l_all = 0.f;
  for (int i0 = 0; i0 < parts.count; i0 += AT_ONCE) {
    float2 x[AT_ONCE];
    float4 o[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float* const slot = first + int64_t(min(i0 + i, parts.count - 1)) * TREE_PARTIAL;
      x[i] = reinterpret_cast<const float2*>(slot + TREE_ROWS * HEAD_DIM)[at];
      o[i] = reinterpret_cast<const float4*>(slot + at * HEAD_DIM)[lane];
    }
    float m_new = m_all;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) m_new = fmaxf(m_new, x[i].x);
    const float alpha = merge_weight(m_all, m_new);
    l_all *= alpha;
    acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      if (i0 + i >= parts.count) break;
      const float f = merge_weight(x[i].x, m_new);
      l_all += f * x[i].y;
      acc.x += f * o[i].x; acc.y += f * o[i].y; acc.z += f * o[i].z; acc.w += f * o[i].w;
    }
    m_all = m_new;
  }
  const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
  const int token = row / rep, head = hk * rep + row - token * rep;
  reinterpret_cast<uint2*>(p.o + ((int64_t(b) * p.n + token) * p.H + head) * HEAD_DIM)[lane] =
      make_uint2(ptx::pack_bf16(acc.x * inv, acc.y * inv), ptx::pack_bf16(acc.z * inv, acc.w * inv));
}
__global__ void __launch_bounds__(32 * TREE_MERGE_WARPS) tree_merge_kernel(const __grid_constant__ TreeParams p, uint32_t grid) {
  const int rows = p.n * (p.H / p.Hkv);
  const int64_t r = int64_t(blockIdx.x) * TREE_MERGE_WARPS + (threadIdx.x >> 5);           // (b, hk, row of the KV head)
  const int kv = int(r / rows), row = int(r - int64_t(kv) * rows);
  const int b = kv / p.Hkv, hk = kv - b * p.Hkv, rg = row / TREE_ROWS;
  if (b >= p.B) return;
  const TreeParts parts(p, b, hk * p.row_groups + rg, grid);
  cudaGridDependencySynchronize();
  if (parts.count == 1) return;                                    // one CTA held the unit and wrote its rows
  tree_merge_row<8>(p, parts, kv * p.row_groups + rg, b, hk, row, row - rg * TREE_ROWS);
}

// weights += each visible key's probabilities summed over its KV head's query heads, from the scores and every row's
// maximum and weight; a thread per four keys, so the order of the sum is fixed. The last CTA of a KV head joins its output rows
// instead. What takes time is the chain of loads - the list, the scores, the rows' statistics - so there are as many CTAs as run
// together, each with several blocks of keys. The whole call, 288 heads of 4,000 keys 111.0 us, 128 heads of 2,048 to 8,192 75.7; with
// a CTA per 1,024 keys and 20 scalar loads a thread 114.7 and 79.2. 92 without the weights.
constexpr int TREE_WEIGHT_THREADS = 256, TREE_WEIGHT_KEYS = 4 * TREE_WEIGHT_THREADS, TREE_WEIGHT_CTAS_PER_SM = 4;
__global__ void __launch_bounds__(TREE_WEIGHT_THREADS, TREE_WEIGHT_CTAS_PER_SM) tree_weights_kernel(const __grid_constant__ TreeParams p, uint32_t grid) {
  __shared__ float2 stats[TREE_ROWS];                              // maximum, inverse sum
  const int hk = blockIdx.y % p.Hkv, b = blockIdx.y / p.Hkv, rows = p.H / p.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool joins = blockIdx.x == gridDim.x - 1;
  const int keys = tree_context(p, b) + 1;
  if (!joins && int(blockIdx.x) * TREE_WEIGHT_KEYS >= keys) return;
  float* const weights = p.weights + b * p.weights_sb + hk * p.weights_sh;
  const uint8_t* const mask = p.mask + b * p.mask_sb;
  for (int rg = 0; rg < p.row_groups; ++rg) {
    const int unit = (b * p.Hkv + hk) * p.row_groups + rg, n_rows = min(rows - rg * TREE_ROWS, TREE_ROWS);
    const TreeParts parts(p, b, hk * p.row_groups + rg, grid);
    if (rg == 0) cudaGridDependencySynchronize();
    if (joins) {
      if (parts.count > 1)
        for (int r = warp; r < n_rows; r += TREE_WEIGHT_THREADS / 32) tree_merge_row<4>(p, parts, unit, b, hk, rg * TREE_ROWS + r, r);
      continue;
    }
    const float* const x = p.scores + int64_t(unit) * p.score_rows * p.score_keys;
    constexpr int AT_ONCE = 4;                                     // rows whose scores are under way together
    bool first_block = true;
    for (int key0 = blockIdx.x * TREE_WEIGHT_KEYS + 4 * threadIdx.x; key0 - 4 * int(threadIdx.x) < keys; key0 += (gridDim.x - 1) * TREE_WEIGHT_KEYS) {
      const bool whole = key0 + 4 <= keys;                         // four keys of the sequence
      float4 y[AT_ONCE];
#pragma unroll
      for (int r = 0; r < AT_ONCE; ++r)
        y[r] = key0 < keys ? *reinterpret_cast<const float4*>(x + int64_t(min(r, n_rows - 1)) * p.score_keys + key0) : make_float4(0.f, 0.f, 0.f, 0.f);
      uint32_t seen = 0;                                           // a bit for each key
      if (whole && (p.mask == nullptr || p.mask_vec)) {
        const uint32_t m = p.mask ? *reinterpret_cast<const uint32_t*>(mask + key0) : 0x01010101u;
        seen = (__vminu4(m, 0x01010101u) * 0x10204080u) >> 28;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) seen |= key0 + c < keys && (p.mask == nullptr || mask[(key0 + c) * p.mask_ss] != 0) ? 1u << c : 0u;
      }
      float before[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
      if (whole && p.weights_vec) {
        const float4 w = *reinterpret_cast<const float4*>(weights + key0);
        before[0] = w.x; before[1] = w.y; before[2] = w.z; before[3] = w.w;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) before[c] = (seen >> c) & 1u ? weights[key0 + c] : 0.f;
      }
      if (first_block) {                                           // the rows' statistics, while the first loads are under way
        first_block = false;
        const float2* const first = reinterpret_cast<const float2*>(p.scratch + (int64_t(parts.first) + unit) * TREE_PARTIAL + TREE_ROWS * HEAD_DIM);
        __syncthreads();                                           // those of the rows before have been read
        for (int r = warp; r < n_rows; r += TREE_WEIGHT_THREADS / 32) {
          float m = -CUDART_INF_F, l = 0.f;
          for (int i = lane; i < parts.count; i += 32) {
            const float2 z = first[int64_t(i) * (TREE_PARTIAL / 2) + r];
            const float m_new = fmaxf(m, z.x);
            l = l * merge_weight(m, m_new) + z.y * merge_weight(z.x, m_new);
            m = m_new;
          }
          for (int d = 1; d < 32 && d < parts.count; d *= 2) {     // lanes from parts.count on have none
            const float m2 = __shfl_xor_sync(0xffffffffu, m, d), l2 = __shfl_xor_sync(0xffffffffu, l, d), m_new = fmaxf(m, m2);
            l = l * merge_weight(m, m_new) + l2 * merge_weight(m2, m_new);
            m = m_new;
          }
          if (lane == 0) stats[r] = make_float2(m, 1.f / l);
        }
        __syncthreads();
      }
      for (int r0 = 0; r0 < n_rows; r0 += AT_ONCE) {
        if (r0 > 0) {
#pragma unroll
          for (int r = 0; r < AT_ONCE; ++r)
            y[r] = key0 < keys ? *reinterpret_cast<const float4*>(x + int64_t(min(r0 + r, n_rows - 1)) * p.score_keys + key0) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int r = 0; r < AT_ONCE; ++r) {
          if (r0 + r >= n_rows) break;
          const float2 st = stats[r0 + r];
          sum[0] += ptx::ex2(y[r].x - st.x) * st.y;                // of keys that are not seen anything, and not used
          sum[1] += ptx::ex2(y[r].y - st.x) * st.y;
          sum[2] += ptx::ex2(y[r].z - st.x) * st.y;
          sum[3] += ptx::ex2(y[r].w - st.x) * st.y;
        }
      }
      if (seen == 0u) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) before[c] = (seen >> c) & 1u ? before[c] + sum[c] : before[c];
      if (whole && p.weights_vec) {
        *reinterpret_cast<float4*>(weights + key0) = make_float4(before[0], before[1], before[2], before[3]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if ((seen >> c) & 1u) weights[key0 + c] = before[c];
      }
    }
  }
}

}  // namespace intra
