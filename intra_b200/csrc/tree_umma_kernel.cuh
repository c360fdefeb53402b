// Attention of drafted tokens over a cache for more rows than a warp's registers hold (tree_mma_kernel.cuh has the definition):
// the products on tcgen05 with 128 rows a tile, K and V tiles of 128 keys.
//
// Up to 256 rows the bound is still reading K and V (64 KB a key tile, 2,800 cycles at an SM's share of the HBM
// bandwidth; the products of 256 rows take 2,048). The work is dealt by key tiles (tree_list.cuh).
//
// Two streams of softmax work run side by side, so that the tensor cores have one's products while the other is at its
// exponentials:
//   PAIR (more than 128 rows): the streams are two tiles of 128 rows that read the same K and V tiles. Tensor memory:
//     one score buffer that a stream hands back as soon as it has copied its scores out, P0 and P1 in bf16, O0, O1.
//   otherwise: the streams are the even and the odd key tiles of the same rows. There is room for P as two bf16 numbers
//     (16 significant bits) over each stream's own scores; O0 and O1 are joined at the end of a unit.
//
// Warp roles (512 threads): warps 0-3 and 4-7 softmax sets of the streams, a thread owning a row, which also write
// the results; 8-11 request the tiles: TMA where a tile's rows are all keys of the sequence and the cache's strides
// allow, else 16-byte copies in which rows past its last key, and rows no token sees, become zeros; 12 issues QK^T (and, but
// for PAIR, PV), 13 PV; 14 and 15 bring the query rows of the units after the first, whose rows the softmax sets fetch.
// Whoever writes operands by plain copies fences them for the tensor cores' proxy before it reports them.
//
// Barriers, all waits bounded (2 s; see attn_kernel.cuh for what a CTA does that gives up):
//   full[r], free[r]   ring of tile buffers, in the order K0 K1 V0 K2 V1 .. over the CTA's tiles
//   q_full, q_free     per unit: the query rows are there / their last QK^T has completed
//   s_full[s]          scores of stream s are there (and all products before them are complete)
//   s_taken[s]         PAIR: set s has copied its scores of a tile
//   p_full[s], pv_done[s]   set s has stored its probabilities / PV_s has completed
//   o_done[s]          the last PV_s of a unit has completed
//   o_free[s]          set s has read O (of both streams, but for PAIR) of a unit
//   ml_ready[s][u & 1] not PAIR: set s has published its rows' maxima and sums of unit u
//   drain[w]           a CTA that gives up: the products that issuing warp w had under way have completed
// Each completes again only after its waiters have seen the completion before. A wait for "the phase before the first"
// (parity 1 of a fresh barrier) returns at once.
#pragma once
#include <cuda.h>

#include "softmax.cuh"
#include "tree_list.cuh"
#include "warp_mma.cuh"

namespace intra {

constexpr int UMMA_THREADS = 512;
constexpr int UMMA_SM_REGS = 184, UMMA_LOAD_REGS = 64, UMMA_ISSUE_REGS = 80;
static_assert(256 * UMMA_SM_REGS + 128 * (UMMA_LOAD_REGS + UMMA_ISSUE_REGS) <= 65536,
              "register budgets exceed what the CTA was launched with: setmaxnreg.inc would never return");
template <bool PAIR> constexpr int UMMA_ROWS = PAIR ? 2 * TILE_M : TILE_M;       // rows of a unit
constexpr int UMMA_RING = 5;                     // tile buffers
template <bool PAIR> constexpr int UMMA_SMEM_BYTES = (UMMA_RING + (PAIR ? 2 : 1)) * TILE_BYTES + 1024;
// Partial results: a CTA leaves at most two, of the unit its part begins in and of the one it ends in. Each is the rows'
// sums, [column][row] so that 32 rows' stores of a column lie together, then their maxima (log2 units) and weights.
template <bool PAIR> constexpr int64_t UMMA_PARTIAL = int64_t(UMMA_ROWS<PAIR>) * (HEAD_DIM + 2);
// A CTA's part is at least this many key tiles: a shorter one costs more in its ends and its merge than it spreads.
constexpr int UMMA_MIN_TILES = 2;
constexpr int UMMA_UNIT_COST = 5;                // places a unit has in front of its tiles, at most (TreeList)
// Tiles that partial results and their merge are worth; more where the host can tell that the merge need not be launched
// (`no_merge`). Measured, us, divided / whole:
//   rows of a unit                               32          96         256
//   128 units of 32 tiles (27.7 a CTA)    63.3 / 53.8 72.4 / 57.3 96.7 / 70.2    no lengths; with lengths 49.2 / 46.6 (20 a CTA)
//   128 units of 8 tiles (6.9)            33.3 / 20.2 40.4 / 21.6 59.7 / 26.4
//   96 units of 32 tiles (20.8)           50.8 / 58.9 55.3 / 62.1 75.8 / 62.7    the merge launched in all but the last
//   72 units of 64 tiles (31.1)          66.2 / 100.5 73.6 / 103.2 91.6 / 116.2
__host__ __device__ constexpr int umma_split_cost(int rows, bool no_merge) { return 5 + rows / 40 + (no_merge ? 3 : 0); }

struct TreeUmmaParams {
  TreeParams t;                // row_groups: units per KV head
  FastDiv by_rep;              // query heads per KV head
  CUtensorMap maps[2];         // K, V: (128, S, 1, Hkv, B)
  int use_tma;
  // The merge may be set up beside this kernel: there are SMs without a CTA of it. 5 tokens over 3,001 keys 15.9 -> 15.1 us; with
  // a CTA on every SM, 32 rows over 65,536 keys, 65 us for 61.
  int early;
  int* status;
};

// The mask of a token as bits, a word for 32 keys.
__device__ __forceinline__ const uint32_t* tree_bits(const TreeParams& p, int b, int token) {
  return p.bits + (int64_t(b) * p.bits_tokens + (p.bits_tokens == 1 ? 0 : token)) * p.bits_words;
}

// Rows whose sums are not finite, once more: an infinite or NaN value row makes every row's sum NaN, also those of tokens that do
// not see it (zero times infinity). Called by whole softmax warps, whose lanes hold the maximum and sum of their rows and
// whether they need it; 16 rows at a time, by warp-level MMAs with operands straight from global memory: finite values as such,
// others added key by key, each only to the rows that see it. Results go over what was written. 8 sequences of 2 x 4,096 keys
// of which one holds a NaN: 0.18 ms for 0.063 (one row at a time in 32 bits: 32 ms). Having the call costs the other inputs
// 1 to 3 %, in registers; hence its few arguments. Spilled bytes, stored / loaded: the kernel
// with the call 40 / 52 (PAIR), 12 / 20, with a mask 64 / 92, without it 8 / 16 in the second form alone; the redo itself 100 / 164 and 8 / 4.
template <bool PAIR>
__device__ __noinline__ void tree_exact_rows(const TreeUmmaParams& params, const TreePiece& pc, float m, float l, bool redo) {
  constexpr int COLS = PAIR ? 128 : 64, ROWS = UMMA_ROWS<PAIR>, NT = COLS / 8;
  const TreeParams& p = params.t;
  const int lane = threadIdx.x & 31, g = lane >> 2, j = lane & 3, warp = threadIdx.x >> 5;
  const int rep = p.H / p.Hkv, all_rows = p.n * rep;
  const int col = PAIR ? 0 : (warp >> 2) * COLS, at0 = 32 * (PAIR ? warp : warp & 3), r0 = pc.rg * ROWS + at0;
  float* const part = pc.count != pc.of ? p.scratch + (int64_t(blockIdx.x) * 2 + pc.starts) * UMMA_PARTIAL<PAIR> + at0 : nullptr;
  const __nv_bfloat16* const kb = p.k + pc.b * p.ks.sb + pc.hk * p.ks.sh;
  const __nv_bfloat16* const vb = p.v + pc.b * p.vs.sb + pc.hk * p.vs.sh + col;
  const uint32_t wanted = __ballot_sync(0xffffffffu, redo);
#pragma unroll 1
  for (int group = 0; group < 2; ++group) {
    if (((wanted >> (16 * group)) & 0xffffu) == 0u) continue;
    int token[2], head[2];
    float m_row[2], l_row[2];
    unsigned long long own[2];
    const uint32_t* mask_row[2] = {nullptr, nullptr};
    uint32_t qf[8][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = min(r0 + 16 * group + 8 * h + g, all_rows - 1);
      token[h] = fdiv(r, params.by_rep);
      head[h] = pc.hk * rep + r - token[h] * rep;
      m_row[h] = __shfl_sync(0xffffffffu, m, 16 * group + 8 * h + g);
      l_row[h] = __shfl_sync(0xffffffffu, l, 16 * group + 8 * h + g);
      own[h] = tree_own_keys(p, pc.b, token[h]);
      if (p.bits != nullptr) mask_row[h] = tree_bits(p, pc.b, token[h]);
      const uint32_t* const q = reinterpret_cast<const uint32_t*>(p.q + pc.b * p.q_sb + head[h] * p.q_sh + token[h] * p.q_sn) + j;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        qf[t][h] = q[8 * t];
        qf[t][2 + h] = q[8 * t + 4];
      }
    }
    float o[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
    const int last = min((pc.first + pc.count) * TILE_N, pc.n_keys);
#pragma unroll 1
    for (int key0 = pc.first * TILE_N; key0 < last; key0 += 16) {
      float s[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        const uint32_t* const k = reinterpret_cast<const uint32_t*>(kb + int64_t(min(key0 + 8 * n + g, last - 1)) * p.ks.ss) + j;
#pragma unroll
        for (int t = 0; t < 8; ++t) mma_m16n8k16(s[n], qf[t][0], qf[t][1], qf[t][2], qf[t][3], k[8 * t], k[8 * t + 4]);
      }
      uint32_t seen[2], hi[4], lo[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = key0 - pc.ctx;
        seen[h] = (last - key0 >= 16 ? 0xffffu : (1u << (last - key0)) - 1u) &
                  (at >= 0 ? (at < 64 ? uint32_t(own[h] >> at) : 0u) : at <= -16 ? 0xffffu : uint32_t(own[h] << -at) | ((1u << -at) - 1u));
        if (p.bits != nullptr) seen[h] &= mask_row[h][key0 >> 5] >> (key0 & 31);
        float pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = 2 * j + (i & 1) + 8 * (i >> 1);
          pr[i] = (seen[h] >> key) & 1u ? ptx::ex2(s[i >> 1][2 * h + (i & 1)] * p.scale_log2 - m_row[h]) : 0.f;
        }
        split_bf16(pr[0], pr[1], hi[h], lo[h]);
        split_bf16(pr[2], pr[3], hi[2 + h], lo[2 + h]);
      }
      bool odd = false;                                   // some value is not finite
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t b[2];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t w = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = key0 + 8 * n + 2 * j + e;
            const uint32_t x = key < last ? reinterpret_cast<const uint16_t*>(vb + int64_t(key) * p.vs.ss)[8 * t + g] : 0u;
            const bool fine = (x & 0x7f80u) != 0x7f80u;
            odd = odd || !fine;
            w |= fine ? x << (16 * e) : 0u;
          }
          b[n] = w;
        }
        mma_m16n8k16(o[t], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
        mma_m16n8k16(o[t], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
      }
      if (!__any_sync(0xffffffffu, odd)) continue;
      bool all_nan = true;
#pragma unroll 1
      for (int c = 0; c < 16 && key0 + c < last; ++c) {
        const int from = (lane & ~3) | ((c & 7) >> 1);    // the lane that has this key's probabilities
        const uint32_t* const v = reinterpret_cast<const uint32_t*>(vb + int64_t(key0 + c) * p.vs.ss) + j;
        all_nan = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t ph = __shfl_sync(0xffffffffu, c < 8 ? hi[h] : hi[2 + h], from);
          const float prob = __uint_as_float(c & 1 ? ph & 0xffff0000u : ph << 16);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint32_t w = v[4 * t];
            if (((seen[h] >> c) & 1u) && (w & 0x7f80u) == 0x7f80u) o[t][2 * h] += prob * __uint_as_float(w << 16);
            if (((seen[h] >> c) & 1u) && (w & 0x7f800000u) == 0x7f800000u) o[t][2 * h + 1] += prob * __uint_as_float(w & 0xffff0000u);
            all_nan = all_nan && isnan(o[t][2 * h]) && isnan(o[t][2 * h + 1]);
          }
        }
      }
      if (__all_sync(0xffffffffu, all_nan)) break;        // nothing changes any more
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 16 * group + 8 * h + g;
      if (r0 + i >= all_rows) continue;
      const float inv = l_row[h] == 0.f ? 0.f : 1.f / l_row[h];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int c = col + 8 * t + 2 * j;
        if (part != nullptr) {
          part[c * ROWS + i] = o[t][2 * h];
          part[(c + 1) * ROWS + i] = o[t][2 * h + 1];
        } else {
          *reinterpret_cast<uint32_t*>(p.o + ((int64_t(pc.b) * p.n + token[h]) * p.H + head[h]) * HEAD_DIM + c) =
              ptx::pack_bf16(o[t][2 * h] * inv, o[t][2 * h + 1] * inv);
        }
      }
    }
  }
}

template <bool PAIR, bool MASK>
__global__ void __launch_bounds__(UMMA_THREADS, 1) tree_umma_kernel(const __grid_constant__ TreeUmmaParams p) {
  constexpr int RING = UMMA_RING, ROWS = UMMA_ROWS<PAIR>, COLS = PAIR ? HEAD_DIM : HEAD_DIM / 2;
  enum : int {
    FULL = 0, FREE = FULL + RING, Q_FULL = FREE + RING, Q_FREE, S_FULL, S_TAKEN = S_FULL + 2, P_FULL = S_TAKEN + 2,
    PV_DONE = P_FULL + 2, O_DONE = PV_DONE + 2, O_FREE = O_DONE + 2, ML_READY = O_FREE + 2, DRAIN = ML_READY + 4, N_BARS = DRAIN + 2
  };
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bars[N_BARS];
  __shared__ uint32_t tmem_base_smem;
  __shared__ int abort_flag;
  __shared__ TreeWalk<TILE_N> walks[UMMA_THREADS / 32];
  __shared__ TreePiece pieces[UMMA_THREADS / 32];
  __shared__ float2 row_ml[2][PAIR ? 1 : 2][PAIR ? 1 : TILE_M];     // [unit parity][stream][row]
  const TreeParams& t = p.t;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t smem_base = (ptx::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = smem_base, ring_smem = smem_base + (PAIR ? 2 : 1) * TILE_BYTES;
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * uint32_t(i); };
  const int rep = t.H / t.Hkv, all_rows = t.n * rep;

  if (tid == 0) {
    abort_flag = 0;
    for (int i = 0; i < N_BARS; ++i) {
      int n = 1;
      if (i < FREE) n = 128;
      if (i == Q_FULL) n = 8;
      if ((i >= S_TAKEN && i < PV_DONE) || (i >= O_FREE && i < DRAIN)) n = 4;
      ptx::mbar_init(&bars[i], n);
    }
    ptx::fence_mbar_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(&tmem_base_smem, 512);
    ptx::tmem_relinquish();
  }
  if (warp == 8 && lane < 2 && p.use_tma) ptx::prefetch_tensormap(&p.maps[lane]);      // else they describe nothing
  cudaGridDependencySynchronize();                       // what is above ran beside the end of the kernel before this one
  if (p.early) cudaTriggerProgrammaticLaunchCompletion();
  TreeWalk<TILE_N>& walk = walks[warp];
  const TreePiece& pc = pieces[warp];
  {
    TreeWalk<TILE_N> w;
    w.start(t, t.B, blockIdx.x, gridDim.x);
    if (lane == 0) walk = w;
  }
  // Copies rows `first`, first + step, .. of a unit's queries, 16 threads a row; rows past the last become zeros.
  auto copy_queries = [&](const TreePiece& x, int first, int step) {
#pragma unroll 4
    for (int at = first; at < ROWS; at += step) {
      const int r = x.rg * ROWS + at, token = fdiv(r, p.by_rep);
      const __nv_bfloat16* const src = t.q + x.b * t.q_sb + (x.hk * rep + r - token * rep) * t.q_sh + token * t.q_sn + (lane & 15) * 8;
      ptx::cp_async_16(q_smem + (at >> 7) * TILE_BYTES + tile_offset(at & 127, lane & 15), r < all_rows ? src : t.q, r < all_rows ? 16u : 0u);
    }
    ptx::cp_async_commit();
    ptx::cp_async_wait<0>();
    ptx::fence_proxy_async_smem();
    __syncwarp();
  };
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_base_smem;
  volatile int* abort_p = &abort_flag;
  bool ok = true;
#define TREE_WAIT(index, parity, code) ptx::mbar_wait_at(bar(index), (parity) & 1, abort_p, code)
  // Ring requests of tile j, counted over the CTA: its K, and its V behind the next tile's K.
  auto k_request = [](uint32_t j) { return j == 0 ? 0u : 2 * j - 1; };
  auto v_request = [](uint32_t j) { return 2 * j + 2; };

  if (warp < 8) {
    // ================================ softmax sets, results =======================================
    ptx::setmaxnreg_inc<UMMA_SM_REGS>();
    const int sx = warp >> 2, row = tid & 127;
    const uint32_t lane_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + (PAIR ? 0 : sx * 128);
    const uint32_t p_addr = PAIR ? lane_addr + 128 + sx * 64 : s_addr;
    const uint32_t o_addr = lane_addr + 256 + sx * 128;
    uint32_t kt = 0, unit = 0, done[2] = {0, 0};          // tiles of this stream, units, units in which a stream had tiles
    while (tree_next(t, walk, pieces[warp])) {
      if (unit == 0) {                                    // the first unit's queries: nobody else has as many hands free
        copy_queries(pc, 2 * warp + (lane >> 4), 16);
        if (lane == 0) ptx::mbar_arrive_at(bar(Q_FULL));
      }
      const int r = pc.rg * ROWS + (PAIR ? sx * TILE_M : 0) + row;
      const bool valid = r < all_rows, busy = __any_sync(0xffffffffu, valid);
      const int token = fdiv(min(r, all_rows - 1), p.by_rep), head = pc.hk * rep + min(r, all_rows - 1) - token * rep;
      const unsigned long long own = (pc.first + pc.count) * TILE_N > pc.ctx ? tree_own_keys(t, pc.b, token) : 0ull;
      const uint32_t* const mask_row = MASK ? tree_bits(t, pc.b, token) : nullptr;
      float m_run = -CUDART_INF_F, l_run = 0.f;
      const int n_mine = PAIR ? pc.count : (pc.count + 1 - sx) / 2, tile0 = pc.first, ctx = pc.ctx;
#pragma unroll 1
      for (int i = 0; i < n_mine; ++i, ++kt) {
        const int tile = tile0 + (PAIR ? i : 2 * i + sx), key0 = tile * TILE_N;
        uint4 seen4 = make_uint4(~0u, ~0u, ~0u, ~0u);     // keys of the tile that the mask lets the row's token see
        if (MASK) seen4 = reinterpret_cast<const uint4*>(mask_row)[tile];
        ok = TREE_WAIT(S_FULL + sx, kt, 11 + sx);
        if (!ok) break;
        ptx::tc_fence_after();
        if (!busy) {                                      // no row of this warp exists: its results are never read
          if (PAIR) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_at(bar(S_TAKEN + sx));
            ok = TREE_WAIT(PV_DONE + sx, kt - 1, 13 + sx);                // P is reported once a PV, as by warps with rows
            if (!ok) break;
          }
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_at(bar(P_FULL + sx));
          continue;
        }
        float s[TILE_N];
        uint32_t* const su = reinterpret_cast<uint32_t*>(s);
        float tile_max;
        auto chunk_max = [&](int c) { return sm::row_max(*reinterpret_cast<const float(*)[32]>(&s[32 * c])); };
        // does every token see the whole tile?
        if (key0 + TILE_N <= ctx && (!MASK || __all_sync(0xffffffffu, (seen4.x & seen4.y & seen4.z & seen4.w) == ~0u))) {
          ptx::tmem_ld32(s_addr, su);
          ptx::tmem_wait_ld();
          ptx::tmem_ld32(s_addr + 32, su + 32);
          tile_max = chunk_max(0);
          ptx::tmem_wait_ld();
          ptx::tmem_ld32(s_addr + 64, su + 64);
          tile_max = fmaxf(tile_max, chunk_max(1));
          ptx::tmem_wait_ld();
          ptx::tmem_ld32(s_addr + 96, su + 96);
          tile_max = fmaxf(tile_max, chunk_max(2));
          ptx::tmem_wait_ld();
          if (PAIR) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_at(bar(S_TAKEN + sx));
          }
          tile_max = fmaxf(tile_max, chunk_max(3));
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) ptx::tmem_ld32(s_addr + 32 * c, su + 32 * c);
          ptx::tmem_wait_ld();
          if (PAIR) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_at(bar(S_TAKEN + sx));
          }
          tile_max = -CUDART_INF_F;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int at = key0 + 32 * c - ctx;        // place of the chunk's first key among the tokens' own
            const uint32_t mine = at >= 0 ? (at < 64 ? uint32_t(own >> at) : 0u) : at <= -32 ? ~0u : uint32_t(own << -at) | ((1u << -at) - 1u);
            const uint32_t seen = mine & (c == 0 ? seen4.x : c == 1 ? seen4.y : c == 2 ? seen4.z : seen4.w);
#pragma unroll
            for (int e = 0; e < 32; ++e) s[32 * c + e] = (seen >> e) & 1u ? s[32 * c + e] : -CUDART_INF_F;
            tile_max = fmaxf(tile_max, chunk_max(c));
          }
        }
        const float m_new = fmaxf(m_run, tile_max);
        // the maximum moves only when the scores outgrow it by 2^8; until then probabilities are merely scaled
        const bool grow = (m_new - m_run) * t.scale_log2 > RESCALE_THRESHOLD;
        float alpha = 1.f;
        if (grow) {
          alpha = ptx::ex2((m_run - m_new) * t.scale_log2);
          l_run *= alpha;
          m_run = m_new;
        }
        // The stream's PV before this one reads P and writes O. Where P stands over the scores, it has completed before
        // they came (one thread issues both, in order); else it is waited for.
        if (PAIR) {
          ok = TREE_WAIT(PV_DONE + sx, kt - 1, 13 + sx);
          if (!ok) break;
          ptx::tc_fence_after();
        }
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < HEAD_DIM / 16; ++c) {
            uint32_t o[16];
            ptx::tmem_ld16(o_addr + c * 16, o);
            ptx::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            ptx::tmem_st16(o_addr + c * 16, o);
          }
        }
        const float base = m_run == -CUDART_INF_F ? 0.f : m_run * t.scale_log2;
        sm::f2 sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
          if (PAIR) {
            // Rounded to bf16, half a step (2^-9) each, their sum being taken before: tensor memory is full (scores 128 columns, P 2 x 64,
            // O 2 x 128), so that low halves would need P of half a tile at a time. 64 tokens over 65,536 keys: error against 64 bits
            // 0.0023 of the output's norm, where rounding the output alone makes 0.0017 and 16 bits of P no more than that.
            sm::exp_chunk<sm::EX2_FMA_PAIRS_NONE>(s, c * 32, t.scale_log2, base, pk, sum);
            ptx::tmem_st16(p_addr + c * 16, pk);
          } else {
            uint32_t lo[16];
            const sm::f2 scale2 = sm::pack2(t.scale_log2, t.scale_log2), nbase2 = sm::pack2(-base, -base);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float x0, x1;
              sm::unpack2(sm::fma2(sm::pack2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), scale2, nbase2), x0, x1);
              const float p0 = ptx::ex2(x0), p1 = ptx::ex2(x1);
              sum[e & 3] = sm::add2(sum[e & 3], sm::pack2(p0, p1));
              split_bf16(p0, p1, pk[e], lo[e]);
            }
            ptx::tmem_st16(p_addr + c * 16, pk);
            ptx::tmem_st16(p_addr + 64 + c * 16, lo);
          }
        }
        l_run += sm::sum4(sum);
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_at(bar(P_FULL + sx));
      }
      if (!ok) break;

      // ---- results ----------------------------------------------------------------------------------------
      const int n_other = PAIR ? 0 : (pc.count + sx) / 2;                 // tiles of the other stream
      float m = m_run == -CUDART_INF_F ? -CUDART_INF_F : m_run * t.scale_log2, l = l_run;
      float w_mine = 1.f, w_other = 0.f;
      if (!PAIR) {                                        // the two streams' sums are of the same rows
        float2(*const ml)[PAIR ? 1 : TILE_M] = row_ml[unit & 1];
        ml[sx][PAIR ? 0 : row] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive_at(bar(ML_READY + 2 * sx + (unit & 1)));
        ok = TREE_WAIT(ML_READY + 2 * (sx ^ 1) + (unit & 1), unit >> 1, 45 + sx);
        if (!ok) break;
        const float2 other = ml[sx ^ 1][PAIR ? 0 : row];
        const float m_all = fmaxf(m, other.x);
        w_mine = n_mine > 0 ? merge_weight(m, m_all) : 0.f;
        w_other = n_other > 0 ? merge_weight(other.x, m_all) : 0.f;
        l = w_mine * l + w_other * other.y;
        m = m_all;
      }
      if (n_mine > 0) ok = TREE_WAIT(O_DONE + sx, done[sx], 41);
      if (ok && n_other > 0) ok = TREE_WAIT(O_DONE + (sx ^ 1), done[sx ^ 1], 42);
      if (!ok) break;
      done[sx] += n_mine > 0;
      done[sx ^ 1] += n_other > 0;
      ptx::tc_fence_after();
      const int col = PAIR ? 0 : sx * COLS;               // !PAIR: set s takes half s of the columns, of both streams
      auto chunk = [&](int c, float (&o)[32]) {           // sums of 32 columns, called by whole warps
        uint32_t y[32];
        if constexpr (PAIR) {
          ptx::tmem_ld32(o_addr + c, y);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(y[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if ((x == sx ? n_mine : n_other) > 0) {
              const float w = x == sx ? w_mine : w_other;
              ptx::tmem_ld32(lane_addr + 256 + x * 128 + col + c, y);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] += w * __uint_as_float(y[e]);
            }
          }
        }
      };
      bool finite = true;
      if (busy) {
        __nv_bfloat16* const out = t.o + ((int64_t(pc.b) * t.n + token) * t.H + head) * HEAD_DIM;
        float* part = nullptr;                            // column c of the row at part[c * ROWS]
        if (pc.count != pc.of) {
          part = t.scratch + (int64_t(blockIdx.x) * 2 + pc.starts) * UMMA_PARTIAL<PAIR>;
          const int at = r - pc.rg * ROWS;
          if (valid && col == 0) reinterpret_cast<float2*>(part + int64_t(ROWS) * HEAD_DIM)[at] = make_float2(m, l);
          part += at;
        }
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32) {
          float o[32];
          chunk(c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) finite = finite && fabsf(o[e]) < CUDART_INF_F;
          if (!valid) continue;
          if (part != nullptr) {
#pragma unroll
            for (int e = 0; e < 32; ++e) part[(col + c + e) * ROWS] = o[e];
          } else {
            uint4* const d = reinterpret_cast<uint4*>(out + col + c);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              d[e] = make_uint4(ptx::pack_bf16(o[8 * e] * inv, o[8 * e + 1] * inv), ptx::pack_bf16(o[8 * e + 2] * inv, o[8 * e + 3] * inv),
                                ptx::pack_bf16(o[8 * e + 4] * inv, o[8 * e + 5] * inv), ptx::pack_bf16(o[8 * e + 6] * inv, o[8 * e + 7] * inv));
          }
        }
        if (__any_sync(0xffffffffu, valid && !finite)) {
          __syncwarp();
          tree_exact_rows<PAIR>(p, pieces[warp], m, l, valid && !finite);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_at(bar(O_FREE + sx));              // the next unit's first PV may overwrite O
      ++unit;
    }
  } else if (warp < 12) {
    // ================================ requests of the tiles ========================================
    ptx::setmaxnreg_dec<UMMA_LOAD_REGS>();
    const int lt = tid - 256;                             // 0 .. 127; in copies: row lt >> 4 of every 8, piece lt & 15
    int copied = -1;                                      // buffer whose copies this thread has issued and not reported
    auto report = [&] {
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive_at(bar(FULL + copied));
      copied = -1;
    };
    // `any`: keys of the tile that some token sees
    struct Place { int b, hk, n_keys; };
    auto request = [&](uint32_t req, int operand, const Place& x, int tile, const uint4& any) {
      const uint32_t slot = req % RING, dst = ring_smem + slot * TILE_BYTES;
      if (!(ok = TREE_WAIT(FREE + slot, req / RING - 1, 21 + operand))) return;
      const int key0 = tile * TILE_N;
      const bool all = (any.x & any.y & any.z & any.w) == ~0u;
      if (p.use_tma && all && (key0 + TILE_N <= x.n_keys || x.n_keys == t.S)) {  // rows past the cache's end come as zeros
        if (copied >= 0) { ptx::cp_async_wait<0>(); report(); }
        if (lt == 0) {
          ptx::mbar_expect_tx_at(bar(FULL + slot), TILE_BYTES);
          ptx::tma_load_5d_at(dst, &p.maps[operand], bar(FULL + slot), 0, key0, 0, x.hk, x.b);
          ptx::tma_load_5d_at(dst + HALF_BYTES, &p.maps[operand], bar(FULL + slot), 64, key0, 0, x.hk, x.b);
        } else {
          ptx::mbar_arrive_at(bar(FULL + slot));
        }
        return;
      }
      const TensorView& st = operand ? t.vs : t.ks;
      const __nv_bfloat16* const src = (operand ? t.v : t.k) + x.b * st.sb + x.hk * st.sh + (lt & 15) * 8;
#pragma unroll 4
      for (int c = 0; c < TILE_N / 8; ++c) {
        const int row = c * 8 + (lt >> 4);
        const uint32_t word = c < 4 ? any.x : c < 8 ? any.y : c < 12 ? any.z : any.w;
        const bool there = key0 + row < x.n_keys && ((word >> (row & 31)) & 1u);
        ptx::cp_async_16(dst + tile_offset(row, lt & 15), there ? src + (key0 + row) * st.ss : src, there ? 16u : 0u);
      }
      ptx::cp_async_commit();
      // A tile is reported when the next one's copies are under way; nothing that the next buffer waits for needs it.
      if (copied >= 0) { ptx::cp_async_wait<1>(); report(); }
      copied = int(slot);
    };
    uint32_t j = 0;
    Place before = {0, 0, 0};                             // of the tile whose V is requested next
    uint4 v_any = make_uint4(~0u, ~0u, ~0u, ~0u);
    int v_tile = -1;
    while (ok && tree_next(t, walk, pieces[warp])) {
      const Place here = {pc.b, pc.hk, pc.n_keys};
      const int first = pc.first, count = pc.count;
      for (int i = 0; i < count && ok; ++i, ++j) {
        uint4 any = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (MASK) any = reinterpret_cast<const uint4*>(t.any + int64_t(here.b) * t.bits_words)[first + i];
        request(k_request(j), 0, here, first + i, any);
        if (ok && v_tile >= 0) request(v_request(j - 1), 1, before, v_tile, v_any);
        before = here;
        v_tile = first + i;
        if (MASK) v_any = any;
      }
    }
    if (ok && v_tile >= 0) request(v_request(j - 1), 1, before, v_tile, v_any);
    ptx::cp_async_wait<0>();
    if (copied >= 0) report();
  } else {
    ptx::setmaxnreg_dec<UMMA_ISSUE_REGS>();
    // ================================ MMA issue ====================================================
    const uint64_t q_desc = tile_desc_kmajor(q_smem), k_desc = tile_desc_kmajor(ring_smem), v_desc = tile_desc_mnmajor(ring_smem);
    constexpr uint64_t STEP = TILE_BYTES >> 4;             // descriptor distance between buffers
    uint32_t j = 0, unit = 0, kt[2] = {0, 0};              // tiles of the CTA before this unit, units, tiles per stream
    // Scores of tile j for stream sx; `last` reads K last, `final` the unit's queries.
    auto qk = [&](uint32_t tile, int sx, bool first_of_unit, bool last, bool final) {
      const uint32_t req = k_request(tile), slot = req % RING;
      ok = (!first_of_unit || TREE_WAIT(Q_FULL, unit, 31)) && TREE_WAIT(FULL + slot, req / RING, 32);
      if (PAIR && ok) ok = TREE_WAIT(S_TAKEN + (sx ^ 1), sx ? tile : tile - 1, 33);      // the other set has copied its scores out
      if (!ok) return;
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        issue_qk_loop(q_desc + (PAIR ? sx : 0) * STEP, k_desc + slot * STEP, tmem + (PAIR ? 0 : sx * 128));
        ptx::mma_commit_at(bar(S_FULL + sx));
        if (last) ptx::mma_commit_at(bar(FREE + slot));
        if (final) ptx::mma_commit_at(bar(Q_FREE));
      }
      __syncwarp();
    };
    auto pv = [&](uint32_t tile, int sx, bool first_of_stream, bool last, bool final) {
      const uint32_t req = v_request(tile), slot = req % RING;
      ok = TREE_WAIT(FULL + slot, req / RING, 40);
      if (ok && first_of_stream) ok = TREE_WAIT(O_FREE + sx, unit - 1, 37) && (PAIR || TREE_WAIT(O_FREE + (sx ^ 1), unit - 1, 38));
      if (ok) ok = TREE_WAIT(P_FULL + sx, kt[sx], 35);
      if (!ok) return;
      ++kt[sx];
      ptx::tc_fence_after();
      if (ptx::elect_one()) {
        const uint32_t p_cols = PAIR ? tmem + 128 + sx * 64 : tmem + sx * 128;
        issue_pv_loop(p_cols, v_desc + slot * STEP, tmem + 256 + sx * 128, first_of_stream ? 0 : 1);
        if (!PAIR) issue_pv_loop(p_cols + 64, v_desc + slot * STEP, tmem + 256 + sx * 128, 1);
        if (PAIR) ptx::mma_commit_at(bar(PV_DONE + sx));
        if (last) ptx::mma_commit_at(bar(FREE + slot));
        if (final) ptx::mma_commit_at(bar(O_DONE + sx));
      }
      __syncwarp();
    };
    if (warp == 12 || (PAIR && warp == 13)) {
      while (ok && tree_next(t, walk, pieces[warp])) {
        const int count = pc.count;
        if (PAIR) {
#pragma unroll 1
          for (int i = 0; i < count && ok; ++i)
#pragma unroll 1
            for (int sx = 0; sx < 2 && ok; ++sx) {
              if (warp == 12) qk(j + i, sx, i == 0 && sx == 0, sx == 1, sx == 1 && i == count - 1);
              else pv(j + i, sx, i == 0, sx == 1, i == count - 1);
            }
        } else {
#pragma unroll 1
          for (int i = -2; i < count && ok; ++i) {         // PV of tile i, then QK^T of tile i + 2 into the scores it has read
            if (i >= 0) pv(j + i, i & 1, i < 2, true, i + 2 >= count);
            if (ok && i + 2 < count) qk(j + i + 2, i & 1, i == -2, true, i + 3 == count);
          }
        }
        j += count;
        ++unit;
      }
      if (!ok) {                                           // let MMAs in flight finish before TMEM is freed
        const int drain = DRAIN + (warp - 12);
        if (ptx::elect_one()) ptx::mma_commit_at(bar(drain));
        __syncwarp();
        int dummy = 0;
        ptx::mbar_wait(&bars[drain], 0, &dummy, 100);
      }
    } else if (warp >= 14) {
      // ================================ query rows ==================================================
      while (ok && tree_next(t, walk, pieces[warp])) {
        if (unit > 0) {
          ok = TREE_WAIT(Q_FREE, unit - 1, 23);
          if (!ok) break;
          copy_queries(pc, 2 * (warp - 14) + (lane >> 4), 4);
          if (lane < 4) ptx::mbar_arrive_at(bar(Q_FULL));
        }
        ++unit;
      }
    }
  }
#undef TREE_WAIT

  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && abort_flag != 0) {
    ptx::drain_copies(bars, FREE);                         // tiles that were requested before the give-up
    atomicCAS(p.status, 0, STATUS_WAIT_BASE + abort_flag);
  }
}

// A boolean mask as bits: per token a word for 32 keys, the same of the keys any token sees, and which tiles hold such keys (a
// byte for eight). CTA: 32 words of one sequence, eight tokens at a time; the words are padded to whole tiles with zeros.
constexpr int TREE_MASK_ROWS = 8;
__global__ void __launch_bounds__(32 * TREE_MASK_ROWS) tree_mask_kernel(const __grid_constant__ TreeParams p) {
  __shared__ uint32_t part[TREE_MASK_ROWS][32];
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, b = blockIdx.y;
  const int word = blockIdx.x * 32 + lane, key0 = word * 32;
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  uint32_t any = 0;
  if (word < p.bits_words) {
    for (int i = y; i < p.bits_tokens; i += TREE_MASK_ROWS) {
      const uint8_t* const m = p.mask + b * p.mask_sb + i * p.mask_sn + key0 * p.mask_ss;
      uint32_t bits = 0;
      if (p.mask_vec && key0 + 32 <= p.S) {
        const uint4 w[2] = {reinterpret_cast<const uint4*>(m)[0], reinterpret_cast<const uint4*>(m)[1]};
        const uint32_t ws[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
        for (int c = 0; c < 8; ++c) bits |= ((__vminu4(ws[c], 0x01010101u) * 0x10204080u) >> 28) << (4 * c);      // a byte's 0 or not, four at a time
      } else {
        for (int c = 0; c < 32 && key0 + c < p.S; ++c) bits |= m[c * p.mask_ss] != 0 ? 1u << c : 0u;
      }
      const_cast<uint32_t*>(p.bits)[(int64_t(b) * p.bits_tokens + i) * p.bits_words + word] = bits;
      any |= bits;
    }
  }
  part[y][lane] = any;
  __syncthreads();
  if (y != 0) return;
#pragma unroll
  for (int i = 1; i < TREE_MASK_ROWS; ++i) any |= part[i][lane];
  if (word < p.bits_words) const_cast<uint32_t*>(p.any)[int64_t(b) * p.bits_words + word] = any;
  const uint32_t words = __ballot_sync(0xffffffffu, any != 0u);
  if (lane == 0) {
    uint32_t tiles = 0;
#pragma unroll
    for (int c = 0; c < 8; ++c) tiles |= (words >> (4 * c)) & 15u ? 1u << c : 0u;
    const_cast<uint8_t*>(p.live)[int64_t(b) * p.live_words * 8 + blockIdx.x] = uint8_t(tiles);
  }
}

// Joins the partial results of units that several CTAs had a part of. A thread has four rows and COLS columns, a warp 32 rows and
// four times as many columns, and every SPLIT-th part; AT_ONCE parts' loads are under way together. What takes time is the
// loads' latency, so with units of many parts two warps share them (COLS 4, SPLIT 2), and where there are more units one
// warp has as much of two parts as it can hold (COLS 8, SPLIT 1). 32 rows: 8 units of 18 parts, the whole call 61.5 us against 68.1 with
// the other form; 128 rows, 96 units of 2 or 3: 55.3 against 81.6 with (2, 4); a thread with one row and scalar loads 62.8.
// `row_blocks`: 32-row blocks of a unit. Loads of rows that do not exist stay inside the buffer and are not used.
constexpr int UMMA_MERGE_WARPS = 4;
constexpr int UMMA_MERGE_FEW = 4;                // parts a unit up to which a warp takes them all
template <int COLS, int SPLIT> constexpr int UMMA_MERGE_CTAS = HEAD_DIM / (4 * COLS * UMMA_MERGE_WARPS / SPLIT);      // per 32 rows
template <bool PAIR, int COLS, int SPLIT>
__global__ void __launch_bounds__(32 * UMMA_MERGE_WARPS) tree_umma_merge_kernel(const __grid_constant__ TreeUmmaParams p, uint32_t grid, int row_blocks) {
  constexpr int ROWS = UMMA_ROWS<PAIR>, CTAS = UMMA_MERGE_CTAS<COLS, SPLIT>, AT_ONCE = COLS == 8 ? 2 : 4;
  __shared__ float joined[SPLIT > 1 ? UMMA_MERGE_WARPS : 1][SPLIT > 1 ? 4 * (COLS + 2) : 1][32];
  const TreeParams& t = p.t;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rep = t.H / t.Hkv;
  const int block = blockIdx.x / CTAS, col_block = blockIdx.x - block * CTAS;
  const int unit = block / row_blocks, block_row = (block - unit * row_blocks) * 32, at = block_row + (lane & 7) * 4;
  const int units = t.Hkv * t.row_groups, b = unit / units, in_b = unit - b * units;
  const int hk = in_b / t.row_groups, rg = in_b - hk * t.row_groups;
  const int col = ((col_block * (UMMA_MERGE_WARPS / SPLIT) + warp / SPLIT) * 4 + (lane >> 3)) * COLS;
  if (rg * ROWS + block_row >= t.n * rep) return;         // the last row group's blocks without rows
  uint32_t start;
  const TreeList<TILE_N> list(t, t.B, grid, b, &start);
  const int tiles = tree_tiles<TILE_N>(t, b);
  start += uint32_t(in_b + 1) * list.places(tiles) - tiles;        // place of the unit's first tile
  const int c0 = int(start / list.per), c1 = int((start + tiles - 1) / list.per);
  cudaGridDependencySynchronize();                        // everything before this ran beside the main kernel's end
  if (c0 == c1) return;                                   // one CTA held the unit and wrote its rows
  // The part in the CTA the unit begins in is that CTA's second slot, in the others the first.
  const float* const first = t.scratch + (int64_t(c0) * 2 + 1) * UMMA_PARTIAL<PAIR>;
  const int parts = c1 - c0 + 1;
  float m_all[4], l_all[4], acc[COLS][4];                 // [column][row]
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m_all[r] = -CUDART_INF_F;
    l_all[r] = 0.f;
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[c][r] = 0.f;
  }
  for (int i0 = warp % SPLIT; i0 < parts; i0 += AT_ONCE * SPLIT) {         // running maximum over batches of parts
    float4 x[AT_ONCE][2], o[AT_ONCE][COLS];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int c = min(i0 + i * SPLIT, parts - 1);
      const float* const slot = first + (c == 0 ? 0 : (int64_t(c) * 2 - 1) * UMMA_PARTIAL<PAIR>);
#pragma unroll
      for (int h = 0; h < 2; ++h) x[i][h] = reinterpret_cast<const float4*>(slot + ROWS * HEAD_DIM + 2 * at)[h];
#pragma unroll
      for (int e = 0; e < COLS; ++e) o[i][e] = *reinterpret_cast<const float4*>(slot + (col + e) * ROWS + at);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      auto max_of = [&](int i) { return r == 0 ? x[i][0].x : r == 1 ? x[i][0].z : r == 2 ? x[i][1].x : x[i][1].z; };
      auto sum_of = [&](int i) { return r == 0 ? x[i][0].y : r == 1 ? x[i][0].w : r == 2 ? x[i][1].y : x[i][1].w; };
      float m_new = m_all[r];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) m_new = fmaxf(m_new, max_of(i));
      const float alpha = merge_weight(m_all[r], m_new);
      l_all[r] *= alpha;
#pragma unroll
      for (int e = 0; e < COLS; ++e) acc[e][r] *= alpha;
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const bool there = i0 + i * SPLIT < parts;
        const float f = there ? merge_weight(max_of(i), m_new) : 0.f;
        l_all[r] += there ? f * sum_of(i) : 0.f;
#pragma unroll
        for (int e = 0; e < COLS; ++e) {
          const float4& y = o[i][e];
          acc[e][r] += there ? f * (r == 0 ? y.x : r == 1 ? y.y : r == 2 ? y.z : y.w) : 0.f;
        }
      }
      m_all[r] = m_new;
    }
  }
  if (SPLIT > 1) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      joined[warp][r][lane] = m_all[r];
      joined[warp][4 + r][lane] = l_all[r];
#pragma unroll
      for (int e = 0; e < COLS; ++e) joined[warp][8 + 4 * e + r][lane] = acc[e][r];
    }
    __syncthreads();
    if (warp % SPLIT != 0) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int w = 1; w < SPLIT; ++w) m_all[r] = fmaxf(m_all[r], joined[warp + w][r][lane]);
      l_all[r] = 0.f;
#pragma unroll
      for (int e = 0; e < COLS; ++e) acc[e][r] = 0.f;
#pragma unroll
      for (int w = 0; w < SPLIT; ++w) {
        const float f = merge_weight(joined[warp + w][r][lane], m_all[r]);
        l_all[r] += f * joined[warp + w][4 + r][lane];
#pragma unroll
        for (int e = 0; e < COLS; ++e) acc[e][r] += f * joined[warp + w][8 + 4 * e + r][lane];
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = rg * ROWS + at + r;
    if (row >= t.n * rep) break;
    const float inv = l_all[r] == 0.f ? 0.f : 1.f / l_all[r];
    const int token = fdiv(row, p.by_rep), head = hk * rep + row - token * rep;
    __nv_bfloat16* const out = t.o + ((int64_t(b) * t.n + token) * t.H + head) * HEAD_DIM + col;
    uint32_t w[COLS / 2];
#pragma unroll
    for (int e = 0; e < COLS / 2; ++e) w[e] = ptx::pack_bf16(acc[2 * e][r] * inv, acc[2 * e + 1][r] * inv);
    if constexpr (COLS == 8) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  }
}

}  // namespace intra
