// How the work of attention over a batch of caches is dealt to CTAs: by key tiles, whatever sequence they belong to. A unit
// is a KV head of a sequence with the rows (tokens times query heads) that one pass over its keys takes. All key tiles of
// all units stand in one list, CTA c takes the c-th part of it: sequences of any lengths, known on the device only, load the
// CTAs evenly. A unit that no CTA holds as a whole leaves partial results - sums, maxima, weights - that a second
// launch joins.
#pragma once
#include <math_constants.h>
#include <stdint.h>

#include "attn_kernel.cuh"

namespace intra {

constexpr int TREE_MAX_TOKENS = 64;              // ancestors of a token fit a 64-bit word

struct TreeParams {
  const __nv_bfloat16* q;      // (B, H, n, 128) by strides
  const __nv_bfloat16* k;      // (B, S, Hkv, 128) by strides
  const __nv_bfloat16* v;
  const int* parents;          // n per sequence, null: each token follows the one before it
  const int* lengths;          // keys before the tokens' own, per sequence; null: S - n
  const uint8_t* mask;         // (B, n, S) by strides, nonzero = visible; null: no further mask
  __nv_bfloat16* o;            // (B, n, H, 128) contiguous
  float* scratch;              // partial results
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
  // tree_mma_kernel.cuh, a decode step that accumulates: (B, Hkv, S) by strides, unit stride over keys, and the scores of
  // every visible key, [unit][row][score_keys], times scale_log2; a unit has as many rows there as it has query heads at most
  float* weights;
  int64_t weights_sb, weights_sh;
  int weights_vec;             // four weights can be loaded at once
  float* scores;
  int score_keys, score_rows;
  int S, H, Hkv, n, B;
  int row_groups;              // units per KV head
  int unit_cost, min_tiles;    // see TreeList; a CTA's part is at least this many tiles
  int split_cost;              // tiles a CTA may have more where in return no unit is divided
  float scale_log2;
};

// Keys before the tokens' own. A length that leaves the tokens no room is brought into range, so that no key outside the
// cache is read whatever it says.
__device__ __forceinline__ int tree_context(const TreeParams& p, int b) {
  const int most = p.S - p.n;
  return p.lengths ? min(max(p.lengths[b], 0), most) : most;
}

struct TreePiece {             // what a CTA does of one unit
  int b, hk, rg;               // sequence, KV head, row group
  int first, count;            // key tiles
  int of;                      // key tiles of the whole unit
  int starts;                  // the piece begins with the unit
  int ctx, n_keys;
};
// Key tiles of KEYS keys of a sequence; where the mask's tiles are known (p.live, tiles of 128 keys) from the first to the last
// of which any token sees a key (one, where there is none).
template <int KEYS>
__device__ __forceinline__ int tree_tiles(const TreeParams& p, int b, int* first = nullptr) {
  const int all = (tree_context(p, b) + p.n + KEYS - 1) / KEYS;
  int lo = 0, hi = all;
  if (KEYS == TILE_N && p.live != nullptr) {
    const unsigned long long* const live = reinterpret_cast<const unsigned long long*>(p.live) + int64_t(b) * p.live_words;
    lo = all;
    hi = 0;
    for (int i = 0; i * 64 < all; ++i) {
      const int left = all - i * 64;
      const unsigned long long x = live[i] & (left >= 64 ? ~0ull : (1ull << left) - 1ull);
      if (x) {
        lo = min(lo, i * 64 + __ffsll(x) - 1);
        hi = i * 64 + 64 - __clzll(x);
      }
    }
    if (hi == 0) { lo = 0; hi = 1; }
  }
  if (first) *first = lo;
  return hi - lo;
}

// Are `units` units of at most `longest` tiles, `tiles` in all, dealt whole? See TreeList. Not where most CTAs would have none: 8 units
// of 8 tiles on 32 CTAs take 13.4 us divided, 18 whole.
__host__ __device__ __forceinline__ bool tree_whole(uint32_t units, uint32_t tiles, uint32_t longest, uint32_t grid, int split_cost) {
  return split_cost > 0 && units * 2 >= grid && uint64_t((units + grid - 1) / grid) * longest <= uint64_t(tiles / grid) + split_cost;
}

// The list of all units' key tiles. A unit counts for `cost` places more than it has tiles, in front of them: what the end of
// one unit and the start of the next cost the CTA that has both; at most a quarter of a CTA's share of tiles, since parts of a
// few tiles would only be spread unevenly by it. 26 tokens over 8 caches of 4,096 to 8,192 keys 59.9 -> 56.5 us, 32 rows over
// 65,536 keys 62 -> 58.8, against 1 place (3 above 128 rows; 4 of 16 keys in the kernel for few rows, now 20) from 16 tiles on;
// with an eighth 58.5 and 60.3, with a third the same, but 32 caches of 300 to 3,000 5 % more.
// Where CTAs that each take the same number of whole units are done about as early as with parts of equal size - by
// p.split_cost tiles, what partial results and their merge take - the list is dealt so: every unit then has as many places as
// the longest. With two or more CTAs a unit, each unit is divided into the same number of parts if those are not longer than
// equal ones by more than a tile, so that no CTA has two pieces: one sequence of 8,000 keys, 32 rows 23.7 -> 19.4 us, 16 rows
// 23.1 -> 20.7, four of 3,000 keys 24.7 -> 22.4; calls of a few tiles lose up to 0.5. At most 2^31 - 1 places.
template <int KEYS>
struct TreeList {
  uint32_t units, cost, per, total;      // units per sequence; places of a CTA's part, of all
  uint32_t even;                         // places of every unit, 0: as many as they have tiles, and `cost`
  __device__ __forceinline__ uint32_t places(uint32_t tiles) const { return even ? even : tiles + cost; }
  // Called by whole warps; all lanes get the same. `before`: places of sequences before `b`.
  __device__ __forceinline__ TreeList(const TreeParams& p, int B, uint32_t grid, int b = 0, uint32_t* before = nullptr) {
    units = p.Hkv * p.row_groups;
    uint32_t tiles = 0, front = 0, longest = 0;
    if (p.lengths == nullptr && p.live == nullptr) {               // all sequences alike
      longest = uint32_t(tree_tiles<KEYS>(p, 0));
      tiles = uint32_t(B) * longest;
      front = uint32_t(b) * longest;
    } else {
      for (int s = threadIdx.x & 31; s < B; s += 32) {
        const uint32_t n = tree_tiles<KEYS>(p, s);
        tiles += n;
        front += s < b ? n : 0u;
        longest = max(longest, n);
      }
      tiles = __reduce_add_sync(0xffffffffu, tiles);
      front = __reduce_add_sync(0xffffffffu, front);
      longest = __reduce_max_sync(0xffffffffu, longest);
    }
    const uint32_t share = tiles * units / grid;
    even = tree_whole(units * B, tiles * units, longest, grid, p.split_cost) ? longest : 0;
    cost = share < uint32_t(p.min_tiles) ? 0 : min(share / 4, uint32_t(p.unit_cost));
    per = max(((tiles + cost * B) * units + grid - 1) / grid, uint32_t(p.min_tiles));
    if (even) {
      per = (units * B + grid - 1) / grid * even;
    } else if (units * B * 2 <= grid) {                            // the same number of parts of every unit
      const uint32_t k = grid / (units * B), part = (longest + k - 1) / k;
      if (part <= per + 1) { per = part; even = k * part; }
    }
    total = (even ? even * B : tiles + cost * B) * units;
    if (before) *before = (even ? even * b : front + cost * b) * units;
  }
};

// A CTA's part [next, end) of the list as a cursor that every warp moves by itself. Cursor and piece stand in shared memory: the
// tcgen05 kernel's softmax warps, which hold a row's 128 scores, have no registers left for them.
template <int KEYS>
struct TreeWalk {
  uint32_t next, end;
  uint32_t b_start;            // place of sequence b's first unit
  uint32_t units, cost, even;
  int b, b_tiles, b_first;     // of one unit: its tiles, the first of them
  // Called by whole warps; all lanes get the same.
  __device__ __forceinline__ void start(const TreeParams& p, int B, uint32_t cta, uint32_t grid) {
    const int lane = threadIdx.x & 31;
    const TreeList<KEYS> list(p, B, grid);
    units = list.units;
    cost = list.cost;
    even = list.even;
    next = list.per * cta < list.total ? list.per * cta : list.total;
    end = list.total - next > list.per ? next + list.per : list.total;
    b = b_tiles = b_first = 0;
    b_start = 0;
    if (next >= end) return;
    for (int s0 = 0; s0 < B; s0 += 32) {                           // the sequence that holds `next`
      const uint32_t mine = s0 + lane < B ? list.places(tree_tiles<KEYS>(p, s0 + lane)) * units : 0u;
      uint32_t upto = mine;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, b_start + upto > next);
      if (past) {
        b = s0 + __ffs(past) - 1;
        b_start += __shfl_sync(0xffffffffu, upto - mine, __ffs(past) - 1);
        break;
      }
      b_start += __shfl_sync(0xffffffffu, upto, 31);
    }
    b_tiles = tree_tiles<KEYS>(p, b, &b_first);
  }
  __device__ __forceinline__ void piece(const TreeParams& p, TreePiece& x) {
    x.count = 0;
    while (next < end) {
      uint32_t places = even ? even : b_tiles + cost;
      if (next - b_start >= places * units) {
        b_start += places * units;
        b_tiles = tree_tiles<KEYS>(p, ++b, &b_first);
        places = even ? even : b_tiles + cost;
      }
      const uint32_t local = next - b_start, unit = local / places, at = local - unit * places;
      const uint32_t take = min(end - next, places - at);
      next += take;
      const int in_front = int(places) - b_tiles;                  // places without tiles
      const int first = max(int(at) - in_front, 0), last = int(at + take) - in_front;
      if (last <= first) continue;                                 // of this unit only places without tiles
      x.b = b;
      x.hk = p.row_groups == 1 ? unit : unit / p.row_groups;
      x.rg = unit - x.hk * p.row_groups;
      x.of = b_tiles;
      x.first = b_first + first;
      x.count = last - first;
      x.starts = first == 0;
      x.ctx = tree_context(p, b);
      x.n_keys = x.ctx + p.n;
      return;
    }
  }
};
// The warp's next piece of its CTA's part; false: there is none.
template <int KEYS>
__device__ __forceinline__ bool tree_next(const TreeParams& p, TreeWalk<KEYS>& walk, TreePiece& x) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) walk.piece(p, x);
  __syncwarp();
  return x.count > 0;
}

// The tokens' own keys that `token` sees, itself included, as bits; called by whole warps, a lane holding tokens lane and
// lane + 32. A parent that is not an earlier token ends the walk. Pointer doubling: six rounds for 64 tokens.
__device__ __forceinline__ unsigned long long tree_own_keys(const TreeParams& p, int b, int token) {
  if (p.all_own) return (2ull << (p.n - 1)) - 1ull;
  if (p.parents == nullptr) return (2ull << token) - 1ull;
  const int lane = threadIdx.x & 31;
  unsigned long long anc[2];
  int up[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int i = lane + 32 * c, parent = i < p.n ? p.parents[b * p.parents_sb + i] : -1;
    up[c] = parent >= 0 && parent < i ? parent : -1;
    anc[c] = 1ull << i;
  }
  auto of_token = [](const unsigned long long (&x)[2], int i) {
    const unsigned long long a = __shfl_sync(0xffffffffu, x[0], i & 31), c = __shfl_sync(0xffffffffu, x[1], i & 31);
    return i & 32 ? c : a;
  };
  for (int reach = 1; reach < p.n; reach *= 2) {
    unsigned long long more[2];
    int next[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = up[c] < 0 ? 0 : up[c];
      const int a = __shfl_sync(0xffffffffu, up[0], i & 31), d = __shfl_sync(0xffffffffu, up[1], i & 31);
      const unsigned long long x = of_token(anc, i);
      more[c] = up[c] < 0 ? 0ull : x;
      next[c] = up[c] < 0 ? -1 : i & 32 ? d : a;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) { anc[c] |= more[c]; up[c] = next[c]; }
  }
  return of_token(anc, token);
}

}  // namespace intra
