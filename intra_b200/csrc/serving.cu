// Host side of the serving operators behind the C ABI of include/intra_b200.h: attention of drafted tokens over a cache,
// their verification, and what happens to the cache between two steps. Argument checks, how the work is split, launches.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <mutex>

#include "cache_kernel.cuh"
#include "host.h"
#include "tma_encode.h"
#include "tree_mma_kernel.cuh"
#include "tree_umma_kernel.cuh"
#include "verify_kernel.cuh"

namespace {

using namespace intra;

// Where this file's kernels record a bounded wait that ran out. Part of the library image, so that nothing is allocated.
__device__ int g_serving_status;

struct ServingState {
  std::once_flag once;
  int init_status = INTRA_OK;
  int sm_count = 0;
  int* status_word = nullptr;     // g_serving_status on this device
};
ServingState g_serving[MAX_DEVICES];

// Runs once per device with that device current. Allocates nothing, so a first call may be captured.
void init_serving(int device) {
  ServingState& st = g_serving[device];
  int major = 0;
  cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (e != cudaSuccess) { st.init_status = cuda_fail(e); return; }
  if (major != 10) { st.init_status = INTRA_ERR_DEVICE; return; }
  e = cudaDeviceGetAttribute(&st.sm_count, cudaDevAttrMultiProcessorCount, device);
  if (e == cudaSuccess) e = opt_in_smem(tree_mma_kernel<false, false>, tree_smem_bytes(TREE_MAX_TOKENS));
  if (e == cudaSuccess) e = opt_in_smem(tree_mma_kernel<false, true>, tree_smem_bytes(TREE_MAX_TOKENS));
  if (e == cudaSuccess) e = opt_in_smem(tree_mma_kernel<true, false>, tree_smem_bytes(TREE_MAX_TOKENS));
  if (e == cudaSuccess) e = opt_in_smem(tree_mma_kernel<true, true>, tree_smem_bytes(TREE_MAX_TOKENS));
  if (e == cudaSuccess) e = opt_in_smem(tree_umma_kernel<false, false>, UMMA_SMEM_BYTES<false>);
  if (e == cudaSuccess) e = opt_in_smem(tree_umma_kernel<false, true>, UMMA_SMEM_BYTES<false>);
  if (e == cudaSuccess) e = opt_in_smem(tree_umma_kernel<true, false>, UMMA_SMEM_BYTES<true>);
  if (e == cudaSuccess) e = opt_in_smem(tree_umma_kernel<true, true>, UMMA_SMEM_BYTES<true>);
  void* word = nullptr;
  if (e == cudaSuccess) e = cudaGetSymbolAddress(&word, g_serving_status);
  st.status_word = static_cast<int*>(word);
  if (e == cudaSuccess) e = opt_in_smem(verify_kernel<float>, VERIFY_SMEM_BYTES);
  if (e == cudaSuccess) e = opt_in_smem(verify_kernel<__nv_bfloat16>, VERIFY_SMEM_BYTES);
  if (e == cudaSuccess) e = opt_in_smem(verify_kernel<__half>, VERIFY_SMEM_BYTES);
  if (e == cudaSuccess) e = opt_in_smem(evict_select_kernel<true>, EVICT_SMEM_KEYS * 4);
  if (e != cudaSuccess) st.init_status = cuda_fail(e);
}

// The device's state, set up on the first call; `guard` has made the device current.
int serving_device(int device, const DeviceGuard& guard, const ServingState** st) {
  if (!guard.ok) return cuda_fail(cudaGetLastError());
  std::call_once(g_serving[device].once, init_serving, device);
  *st = &g_serving[device];
  return (*st)->init_status;
}

bool rows_aligned(const int64_t s[3]) { return ((s[0] | s[1] | s[2]) & 7) == 0; }
TensorView view_of(const int64_t s[3]) { return {s[0], s[1], s[2]}; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

template <typename K, typename P>
cudaError_t launch_cluster(K kernel, int64_t clusters, int cluster, int threads, int smem, cudaStream_t stream, const P& p,
                           int early = 0) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {unsigned(cluster), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = early;
  cfg.gridDim = dim3(unsigned(clusters * cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

// Launch of a kernel that may be set up while the kernel before it in the stream still runs, and that waits for that one's
// end (cudaGridDependencySynchronize) before it touches memory.
template <typename K, typename... P>
cudaError_t launch_early(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const P&... p) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p...);
}

// Up to 16 rows per KV head, or any number of one token's whose weights are accumulated.
template <bool ACCUMULATE>
int launch_tree_mma(TreeParams p, const ServingState& st, int64_t scratch_bytes, int64_t* scratch_needed, cudaStream_t stream) {
  const int all_rows = p.n * (p.H / p.Hkv);
  p.row_groups = ceil_div(all_rows, TREE_ROWS);
  p.unit_cost = TREE_UNIT_COST;
  p.min_tiles = TREE_MIN_BLOCKS;
  const int64_t units = int64_t(p.B) * p.Hkv * p.row_groups, rows = int64_t(p.B) * p.Hkv * all_rows;
  const int64_t blocks = units * ceil_div(p.S, TREE_BLOCK), places = blocks + units * TREE_UNIT_COST;      // at most
  const int slots = st.sm_count * TREE_CTAS_PER_SM;
  if (places + slots * int64_t(TREE_MIN_BLOCKS) > 0x7fffffffLL || rows > 0x7fffffffLL) return INTRA_ERR_UNSUPPORTED;
  const int64_t parts = (blocks + TREE_MIN_BLOCKS - 1) / TREE_MIN_BLOCKS, ctas = parts > units ? parts : units;
  const int grid = ctas < slots ? int(ctas) : slots;
  p.split_cost = TREE_SPLIT_COST;
  int64_t floats = (grid + units) * int64_t(TREE_PARTIAL);
  if (ACCUMULATE) {
    if (int64_t(p.B) * p.Hkv > 65535) return INTRA_ERR_UNSUPPORTED;      // grid.y of the accumulation
    p.score_keys = ceil_div(p.S, TREE_BLOCK) * TREE_BLOCK;
    p.scores = p.scratch + floats;
    p.score_rows = imin(all_rows, TREE_ROWS);
    floats += units * p.score_rows * p.score_keys;
  }
  *scratch_needed = floats * int64_t(sizeof(float));
  if (!p.scratch || scratch_bytes < *scratch_needed) return INTRA_NEED_SCRATCH;
  const int smem = tree_smem_bytes(p.mask ? (p.mask_sn ? p.n : 1) : 0);
  cudaError_t e = all_rows <= TREE_ROWS / 2 ? launch_early(tree_mma_kernel<ACCUMULATE, true>, dim3(unsigned(grid)), TREE_THREADS, smem, stream, p)
                                            : launch_early(tree_mma_kernel<ACCUMULATE, false>, dim3(unsigned(grid)), TREE_THREADS, smem, stream, p);
  if (!ACCUMULATE && !p.lengths && tree_whole(uint32_t(units), uint32_t(blocks), ceil_div(p.S, TREE_BLOCK), grid, p.split_cost))
    return e == cudaSuccess ? INTRA_OK : cuda_fail(e);             // nothing to join
  if (e == cudaSuccess)
    e = ACCUMULATE ? launch_early(tree_weights_kernel, dim3(unsigned(imin(ceil_div(p.S, TREE_WEIGHT_KEYS), ceil_div(st.sm_count * TREE_WEIGHT_CTAS_PER_SM, p.B * p.Hkv))) + 1, unsigned(p.B * p.Hkv)),
                                  TREE_WEIGHT_THREADS, 0, stream, p, uint32_t(grid))
                   : launch_early(tree_merge_kernel, dim3(unsigned((rows + TREE_MERGE_WARPS - 1) / TREE_MERGE_WARPS)), 32 * TREE_MERGE_WARPS, 0, stream, p, uint32_t(grid));
  return e == cudaSuccess ? INTRA_OK : cuda_fail(e);
}

bool cache_map(const __nv_bfloat16* ptr, const TensorView& v, int S, int Hkv, int B, CUtensorMap* map) {
  const cuuint64_t dims[5] = {HEAD_DIM, cuuint64_t(S), 1, cuuint64_t(Hkv), cuuint64_t(B)};
  const int64_t row = S > 1 ? v.ss : HEAD_DIM, head = Hkv > 1 ? v.sh : HEAD_DIM, batch = B > 1 ? v.sb : HEAD_DIM;
  if (row <= 0 || head <= 0 || batch <= 0) return false;
  const cuuint64_t strides[4] = {cuuint64_t(row) * 2, cuuint64_t(row) * 2, cuuint64_t(head) * 2, cuuint64_t(batch) * 2};
  const cuuint32_t box[5] = {64, TILE_N, 1, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
  return encode_map(map, ptr, 5, dims, strides, box, ones);
}

template <bool PAIR>
int launch_tree_umma(const TreeParams& t, const ServingState& st, int64_t scratch_bytes, int64_t* scratch_needed, cudaStream_t stream) {
  TreeUmmaParams p = {};
  p.t = t;
  const int B = t.B;
  p.t.row_groups = ceil_div(t.n * (t.H / t.Hkv), UMMA_ROWS<PAIR>);
  p.by_rep = fast_div(t.H / t.Hkv);
  const int64_t tiles = int64_t(B) * t.Hkv * p.t.row_groups * ceil_div(t.S, TILE_N);       // at most
  const int64_t parts = (tiles + UMMA_MIN_TILES - 1) / UMMA_MIN_TILES;
  const int64_t rows = int64_t(B) * t.n * t.H;
  const int64_t places = tiles + int64_t(B) * t.Hkv * p.t.row_groups * UMMA_UNIT_COST;
  const int row_blocks = ceil_div(imin(t.n * (t.H / t.Hkv), UMMA_ROWS<PAIR>), 32);
  const bool split = int64_t(B) * t.Hkv * p.t.row_groups * UMMA_MERGE_FEW < st.sm_count;      // many parts a unit
  const int64_t merge_ctas = int64_t(B) * t.Hkv * p.t.row_groups * row_blocks * (split ? UMMA_MERGE_CTAS<4, 2> : UMMA_MERGE_CTAS<8, 1>);
  if (places + st.sm_count > 0x7fffffffLL || rows > 0x7fffffffLL || merge_ctas > 0x7fffffffLL) return INTRA_ERR_UNSUPPORTED;
  const int64_t units = int64_t(B) * t.Hkv * p.t.row_groups, ctas = parts > units ? parts : units;
  const int grid = ctas < st.sm_count ? int(ctas) : st.sm_count;
  p.t.unit_cost = UMMA_UNIT_COST;
  p.t.split_cost = umma_split_cost(imin(t.n * (t.H / t.Hkv), UMMA_ROWS<PAIR>), !t.lengths && !t.mask);
  p.t.min_tiles = UMMA_MIN_TILES;
  *scratch_needed = grid * 2 * UMMA_PARTIAL<PAIR> * int64_t(sizeof(float));
  if (t.mask) {                   // behind the partial results: the mask's bits, those of any token, the tiles
    char* const at = reinterpret_cast<char*>(t.scratch) + *scratch_needed;
    p.t.bits_tokens = t.mask_sn ? t.n : 1;
    p.t.bits_words = ceil_div(t.S, TILE_N) * (TILE_N / 32);
    p.t.live_words = ceil_div(ceil_div(t.S, TILE_N), 64);
    const int64_t row = int64_t(p.t.bits_words) * 4;
    p.t.bits = reinterpret_cast<uint32_t*>(at);
    p.t.any = reinterpret_cast<uint32_t*>(at + row * B * p.t.bits_tokens);
    p.t.live = reinterpret_cast<uint8_t*>(at + row * B * (p.t.bits_tokens + 1));
    *scratch_needed += row * B * (p.t.bits_tokens + 1) + int64_t(p.t.live_words) * 8 * B;
    if (B > 65535) return INTRA_ERR_UNSUPPORTED;                   // grid.y of the bits
  }
  if (!t.scratch || scratch_bytes < *scratch_needed) return INTRA_NEED_SCRATCH;
  p.use_tma = cache_map(t.k, t.ks, t.S, t.Hkv, B, &p.maps[0]) && cache_map(t.v, t.vs, t.S, t.Hkv, B, &p.maps[1]);
  p.early = grid < st.sm_count;
  p.status = st.status_word;
  cudaError_t e = cudaSuccess;
  if (t.mask) e = launch_early(tree_mask_kernel, dim3(unsigned(ceil_div(p.t.bits_words, 32)), unsigned(B)), 32 * TREE_MASK_ROWS, 0, stream, p.t);
  if (e == cudaSuccess)
    e = t.mask ? launch_early(tree_umma_kernel<PAIR, true>, dim3(unsigned(grid)), UMMA_THREADS, UMMA_SMEM_BYTES<PAIR>, stream, p)
               : launch_early(tree_umma_kernel<PAIR, false>, dim3(unsigned(grid)), UMMA_THREADS, UMMA_SMEM_BYTES<PAIR>, stream, p);
  // Nothing to join where all sequences are alike and their units are dealt whole.
  if (!t.lengths && !t.mask && tree_whole(uint32_t(units), uint32_t(tiles), ceil_div(t.S, TILE_N), grid, p.t.split_cost))
    return e == cudaSuccess ? INTRA_OK : cuda_fail(e);
  if (e == cudaSuccess)
    e = launch_early(split ? tree_umma_merge_kernel<PAIR, 4, 2> : tree_umma_merge_kernel<PAIR, 8, 1>, dim3(unsigned(merge_ctas)),
                     32 * UMMA_MERGE_WARPS, 0, stream, p, uint32_t(grid), row_blocks);
  return e == cudaSuccess ? INTRA_OK : cuda_fail(e);
}

}  // namespace

cudaError_t intra::serving_status_word(int** word) {
  void* ptr = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&ptr, g_serving_status);
  *word = static_cast<int*>(ptr);
  return e;
}

extern "C" {

int intra_b200_tree_attn(const void* q, const void* k, const void* v, const int* parents, const int* lengths, const void* mask,
                         void* out, void* scratch, int64_t scratch_bytes, int64_t* scratch_needed, int B, int S, int H, int Hkv,
                         int n, const int64_t q_strides[3], const int64_t k_strides[3], const int64_t v_strides[3],
                         int64_t parents_batch_stride, int all_own, const int64_t mask_strides[3], float softmax_scale,
                         int device, void* cuda_stream) {
  if (!q || !k || !v || !out || !scratch_needed || !q_strides || !k_strides || !v_strides || (mask && !mask_strides) || B <= 0 ||
      S <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || n <= 0 || n > S || !(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return INTRA_ERR_BAD_ARG;
  if (n > TREE_MAX_TOKENS) return INTRA_ERR_UNSUPPORTED;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(scratch) || !aligned4(parents) ||
      !aligned4(lengths) || !rows_aligned(q_strides) || !rows_aligned(k_strides) || !rows_aligned(v_strides))
    return INTRA_ERR_ALIGNMENT;
  if (device < 0 || device >= MAX_DEVICES) return INTRA_ERR_BAD_ARG;
  DeviceGuard guard(device);
  const ServingState* st;
  const int rc = serving_device(device, guard, &st);
  if (rc != INTRA_OK) return rc;
  TreeParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.parents = parents;
  p.lengths = lengths;
  p.mask = static_cast<const uint8_t*>(mask);
  p.o = static_cast<__nv_bfloat16*>(out);
  p.scratch = static_cast<float*>(scratch);
  p.q_sb = q_strides[0]; p.q_sn = q_strides[1]; p.q_sh = q_strides[2];
  p.ks = view_of(k_strides);
  p.vs = view_of(v_strides);
  p.parents_sb = parents_batch_stride;
  p.all_own = all_own != 0;
  if (mask) {
    p.mask_sb = mask_strides[0]; p.mask_sn = mask_strides[1]; p.mask_ss = mask_strides[2];
    p.mask_vec = p.mask_ss == 1 && aligned16(mask) && ((p.mask_sb | p.mask_sn) & 15) == 0;
  }
  p.S = S; p.H = H; p.Hkv = Hkv; p.n = n; p.B = B;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  // By rows of a KV head. 12 and 16 rows on the kernel for few / for more, us: 16 sequences of 4,096 keys 52.8 / 60.5, of 1,000 23.1 / 20.2,
  // one of 30,000 40.7 / 39.6, of 3,001 16.0 / 15.0; with a mask or lengths the first has no kernel before it. 96 and 128 rows as two streams of key tiles /
  // in the form for two tiles of rows: 56.6 and 58.9 / 58.4 and 59.9, one of 30,000 40.9 and 42.3 / 41.2 and 41.0, and more
  // of the probabilities' bits.
  if (n * (H / Hkv) > 128) return launch_tree_umma<true>(p, *st, scratch_bytes, scratch_needed, stream);
  if (n * (H / Hkv) > TREE_ROWS) return launch_tree_umma<false>(p, *st, scratch_bytes, scratch_needed, stream);
  return launch_tree_mma<false>(p, *st, scratch_bytes, scratch_needed, stream);
}

int intra_b200_decode_accumulate(const void* q, const void* k, const void* v, const void* mask, const int* lengths, void* out,
                                 float* weights, void* scratch, int64_t scratch_bytes, int64_t* scratch_needed, int B, int S,
                                 int H, int Hkv, const int64_t q_strides[3], const int64_t k_strides[3],
                                 const int64_t v_strides[3], const int64_t mask_strides[2], int64_t weights_batch_stride,
                                 int64_t weights_head_stride, float softmax_scale, int device, void* cuda_stream) {
  if (!q || !k || !v || !out || !weights || !scratch_needed || !q_strides || !k_strides || !v_strides || (mask && !mask_strides) ||
      B <= 0 || S <= 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || !(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return INTRA_ERR_BAD_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(scratch) || !rows_aligned(q_strides) ||
      !rows_aligned(k_strides) || !rows_aligned(v_strides) || !aligned4(weights) || !aligned4(lengths))
    return INTRA_ERR_ALIGNMENT;
  if ((B > 1 && weights_batch_stride <= 0) || (Hkv > 1 && weights_head_stride <= 0)) return INTRA_ERR_BAD_ARG;
  if (device < 0 || device >= MAX_DEVICES) return INTRA_ERR_BAD_ARG;
  DeviceGuard guard(device);
  const ServingState* st;
  const int rc = serving_device(device, guard, &st);
  if (rc != INTRA_OK) return rc;
  TreeParams p = {};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.lengths = lengths;
  p.mask = static_cast<const uint8_t*>(mask);
  p.o = static_cast<__nv_bfloat16*>(out);
  p.weights = weights;
  p.weights_sb = weights_batch_stride; p.weights_sh = weights_head_stride;
  p.weights_vec = aligned16(weights) && ((p.weights_sb | p.weights_sh) & 3) == 0;
  p.scratch = static_cast<float*>(scratch);
  p.q_sb = q_strides[0]; p.q_sn = q_strides[1]; p.q_sh = q_strides[2];
  p.ks = view_of(k_strides);
  p.vs = view_of(v_strides);
  if (mask) {
    p.mask_sb = mask_strides[0]; p.mask_ss = mask_strides[1];
    p.mask_vec = p.mask_ss == 1 && aligned16(mask) && (p.mask_sb & 15) == 0;
  }
  p.S = S; p.H = H; p.Hkv = Hkv; p.n = 1; p.B = B;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  return launch_tree_mma<true>(p, *st, scratch_bytes, scratch_needed, static_cast<cudaStream_t>(cuda_stream));
}

int intra_b200_verify_drafts(const void* tokens, int tokens_int64, const void* target, const void* draft, int prob_type,
                             const float* uniform, const int* parents, int* accepted, int* path, int64_t* out_tokens, int B, int n,
                             int V, const int64_t target_strides[2], const int64_t draft_strides[2], int64_t tokens_batch_stride,
                             int64_t uniform_batch_stride, int64_t parents_batch_stride, int device, void* cuda_stream) {
  if (!tokens || !target || !uniform || !accepted || !path || !out_tokens || !target_strides || (draft && !draft_strides) ||
      B <= 0 || n <= 0 || V <= 0 || prob_type < 0 || prob_type > 2)
    return INTRA_ERR_BAD_ARG;
  if (n > VERIFY_MAX_TOKENS || V > VERIFY_MAX_VOCABULARY || B > 0x7fffffff / VERIFY_MAX_CLUSTER) return INTRA_ERR_UNSUPPORTED;
  const uintptr_t size = prob_type == INTRA_PROB_F32 ? 4 : 2, token_size = tokens_int64 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(target) % size || reinterpret_cast<uintptr_t>(draft) % size || !aligned4(uniform) ||
      !aligned4(parents) || !aligned4(accepted) || !aligned4(path) || reinterpret_cast<uintptr_t>(out_tokens) % 8 ||
      reinterpret_cast<uintptr_t>(tokens) % token_size)
    return INTRA_ERR_ALIGNMENT;
  if (device < 0 || device >= MAX_DEVICES) return INTRA_ERR_BAD_ARG;
  DeviceGuard guard(device);
  const ServingState* st;
  const int rc = serving_device(device, guard, &st);
  if (rc != INTRA_OK) return rc;
  VerifyParams p = {};
  p.tokens = tokens; p.tokens_wide = tokens_int64 != 0;
  p.target = target; p.draft = draft; p.uniform = uniform; p.parents = parents;
  p.accepted = accepted; p.path = path; p.out_tokens = reinterpret_cast<long long*>(out_tokens);
  p.target_sb = target_strides[0]; p.target_sn = target_strides[1];
  if (draft) { p.draft_sb = draft_strides[0]; p.draft_sn = draft_strides[1]; }
  p.tokens_sb = tokens_batch_stride; p.uniform_sb = uniform_batch_stride; p.parents_sb = parents_batch_stride;
  p.n = n; p.V = V;
  // CTAs of a sequence's cluster: as many as fit the GPU at once (two CTAs an SM) and have a few thousand tokens each. Measured with
  // 1 / 2 / 4 / 8, us, fp32 with draft probabilities, chains of 9 nodes: 1 x 50257 tokens 18.6 / 13.4 / 10.4 / 9.1, 32 x 128257 39.9 / 24.3 /
  // 17.4 / 17.3, 64 x 50257 21.4 / 16.1 / 16.6 / 24.5, 150 x 30000 21.2 / 22.7 / 28.4 / 47.0, 1 x 4000 7.9 / 7.6 / 7.3 / 7.4; trees of
  // 26, whose slowest sequence takes several passes: 32 x 128257 114 / 65 / 41 / 33, 64 x 50257 58 / 37 / 32 / 41, 150 x 30000 41 / 39 / 40 / 61.
  int c = 1;
  while (c < VERIFY_MAX_CLUSTER && int64_t(B) * 2 * c <= 2 * st->sm_count && V >= 2048 * c) c *= 2;
  p.cluster = c;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e;
  if (prob_type == INTRA_PROB_F32) e = launch_cluster(verify_kernel<float>, B, c, VERIFY_THREADS, VERIFY_SMEM_BYTES, stream, p);
  else if (prob_type == INTRA_PROB_BF16) e = launch_cluster(verify_kernel<__nv_bfloat16>, B, c, VERIFY_THREADS, VERIFY_SMEM_BYTES, stream, p);
  else e = launch_cluster(verify_kernel<__half>, B, c, VERIFY_THREADS, VERIFY_SMEM_BYTES, stream, p);
  return e == cudaSuccess ? INTRA_OK : cuda_fail(e);
}

int intra_b200_keep_drafts(void* const* caches, const int64_t* strides, int strides_step, int n_caches, const int* lengths,
                           const int* path, int64_t path_batch_stride, int B, int S, int Hkv, int n, int device, void* cuda_stream) {
  if (!caches || !strides || (strides_step != 0 && strides_step != 3) || !lengths || !path || n_caches <= 0 || B <= 0 || S <= 0 || Hkv <= 0 || n <= 0 || n > S)
    return INTRA_ERR_BAD_ARG;
  if (n > KEEP_MAX_TOKENS || int64_t(B) * Hkv > 0x7fffffffLL) return INTRA_ERR_UNSUPPORTED;
  if (!aligned4(lengths) || !aligned4(path)) return INTRA_ERR_ALIGNMENT;
  for (int i = 0; i < n_caches; ++i) {
    if (!caches[i]) return INTRA_ERR_BAD_ARG;
    const int64_t* s = strides + strides_step * i;
    if (s[0] <= 0 || s[1] <= 0 || s[2] <= 0) return INTRA_ERR_BAD_ARG;       // rows that share memory cannot be moved apart
    if (!aligned16(caches[i]) || !rows_aligned(s)) return INTRA_ERR_ALIGNMENT;
  }
  if (device < 0 || device >= MAX_DEVICES) return INTRA_ERR_BAD_ARG;
  DeviceGuard guard(device);
  const ServingState* st;
  const int rc = serving_device(device, guard, &st);
  if (rc != INTRA_OK) return rc;
  KeepParams p;
  p.lengths = lengths; p.path = path; p.path_sb = path_batch_stride;
  p.S = S; p.Hkv = Hkv; p.n = n;
  for (int first = 0; first < n_caches; first += KEEP_TENSORS) {
    const int count = imin(n_caches - first, KEEP_TENSORS);
    for (int i = 0; i < count; ++i) {
      p.cache[i] = static_cast<__nv_bfloat16*>(caches[first + i]);
      p.s[i] = view_of(strides + strides_step * (first + i));
    }
    keep_rows_kernel<<<dim3(unsigned(B * Hkv), unsigned(count)), KEEP_THREADS, 0, static_cast<cudaStream_t>(cuda_stream)>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_fail(e);
  }
  return INTRA_OK;
}

int intra_b200_evict(const void* k, const void* v, const float* weights, const int* lengths, void* k_out, void* v_out,
                     float* weights_out, int* kept, int B, int S, int Hkv, int keep, int recent, const int64_t k_strides[3],
                     const int64_t v_strides[3], const int64_t weights_strides[2], const int64_t k_out_strides[3],
                     const int64_t v_out_strides[3], const int64_t weights_out_strides[2], int device, void* cuda_stream) {
  if (!k || !v || !weights || !k_out || !v_out || !weights_out || !kept || !k_strides || !v_strides || !weights_strides ||
      !k_out_strides || !v_out_strides || !weights_out_strides || B <= 0 || S <= 0 || Hkv <= 0 || keep <= 0 || recent < 0 ||
      recent > keep)
    return INTRA_ERR_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (k_out_strides[i] <= 0 || v_out_strides[i] <= 0) return INTRA_ERR_BAD_ARG;
  if (weights_out_strides[0] <= 0 || weights_out_strides[1] <= 0) return INTRA_ERR_BAD_ARG;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_out) || !aligned16(v_out) || !aligned4(weights) || !aligned4(weights_out) ||
      !aligned4(lengths) || !aligned4(kept) || !rows_aligned(k_strides) || !rows_aligned(v_strides) ||
      !rows_aligned(k_out_strides) || !rows_aligned(v_out_strides))
    return INTRA_ERR_ALIGNMENT;
  if (device < 0 || device >= MAX_DEVICES) return INTRA_ERR_BAD_ARG;
  const int64_t units = int64_t(B) * Hkv;
  const int64_t copies = units * ceil_div(keep, EVICT_COPY_THREADS / 16 * EVICT_ROWS);
  if (units * EVICT_MAX_CLUSTER > 0x7fffffffLL || copies > 0x7fffffffLL || int64_t(S) + EVICT_THREADS * EVICT_MAX_CLUSTER > 0x7fffffffLL ||
      int64_t(keep) + EVICT_THREADS * EVICT_MAX_CLUSTER > 0x7fffffffLL)
    return INTRA_ERR_UNSUPPORTED;
  DeviceGuard guard(device);
  const ServingState* st;
  const int rc = serving_device(device, guard, &st);
  if (rc != INTRA_OK) return rc;
  EvictParams p = {};
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.weights = weights; p.lengths = lengths;
  p.k2 = static_cast<__nv_bfloat16*>(k_out);
  p.v2 = static_cast<__nv_bfloat16*>(v_out);
  p.weights2 = weights_out; p.kept = kept;
  p.ks = view_of(k_strides); p.vs = view_of(v_strides); p.k2s = view_of(k_out_strides); p.v2s = view_of(v_out_strides);
  p.weights_sb = weights_strides[0]; p.weights_sh = weights_strides[1];
  p.weights2_sb = weights_out_strides[0]; p.weights2_sh = weights_out_strides[1];
  p.S = S; p.Hkv = Hkv; p.keep = keep; p.recent = recent;
  // CTAs of a head's cluster: as many as fit the GPU at once (two an SM) and have a few thousand weights each; more where a part
  // would not fit shared memory. Measured with 1 / 2 / 4 / 8, us: 8 heads of 4,096 rows 10.0 / 10.8 / 12.5 / 15.5, of 65,536 - / 28.0 /
  // 21.3 / 20.3, 32 heads of 16,384 - / 20.7 / 20.6 / 34.5, 128 heads of 16,384 - / 59.3 / 73.1 / 139.5.
  int c = 1;
  while (c < EVICT_MAX_CLUSTER && units * 2 * c <= 2 * st->sm_count && S > 6144 * c) c *= 2;
  while (c < EVICT_MAX_CLUSTER && ceil_div(S, c) > EVICT_SMEM_KEYS) c *= 2;
  p.cluster = c;
  const int part = (ceil_div(S, c) + 3) & ~3;
  cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
  cudaError_t e = part <= EVICT_SMEM_KEYS ? launch_cluster(evict_select_kernel<true>, units, c, EVICT_THREADS, part * 4, stream, p, 1)
                                          : launch_cluster(evict_select_kernel<false>, units, c, EVICT_THREADS, 0, stream, p, 1);
  if (e == cudaSuccess) e = launch_early(evict_copy_kernel, dim3(unsigned(copies)), EVICT_COPY_THREADS, 0, stream, p);
  return e == cudaSuccess ? INTRA_OK : cuda_fail(e);
}

}  // extern "C"
