// Eviction from an uncompressed paged cache by accumulated attention weight.
//
// Per request and KV head the `budget` tokens of most worth stay: those whose position is below `sink` or among the
// last `recent` that were seen, whatever their weight, then by falling weight (ties: the lowest place).  The kept tokens
// behind the budget move into the places that fall free in front of it, both in rising order; the others stay where
// they are.  So a step that evicts a few tokens of many moves few rows, no row is both read and written, and attention,
// for which the order of tokens in the cache means nothing, goes on as before.
//
// evict_select_kernel finds the worth of the last token that stays by a radix select over 32-bit keys (four digits of 8
// bits, histograms in shared memory): one cluster per row (request, KV head), each CTA with a slice of it, the
// histograms added over distributed shared memory.  It writes the lists of free places and of tokens that move.
// Its passes depend on one another, which is what bounds it: 15 us for 256 rows of 2304 tokens, 24 for 16 of 32768.
// evict_move_kernel moves the rows of K and V: 4 D elements read and written per token, which is what bounds it (67 MB 10 us).
// Where many short rows are selected, the selecting CTAs move them instead, and one row's moves overlap the next's passes.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"

namespace cg = cooperative_groups;

namespace inq {

constexpr int kEvThreads = 512, kEvBins = 256, kEvPasses = 4, kEvMaxCluster = 8;

struct EvictParams {
  void *k, *v;
  long long k_sp, k_sh, k_st, v_sp, v_sh, v_st;
  const int *table, *lengths, *seen, *positions;
  const float* weights;
  int *out_positions, *out_lengths;
  float* out_weights;
  long long table_stride, w_sb, w_sh, p_sb, p_sh, ow_sb, ow_sh, op_sb, op_sh;
  long long pages, capacity;
  int requests, kv_heads, page_tokens, page_shift, budget, sink, recent, row_bytes;
  long long list_columns;
  int moves_here;
  int* lists;          // per row: count, then up to list_columns free places, then as many tokens that move
  int* status;
};

// Rises with the worth of a token; a NaN is worth less than anything.
__device__ __forceinline__ unsigned worth(float w) {
  if (w != w) return 0u;
  const unsigned u = __float_as_uint(w + 0.f);          // -0 counts as 0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Sum over the warps in front of this one, and over all of them, of a number that a warp's lanes agree on.
__device__ __forceinline__ int warps_before(int mine, int& all, int* scratch /* one per warp */) {
  const int warp = threadIdx.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[warp] = mine;
  __syncthreads();
  int before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < kEvThreads / 32; ++w) {
    const int n = scratch[w];
    if (w < warp) before += n;
    all += n;
  }
  return before;
}

// Moves tokens i0 .. of a row's lists, eight at once, by a warp that asks for all of them before it writes the first: half of
// its lanes the key rows, the others the value rows, 16 bytes each.
constexpr int kEvMoveEach = 8;
__device__ __forceinline__ void move_tokens(const EvictParams& P, int b, int h, const int* list, int i0, int count) {
  const int lane = threadIdx.x & 31;
  // lane 2 i (+ 1) finds the page and offset of where token i goes (comes from), and moves its weight and position
  const int i = i0 + (lane >> 1);
  const bool some = lane < 2 * kEvMoveEach && i < count;
  const int j = some ? __ldcg(list + 1 + (lane & 1 ? P.list_columns : 0) + i) : 0;
  const int column = P.page_shift >= 0 ? j >> P.page_shift : j / P.page_tokens, o = j - column * P.page_tokens;
  int page = some ? __ldg(P.table + b * P.table_stride + column) : -1;
  if (some && (page < 0 || page >= P.pages)) {
    atomicOr(P.status, INQ_STATUS_BAD_INDEX);
    page = -1;
  }
  const int place = __shfl_xor_sync(0xffffffffu, j, 1);
  if (some && (lane & 1)) {
    P.out_weights[b * P.ow_sb + h * P.ow_sh + place] = P.weights[b * P.w_sb + h * P.w_sh + j];
    P.out_positions[b * P.op_sb + h * P.op_sh + place] = P.positions[b * P.p_sb + h * P.p_sh + j];
  }
  const bool key = lane < 16;
  const long long sp = key ? P.k_sp : P.v_sp, st = key ? P.k_st : P.v_st;
  char* const base = (char*)(key ? P.k : P.v) + 2 * h * (key ? P.k_sh : P.v_sh) + (lane & 15) * 16;
  const bool mine = (lane & 15) * 16 < P.row_bytes;
  uint4 rows[kEvMoveEach];
#pragma unroll
  for (int n = 0; n < kEvMoveEach; ++n) {
    const int to = __shfl_sync(0xffffffffu, page, 2 * n), from = __shfl_sync(0xffffffffu, page, 2 * n + 1), from_o = __shfl_sync(0xffffffffu, o, 2 * n + 1);
    if (to >= 0 && from >= 0 && mine) rows[n] = __ldcs((const uint4*)(base + 2 * (from * sp + from_o * st)));
  }
#pragma unroll
  for (int n = 0; n < kEvMoveEach; ++n) {
    const int to = __shfl_sync(0xffffffffu, page, 2 * n), from = __shfl_sync(0xffffffffu, page, 2 * n + 1), to_o = __shfl_sync(0xffffffffu, o, 2 * n);
    if (to >= 0 && from >= 0 && mine) *(uint4*)(base + 2 * (to * sp + to_o * st)) = rows[n];
  }
}

// KEYS: tokens per thread whose keys stay in registers over all passes; a slice of more is read anew for each.
template <int KEYS>
__global__ void __launch_bounds__(kEvThreads, KEYS <= 5 ? 2 : 1) evict_select_kernel(const EvictParams P) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const int row = blockIdx.x / ctas, b = row / P.kv_heads, h = row % P.kv_heads, tid = threadIdx.x;
  __shared__ int histograms[kEvPasses][kEvBins];      // one per pass: none is cleared while others read it
  __shared__ int shared_counts[2];                    // this CTA's free places and moving tokens
  __shared__ int scratch[kEvThreads / 32], chosen[kEvPasses][3];
  const int warp = tid >> 5, lane = tid & 31;
  follow_stream();
  allow_next();
  const long long asked = P.lengths[b];
  const int length = (int)min(max(asked, 0LL), P.capacity), budget = P.budget;
  if (asked > P.capacity && row % P.kv_heads == 0 && me == 0 && tid == 0) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
  const int left = min(length, budget);
  if (P.moves_here && h == 0 && me == 0 && tid == 0) P.out_lengths[b] = (int)min(min(asked, (long long)budget), P.capacity);
  const float* const w = P.weights + b * P.w_sb + h * P.w_sh;
  const int* const pos = P.positions + b * P.p_sb + h * P.p_sh;
  float* const out_w = P.out_weights + b * P.ow_sb + h * P.ow_sh;
  int* const out_p = P.out_positions + b * P.op_sb + h * P.op_sh;
  int* const list = P.lists + row * (2 * P.list_columns + 1);
  // places that no token fills
  for (int j = left + me * kEvThreads + tid; j < budget; j += ctas * kEvThreads) {
    out_w[j] = 0.f;
    out_p[j] = -1;
  }
  if (length <= budget) {       // the same in every CTA of the cluster
    for (int j = me * kEvThreads + tid; j < left; j += ctas * kEvThreads) {
      out_w[j] = w[j];
      out_p[j] = pos[j];
    }
    if (me == 0 && tid == 0) list[0] = 0;
    return;
  }
  const long long safe_from = (long long)P.seen[b] - P.recent;
  const int slice = (length + ctas - 1) / ctas, lo = min(me * slice, length), hi = min(lo + slice, length);
  constexpr int kGroup = kEvThreads * KEYS;
  const int groups = (hi - lo + kGroup - 1) / kGroup;
  // A warp owns 32 KEYS neighbouring tokens of a group, lane l every 32nd of them from the l-th: loads and stores of a
  // warp are whole lines, and the order of tokens is that of (i, lane), which ballots count.
  unsigned keys[KEYS];          // 0 behind the slice, where no token is looked for
  int p[KEYS];
  float x[KEYS];
  auto first_token = [&](int g) { return lo + g * kGroup + warp * (32 * KEYS) + lane; };
  auto load = [&](int g) {
    const int j0 = first_token(g);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      p[i] = j0 + 32 * i < hi ? __ldg(pos + j0 + 32 * i) : 0;
      x[i] = j0 + 32 * i < hi ? __ldg(w + j0 + 32 * i) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < KEYS; ++i) keys[i] = j0 + 32 * i >= hi ? 0u : p[i] < P.sink || p[i] >= safe_from ? 0xffffffffu : worth(x[i]);
  };
  if (groups <= 1) load(0);
  for (int i = tid; i < kEvPasses * kEvBins; i += kEvThreads) histograms[0][i] = 0;
  __syncthreads();

  // ---- the key of the last token that stays: `want` tokens of those that begin with `prefix` are still to be found
  unsigned prefix = 0;
  int want = budget;
#pragma unroll 1
  for (int pass = 0; pass < kEvPasses; ++pass) {
    const int shift = 24 - 8 * pass;
    int* const histogram = histograms[pass];
#pragma unroll 1
    for (int g = 0; g < groups; ++g) {
      if (groups > 1) load(g);
      const int j0 = first_token(g);
#pragma unroll
      for (int i = 0; i < KEYS; ++i)
        if (j0 + 32 * i < hi && (pass == 0 || keys[i] >> (shift + 8) == prefix)) atomicAdd(histogram + ((keys[i] >> shift) & 255u), 1);
    }
    cluster.sync();
    // every CTA finds the digit for itself: a thread adds a bin over the cluster, the highest first
    int mine = 0, all;
    if (tid < kEvBins) {
#pragma unroll
      for (int c = 0; c < kEvMaxCluster; ++c)
        if (c < ctas) mine += cluster.map_shared_rank(histogram, c)[kEvBins - 1 - tid];
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    const int before = sum - mine + warps_before(__shfl_sync(0xffffffffu, sum, 31), all, scratch);
    if (before < want && before + mine >= want) {
      chosen[pass][0] = kEvBins - 1 - tid;
      chosen[pass][1] = want - before;
      chosen[pass][2] = mine == want - before;
    }
    __syncthreads();
    prefix = prefix << 8 | (unsigned)chosen[pass][0];
    want = chosen[pass][1];
    if (chosen[pass][2]) {
      // all tokens that begin like this stay, as they mostly do after three digits: no order among them is needed
      prefix <<= shift;
      want = 0x7fffffff;
      break;
    }
  }
  // tokens above the threshold stay, and the first `want` of those at it
  int ties_before = 0;
  for (int c = 0; c < me; ++c) ties_before += cluster.map_shared_rank(histograms[kEvPasses - 1], c)[prefix & 255u];

  // ---- which tokens stay; the free places and moving tokens, counted over the slice and then listed
  const unsigned behind = (1u << lane) - 1u;        // lanes in front of this one
  unsigned kept = 0;
  int ties = ties_before, holes = 0, moves = 0, mine_before = 0;        // of the groups in front of the one in work, and inside it
  int group_holes = 0, group_moves = 0;
  auto decide = [&](int g) {
    const int j0 = first_token(g);
    int equal = 0, all_equal, all_packed;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) equal += __popc(__ballot_sync(0xffffffffu, j0 + 32 * i < hi && keys[i] == prefix));
    int rank = ties + warps_before(equal, all_equal, scratch), mine_holes = 0, mine_moves = 0;
    ties += all_equal;
    kept = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = j0 + 32 * i;
      const bool tie = j < hi && keys[i] == prefix;
      const unsigned tied = __ballot_sync(0xffffffffu, tie);
      const bool stays = j < hi && (keys[i] > prefix || (tie && rank + __popc(tied & behind) < want));
      rank += __popc(tied);
      kept |= (unsigned)stays << i;
      mine_holes += __popc(__ballot_sync(0xffffffffu, j < left && j < hi && !stays));
      mine_moves += __popc(__ballot_sync(0xffffffffu, j >= left && stays));
    }
    mine_before = warps_before(mine_holes | (mine_moves << 16), all_packed, scratch);
    group_holes = all_packed & 0xffff;
    group_moves = all_packed >> 16;
  };
  if (groups == 1) {
    decide(0);
  } else {
    for (int g = 0; g < groups; ++g) {
      load(g);
      decide(g);
      holes += group_holes;
      moves += group_moves;
    }
  }
  if (ctas > 1) {
    if (tid == 0) {
      shared_counts[0] = groups == 1 ? group_holes : holes;
      shared_counts[1] = groups == 1 ? group_moves : moves;
    }
    cluster.sync();
  }
  holes = moves = 0;
#pragma unroll
  for (int c = 0; c < kEvMaxCluster - 1; ++c) {
    if (c < me) {
      holes += cluster.map_shared_rank(shared_counts, c)[0];
      moves += cluster.map_shared_rank(shared_counts, c)[1];
    }
  }
  ties = ties_before;
#pragma unroll 1
  for (int g = 0; g < groups; ++g) {
    if (groups > 1) {
      load(g);
      decide(g);
    }
    const int j0 = first_token(g);
    int hole = holes + (mine_before & 0xffff), move = moves + (mine_before >> 16);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int j = j0 + 32 * i;
      const bool stays = (kept >> i) & 1u, free = j < left && j < hi && !stays, moving = j >= left && stays;
      const unsigned all_free = __ballot_sync(0xffffffffu, free), all_moving = __ballot_sync(0xffffffffu, moving);
      if (free) list[1 + hole + __popc(all_free & behind)] = j;
      if (moving) list[1 + P.list_columns + move + __popc(all_moving & behind)] = j;
      hole += __popc(all_free);
      move += __popc(all_moving);
      if (j < left && stays) {
        out_w[j] = x[i];
        out_p[j] = p[i];
      }
    }
    holes += group_holes;
    moves += group_moves;
  }
  if (me == ctas - 1 && tid == 0) list[0] = moves;
  cluster.sync();       // the counts of a CTA are read until here, and the lists of the cluster are complete
  if (!P.moves_here) return;
  const int count = __ldcg(list);
  for (int i0 = (me * (kEvThreads / 32) + warp) * kEvMoveEach; i0 < count; i0 += ctas * (kEvThreads / 32) * kEvMoveEach)
    move_tokens(P, b, h, list, i0, count);
}

constexpr int kEvMoveThreads = 256, kEvMoveTokens = kEvMoveThreads / 32 * kEvMoveEach;      // tokens of a block
__global__ void __launch_bounds__(kEvMoveThreads) evict_move_kernel(const EvictParams P) {
  follow_stream();
  const int row = blockIdx.x, b = row / P.kv_heads, h = row % P.kv_heads, warp = threadIdx.x >> 5;
  const int* const list = P.lists + row * (2 * P.list_columns + 1);
  if (blockIdx.y == 0 && h == 0 && threadIdx.x == 0) P.out_lengths[b] = (int)min((long long)min(P.lengths[b], P.budget), P.capacity);
  const int count = __ldcg(list), i0 = blockIdx.y * kEvMoveTokens + warp * kEvMoveEach;
  if (i0 < count) move_tokens(P, b, h, list, i0, count);
}

}  // namespace inq

using namespace inq;

extern "C" int64_t inq_evict_workspace_bytes(int32_t requests, int32_t kv_heads, int32_t budget, int64_t capacity) {
  return requests < 1 || kv_heads < 1 || budget < 1 || capacity < 1
             ? 0 : (int64_t)requests * kv_heads * (2 * std::min<int64_t>(budget, capacity) + 1) * (int64_t)sizeof(int);
}

extern "C" int inq_evict_tokens(const inq_evict_args_t* a, inq_stream_t stream_) {
  if (!a || !a->k || !a->v || !a->table || !a->lengths || !a->seen || !a->positions || !a->weights || !a->out_positions ||
      !a->out_lengths || !a->out_weights || !a->status)
    return INQ_ERR_ARGUMENT;
  if (a->requests < 1 || a->kv_heads < 1 || a->pages < 1 || a->page_tokens < 1 || a->table_columns < 1) return INQ_ERR_ARGUMENT;
  if (a->budget < 1 || a->sink < 0 || a->recent < 0 || (long long)a->sink + a->recent > a->budget) return INQ_ERR_ARGUMENT;
  if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) return INQ_ERR_UNSUPPORTED;
  if ((a->k_stride_p | a->k_stride_h | a->k_stride_t | a->v_stride_p | a->v_stride_h | a->v_stride_t) & 7) return INQ_ERR_ARGUMENT;
  if (((uintptr_t)a->k | (uintptr_t)a->v) & 15) return INQ_ERR_ARGUMENT;
  const long long capacity = (long long)a->table_columns * a->page_tokens, rows = (long long)a->requests * a->kv_heads;
  if (capacity > 0x3fffffLL || a->budget > 0x3fffffff || rows * kEvMaxCluster > 0x7fffffffLL) return INQ_ERR_CAPACITY;
  if (!a->workspace || a->workspace_bytes < inq_evict_workspace_bytes(a->requests, a->kv_heads, a->budget, capacity)) return INQ_ERR_CAPACITY;
  int device = 0, n_sm = 0;
  INQ_CUDA_CHECK(cudaGetDevice(&device));
  INQ_CUDA_CHECK(cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, device));
  EvictParams P = {};
  P.k = a->k; P.v = a->v;
  P.k_sp = a->k_stride_p; P.k_sh = a->k_stride_h; P.k_st = a->k_stride_t;
  P.v_sp = a->v_stride_p; P.v_sh = a->v_stride_h; P.v_st = a->v_stride_t;
  P.table = a->table; P.lengths = a->lengths; P.seen = a->seen; P.positions = a->positions; P.weights = a->weights;
  P.out_positions = a->out_positions; P.out_lengths = a->out_lengths; P.out_weights = a->out_weights;
  P.table_stride = a->table_stride; P.w_sb = a->w_stride_b; P.w_sh = a->w_stride_h; P.p_sb = a->p_stride_b; P.p_sh = a->p_stride_h;
  P.ow_sb = a->ow_stride_b; P.ow_sh = a->ow_stride_h; P.op_sb = a->op_stride_b; P.op_sh = a->op_stride_h;
  P.pages = a->pages; P.capacity = std::min<long long>(capacity, a->columns);
  P.requests = a->requests; P.kv_heads = a->kv_heads; P.page_tokens = a->page_tokens;
  P.page_shift = -1;
  for (int i = 0; i < 30; ++i)
    if (a->page_tokens == 1 << i) P.page_shift = i;
  P.list_columns = std::min<long long>(a->budget, capacity);
  P.budget = a->budget; P.sink = a->sink; P.recent = a->recent; P.row_bytes = 2 * a->head_dim;
  P.lists = (int*)a->workspace; P.status = a->status;
  // slices of a row: while they fill the SMs and hold 2048 tokens at least
  int ctas = 1;
  while (ctas < kEvMaxCluster && rows * ctas * 2 <= 2 * n_sm && P.capacity / (2 * ctas) >= 2048) ctas *= 2;
  const long long slice = (P.capacity + ctas - 1) / ctas;
  // As many tokens move as places fall free, at most, and as there are behind the budget.  Where the rows fill the SMs and two
  // CTAs fit on one, few moves are done at once, beside the selection of other rows (256 rows of 2304 tokens, 256 of them
  // evicted: 24.7 us in a graph against 26.8; 512 rows of 1024, a half evicted: 48.6 against 50.9).  Else they take a launch
  // of their own, over all SMs (256 rows of 4096, one CTA per SM: 46 us against 49.5; 16 of 32768 to 8192: 42.6 against 54).
  // Rows are as long here as the table and `columns` allow, since the lengths are on the device: 256 rows of 2304 tokens
  // take 48 us with a table of 32768.  Other heads may still read a length when one writes it, so that it is not written in place.
  const long long most = std::min<long long>(P.budget, std::max<long long>(P.capacity - P.budget, 1));
  P.moves_here = slice <= 5 * kEvThreads && rows * ctas > n_sm && most <= 4LL * ctas * (kEvThreads / 32) * kEvMoveEach && P.out_lengths != P.lengths;
  cudaStream_t stream = (cudaStream_t)stream_;
  {
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = ctas;
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * ctas));
    config.blockDim = dim3(kEvThreads);
    config.stream = stream;
    config.attrs = attrs;
    config.numAttrs = 2;
    // the keys of a slice in registers where 16 per thread do, in fewer where a power of two and some slack fit
    INQ_CUDA_CHECK(slice <= 5 * kEvThreads ? cudaLaunchKernelEx(&config, evict_select_kernel<5>, P)
                                           : slice <= 9 * kEvThreads ? cudaLaunchKernelEx(&config, evict_select_kernel<9>, P)
                                                                     : cudaLaunchKernelEx(&config, evict_select_kernel<16>, P));
  }
  if (!P.moves_here) INQ_CUDA_CHECK(launch_following(evict_move_kernel, dim3((unsigned)rows, (unsigned)((most + kEvMoveTokens - 1) / kEvMoveTokens)),
                                                     kEvMoveThreads, 0, stream, P));
  return INQ_OK;
}
