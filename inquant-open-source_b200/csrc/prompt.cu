// Prompts of several requests packed into one launch: causal attention with its log-sum-exp, and the
// attention weight that every key received.
//
// Sequence b owns query rows cu_q[b] .. cu_q[b + 1] and key rows cu_k[b] .. cu_k[b + 1] of token-major
// tensors; its last query sits at its last key, so query i sees the keys at positions <= i + keys - queries.
// The lengths are read on the device: no host copy of them exists, and a captured launch serves others.
//
// prompt_kernel.  o_i = sum_j p_ij v_j / l_i with p_ij = 2^(s_ij - m_i), one pass over the keys with a running
// reference maximum (csrc/prefill.cu describes the roles: softmax warps with one thread per query row, one
// warp that issues the contractions, one that issues the copies).  What this kernel has besides:
//   * CTAs are persistent: a warp deals items (256 query rows of one head) to the others, found by their rank in the
//     order of falling cost whatever the mix of lengths (find_item), and the copies and contractions of one item
//     follow those of the one before without a break;
//   * one more warp cleans the value tiles that hold rows some query must not see.  The contraction multiplies
//     such rows by probability zero, which is no help against infinities and NaN: rows behind the sequence (those
//     of its neighbour, or memory that nothing has written) are set to zero, non-finite values at the positions that
//     only later queries see are set to zero and put back, by position, into the rows that do see them.
// A step (two tiles, 128 keys) takes about 3700 cycles against 2048 of the tensor core and of the exponential unit alike:
// the chain S -> P -> S of a tile bounds it, and beyond 1.06 PFLOP/s the power cap.  Back to back, at the clock that the cap
// leaves, 8192 tokens of 28 heads take 450 to 463 us and 16 prompts of 16 to 2000 tokens of 32 heads 364 to 380 (in bursts too
// short for the cap 390 to 400 and 320 to 330); 301 tokens of 28 heads 12.5.
//
// prompt_weights_kernel.  w_j = sum over the group's heads and the last `window` queries of 2^(s_ij - lse_i).  The
// contraction is transposed, S^T = K Q^T: two threads own a KEY row and add over columns, so that no atomics order a
// sum.  4096 tokens of 28 heads 82 to 84 us, 54 of them exponentials; 8 requests of 900 to 16000 tokens of 32 heads, judged
// by their last 64 queries, 55 to 65 us (the clock), 24 of them memory.
#include <algorithm>

#include "attention.cuh"

namespace inq {

constexpr int kPrThreads = 384;              // 8 softmax warps, the MMA warp, the TMA warp, one that cleans value tiles, one that deals
constexpr int kPrSoftmaxWarps = 8;
constexpr int kPrLaunchRegs = 168, kPrIssueRegs = 72, kPrSoftmaxRegs = (3 * kPrLaunchRegs - kPrIssueRegs) / 2;
constexpr int kPrTile = 128;                 // rows per tile
constexpr int kPrRows = 2 * kPrTile;         // rows per item (tiles A and B)
constexpr int kPrSlab = kPrTile * 128;       // 128 rows x 128 bytes
constexpr float kPrNegBig = -3.0e38f;        // stands for the maximum of nothing: below every finite logit that matters
constexpr float kPrSlack = 8.f;              // the reference maximum may lag the true one by 2^8
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct CutItem;
struct PromptParams {
  void* out;
  float* lse;                       // attention: written, weights: read; [q_heads][lse_stride]
  float* weights;                   // [kv_heads][weights_stride]
  long long o_sh, o_st, lse_stride, weights_stride;
  const int *cu_q, *cu_k;
  int n_seq, q_rows, k_rows, q_heads, kv_heads;
  int window;                       // weights: queries per sequence that count, 0 = all
  int width;                        // weights: columns of a step per query head
  float* records;                   // partial results of cut items
  CutItem* cuts;                    // of attention, per CTA
  float scale_log2e;
  int* status;
};

// One sequence, with bounds that the tensors hold whatever cu_q and cu_k say.
struct Sequence {
  int q0, nq, k0, nk;
};
__device__ __forceinline__ Sequence load_sequence(const PromptParams& P, int b) {
  Sequence s;
  s.q0 = min(max(__ldg(P.cu_q + b), 0), P.q_rows);
  s.nq = max(min(__ldg(P.cu_q + b + 1), P.q_rows) - s.q0, 0);
  s.k0 = min(max(__ldg(P.cu_k + b), 0), P.k_rows);
  s.nk = max(min(__ldg(P.cu_k + b + 1), P.k_rows) - s.k0, 0);
  return s;
}
__device__ __forceinline__ bool bad_sequence(const PromptParams& P, int b) {
  const int q0 = P.cu_q[b], q1 = P.cu_q[b + 1], k0 = P.cu_k[b], k1 = P.cu_k[b + 1];
  return q0 < 0 || q1 < q0 || q1 > P.q_rows || k0 < 0 || k1 < k0 || k1 > P.k_rows;
}

// Items (256 query rows) of one sequence that cost at least c, cost being the tiles of 128 keys that the last row sees.
// Costs rise with the item's index, so that these are the last ones and their number a closed form.
__device__ __forceinline__ int items_at_least(const Sequence& s, int c) {
  const int n = (s.nq + kPrRows - 1) / kPrRows;
  if (c <= 0) return n;
  const int keys = (c - 1) * kPrTile;                       // more than these have to be visible
  if (s.nk <= keys) return 0;
  return n - min(max((keys - (s.nk - s.nq)) >> 8, 0), n);
}
// The item of rank `rank` in the order of falling cost (sequences in order among equals).  The whole warp takes
// part: a binary search over the cost, each lane counting the items of its sequences; the sequence and the item
// inside it follow from prefix sums.  32 sequences stay in registers, further ones are read again (from L1) in
// every turn.  Hundreds of sequences are dealt in their own order, without the search: it would take longer than
// their items do.  Returns the sequence, or -1 where there are fewer items.
constexpr int kPrSorted = 256;
__device__ __forceinline__ int find_item(const PromptParams& P, int rank, int max_cost, Sequence& seq, int& index) {
  const int lane = threadIdx.x & 31;
  Sequence mine = {0, 0, 0, 0};
  if (lane < P.n_seq) mine = load_sequence(P, lane);
  auto count = [&](int c) {
    int n = items_at_least(mine, c);
    for (int b = 32 + lane; b < P.n_seq; b += 32) n += items_at_least(load_sequence(P, b), c);
    return __reduce_add_sync(0xffffffffu, n);
  };
  if (rank >= count(0)) return -1;
  const bool sorted = P.n_seq <= kPrSorted;
  int lo = 0, hi = sorted ? max_cost + 1 : 1;      // count(lo) > rank >= count(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) > rank) lo = mid;
    else hi = mid;
  }
  int left = sorted ? rank - count(lo + 1) : rank;
  for (int b0 = 0; b0 < P.n_seq; b0 += 32) {
    const Sequence s = b0 == 0 ? mine : b0 + lane < P.n_seq ? load_sequence(P, b0 + lane) : Sequence{0, 0, 0, 0};
    const int ge = items_at_least(s, lo), equal = sorted ? ge - items_at_least(s, lo + 1) : ge;
    int before = equal;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, before > left);
    if (found) {
      const int who = __ffs(found) - 1;
      left -= __shfl_sync(0xffffffffu, before - equal, who);
      index = __shfl_sync(0xffffffffu, items_at_least(s, 0) - ge, who) + left;
      seq.q0 = __shfl_sync(0xffffffffu, s.q0, who);
      seq.nq = __shfl_sync(0xffffffffu, s.nq, who);
      seq.k0 = __shfl_sync(0xffffffffu, s.k0, who);
      seq.nk = __shfl_sync(0xffffffffu, s.nk, who);
      return b0 + who;
    }
    left -= __shfl_sync(0xffffffffu, before, 31);
  }
  return -1;
}

// How the items of a launch are dealt to its CTAs.  Ordinarily whole: in the order of falling cost, every other round through
// the CTAs backwards, so that they end at about the same time.  Where that leaves most SMs idle -- few items behind long
// histories -- the steps (tiles of 128 keys) of all items form one list (request, head, item) that is cut into equal
// ranges; what the ranges leave of a cut item is joined by a second launch.  The estimates, in steps: whole items
// max(dearest, mean + dearest / rounds), ranges mean + 6 (parts written, read and joined), and a tenth less.
constexpr int kPrCut = 6;
constexpr int kPrShortest = 12;      // steps of a range, where items have as many
// Item i of a sequence: query rows 256 i ..; it takes ceil(keys that its last row sees / 128) steps.
struct ItemSteps {
  int items, lag, last;        // lag: ceil((nk - nq) / 128); last: steps of the last item
  __device__ __forceinline__ explicit ItemSteps(const Sequence& s) {
    items = (s.nq + kPrRows - 1) / kPrRows;
    lag = (s.nk - s.nq + kPrTile - 1) >> 7;
    last = (s.nk + kPrTile - 1) / kPrTile;
  }
  __device__ __forceinline__ int cost(int i) const { return i + 1 < items ? max(2 * (i + 1) + lag, 0) : items > 0 ? last : 0; }
  __device__ __forceinline__ long long before(int i) const {
    // the sum of 2 (j + 1) + lag over j = 0 .. i - 1, as far as positive, where item i exists
    const long long first = min((long long)max(-lag >> 1, 0), (long long)i);
    return (long long)i * (i - 1) - first * (first - 1) + (i - first) * (2 + lag);
  }
  __device__ __forceinline__ long long all() const { return items > 0 ? before(items - 1) + last : 0; }
};
__device__ __forceinline__ long long shuffle64(long long v, int lane) {
  return (long long)__shfl_sync(0xffffffffu, (unsigned long long)v, lane);
}
// An item, or the part of it that a range holds.
struct Segment {
  int valid, q_base, nq, k_base, nk, head, q0, t_lo, n_t, part;      // part: 0 the whole item, 1 not its beginning, 2 its beginning
};
// What the joining launch has to know of a range: the item that is cut where it ends, if the item begins in it.
struct CutItem {
  int valid, q_base, nq, hist, head, q0, last, reserved;      // last: the range that holds the item's end
};
struct Deal {
  long long total, items;      // steps and items of all heads
  int dearest, ranges;         // ranges: 0 where items stay whole
  // The whole warp takes part.
  __device__ __forceinline__ Deal(const PromptParams& P, int ctas) {
    total = items = 0;
    dearest = 0;
    for (int b = threadIdx.x & 31; b < P.n_seq; b += 32) {
      const ItemSteps k(load_sequence(P, b));
      total += k.all();
      items += k.items;
      if (k.items > 0) dearest = max(dearest, k.last);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      total += (long long)__shfl_xor_sync(0xffffffffu, (unsigned long long)total, d);
      items += (long long)__shfl_xor_sync(0xffffffffu, (unsigned long long)items, d);
    }
    dearest = __reduce_max_sync(0xffffffffu, dearest);
    total *= P.q_heads;
    items *= P.q_heads;
    ranges = 0;
    const int most = (int)min((long long)ctas, total / max(min(kPrShortest, dearest), 1));
    if (most < 2 || !P.records) return;
    // in whole numbers, so that the launches agree: times ctas x rounds, and a tenth less
    const long long rounds = (items + ctas - 1) / ctas;
    if (rounds > 64) return;
    const long long whole = max(dearest * ctas * rounds, rounds > 1 ? total * rounds + (long long)dearest * ctas : 0);
    if (10 * (total + (long long)kPrCut * most) * ctas * rounds < 9 * most * whole) ranges = most;
  }
  __device__ __forceinline__ long long cut(int range) const { return (long long)((double)total / ranges * range); }
  // A cut near the edge of an item moves there.
  __device__ __forceinline__ int slack() const { return max((int)(total / ranges / 16), 1); }
};
// A place in the list of steps.
struct ItemCursor {
  int b, head, item, step, cost;      // step: inside the item
  Sequence s;
};
// The place of step u, which exists; the whole warp takes part.
__device__ __forceinline__ ItemCursor seek_item(const PromptParams& P, long long u) {
  const int lane = threadIdx.x & 31;
  ItemCursor c = {};
  for (int b0 = 0; b0 < P.n_seq; b0 += 32) {
    const Sequence s = b0 + lane < P.n_seq ? load_sequence(P, b0 + lane) : Sequence{0, 0, 0, 0};
    const long long mine = ItemSteps(s).all() * P.q_heads;
    long long sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = (long long)__shfl_up_sync(0xffffffffu, (unsigned long long)sum, d);
      if (lane >= d) sum += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, sum > u);
    if (found) {
      const int who = __ffs(found) - 1;
      c.b = b0 + who;
      c.s.q0 = __shfl_sync(0xffffffffu, s.q0, who);
      c.s.nq = __shfl_sync(0xffffffffu, s.nq, who);
      c.s.k0 = __shfl_sync(0xffffffffu, s.k0, who);
      c.s.nk = __shfl_sync(0xffffffffu, s.nk, who);
      u -= shuffle64(sum - mine, who);
      break;
    }
    u -= shuffle64(sum, 31);
  }
  const ItemSteps k(c.s);
  const long long per_head = k.all();
  c.head = (int)(u / per_head);
  u -= c.head * per_head;
  int lo = 0, hi = k.items;      // before(lo) <= u, and u < before(hi) or hi is behind the last item
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (k.before(mid) <= u) lo = mid;
    else hi = mid;
  }
  c.item = lo;
  c.step = (int)(u - k.before(lo));
  c.cost = k.cost(lo);
  return c;
}
// The item behind, if there is one; items without a key, of which there is no step, are passed over.
__device__ __forceinline__ void next_item(const PromptParams& P, ItemCursor& c) {
  c.step = 0;
  do {
    if (++c.item >= ItemSteps(c.s).items) {
      c.item = 0;
      if (++c.head == P.q_heads) {
        c.head = 0;
        do {
          if (++c.b >= P.n_seq) return;
          c.s = load_sequence(P, c.b);
        } while (ItemSteps(c.s).all() == 0);
      }
    }
    c.cost = ItemSteps(c.s).cost(c.item);
  } while (c.cost == 0);
}
// The first step of a range and its place; step `total` behind the last range.
__device__ __forceinline__ ItemCursor range_begin(const PromptParams& P, const Deal& deal, int range, long long& step) {
  step = deal.total;
  if (range >= deal.ranges) return ItemCursor{};
  step = deal.cut(range);
  ItemCursor c = seek_item(P, step);
  if (c.step <= deal.slack()) {
    step -= c.step;
    c.step = 0;
  } else if (c.cost - c.step <= deal.slack()) {
    step += c.cost - c.step;
    next_item(P, c);
  }
  return c;
}

constexpr int kPrAhead = 4;                // segments described ahead
template <int D>
struct PromptShape {
  static constexpr int kSlabs = D / 64;                       // column slabs of an operand tile
  static constexpr int kTileBytes = kSlabs * kPrSlab;
  static constexpr int kStages = D == 128 ? 2 : 4;            // K and V tiles in flight
  static constexpr int kTiles = (2 + 2 * kStages) * kTileBytes;
  static constexpr int kBars = 2 + 4 * kStages + 4 * kStages + 6 + 2 * kPrAhead;
  // Columns of tensor memory: S_A, S_B, O_A, O_B.  Two outputs of 64 channels leave room for P beside S, so that the next S
  // is contracted while the softmax of this one runs (four chunks of up to 700 queries behind 2500 to 7000 keys, 32 heads:
  // 105 us against 119); with 128 channels P lies over the first half of S.
  static constexpr bool kApart = D == 64;
  static constexpr int kOutput = 2 * kPrTile, kP = kApart ? kOutput + 2 * D : 0, kPEach = kApart ? kPrTile / 2 : kPrTile;
  // then: TMEM base, flags, the softmax warps' progress; segments; barriers; two sets of three lists of D positions
  static constexpr int kSegmentOffset = kTiles + 64, kBarOffset = kSegmentOffset + kPrAhead * 64, kListOffset = kBarOffset + 8 * kBars;
  static constexpr int kSmem = kListOffset + 2 * 3 * D * 4;
};
static_assert(sizeof(Segment) <= 64, "a segment's place");

constexpr int kFar = 0x7fffffff;
// positions of the first +infinity, -infinity and NaN of each channel among the cleaned values
enum { kBadPlus = 0, kBadMinus = 1, kBadNan = 2 };

// What the roles derive from a segment.
struct SegmentTiles {
  int hist, n_a, n_b, t_dark;
  __device__ __forceinline__ explicit SegmentTiles(const Segment& g) {
    hist = g.nk - g.nq;       // negative where the first queries have no key at all
    // tiles that A and B walk; B may hold no query at all, and a tile no key
    const int all_a = (max(min(g.nk, hist + g.q0 + kPrTile), 0) + kPrTile - 1) / kPrTile;
    const int all_b = g.q0 + kPrTile < g.nq ? (max(min(g.nk, hist + g.q0 + kPrRows), 0) + kPrTile - 1) / kPrTile : 0;
    n_a = max(0, min(all_a, g.t_lo + g.n_t) - g.t_lo);
    n_b = max(0, min(all_b, g.t_lo + g.n_t) - g.t_lo);
    // Tiles from t_dark on hold rows that some query of this item must not see.  Their values arrive at barriers of
    // their own: the warp that cleans them looks at no earlier tile, and a parity alone does not tell phases apart.
    t_dark = max(0, (max(hist + g.q0 + 1, 0) >> 7) - g.t_lo);
  }
};

template <typename QT, int D>
__global__ void __launch_bounds__(kPrThreads, 1) prompt_kernel(const PromptParams P, const __grid_constant__ CUtensorMap map_q,
                                                               const __grid_constant__ CUtensorMap map_k,
                                                               const __grid_constant__ CUtensorMap map_v) {
  using S = PromptShape<D>;
  constexpr int kStages = S::kStages, kTileBytes = S::kTileBytes;
  extern __shared__ __align__(1024) unsigned char pr_raw[];
  const unsigned smem0 = tc_smem(pr_raw);
  const unsigned sQ = smem0, sKb = smem0 + 2 * kTileBytes, sVb = sKb + kStages * kTileBytes;
  unsigned* const tmem_base_p = (unsigned*)(pr_raw + S::kTiles);
  volatile int* const abort_flag = (volatile int*)(pr_raw + S::kTiles + 4);
  volatile int* const any_bad = (volatile int*)(pr_raw + S::kTiles + 16);      // of even and odd segments
  volatile int* const ended = (volatile int*)(pr_raw + S::kTiles + 32);        // per softmax warp: segments that it is done with
  int* const lists = (int*)(pr_raw + S::kListOffset);         // [2][3][D]
  const unsigned bars = smem0 + S::kBarOffset;
  // Per stage: K and V tiles, V tiles that want cleaning, such tiles cleaned, S and O of tiles A and B; A and B: P,
  // first half of P, S read (where P lies apart); segments.  Barriers of a stage, because a parity alone does not tell
  // phases apart: a stage is not used again before everyone has seen its last phase.
  const unsigned bar_q = bars, bar_e = bars + 8, bar_k = bars + 16, bar_v = bar_k + 8 * kStages, bar_d = bar_v + 8 * kStages;
  const unsigned bar_c = bar_d + 8 * kStages, bar_s = bar_c + 8 * kStages /* [x][stage] */, bar_o = bar_s + 16 * kStages /* [x][stage] */;
  const unsigned bar_p = bar_o + 16 * kStages, bar_h = bar_p + 16;
  const unsigned bar_r = bar_h + 16;
  const unsigned bar_g = bar_r + 16, bar_gfree = bar_g + 8 * kPrAhead;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  follow_stream();       // cu_q and cu_k may come from the launch before this one
  if (smem0 & 1023u) {
    if (tid == 0) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
    return;
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_base_p)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == 9 && lane == 0) {
    *abort_flag = any_bad[0] = any_bad[1] = 0;
#pragma unroll
    for (int i = 0; i < kPrSoftmaxWarps; ++i) ended[i] = 0;
    tc_bar_init(bar_q, 1);
    tc_bar_init(bar_e, 1);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      tc_bar_init(bar_s + 8 * i, 1);
      tc_bar_init(bar_s + 8 * (kStages + i), 1);
      tc_bar_init(bar_o + 8 * i, 1);
      tc_bar_init(bar_o + 8 * (kStages + i), 1);
      tc_bar_init(bar_k + 8 * i, 1);
      tc_bar_init(bar_v + 8 * i, 1);
      tc_bar_init(bar_d + 8 * i, 1);
      tc_bar_init(bar_c + 8 * i, 1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      tc_bar_init(bar_p + 8 * i, kPrTile);
      tc_bar_init(bar_h + 8 * i, kPrTile);
      tc_bar_init(bar_r + 8 * i, kPrTile);
    }
#pragma unroll
    for (int i = 0; i < kPrAhead; ++i) {
      tc_bar_init(bar_g + 8 * i, 1);
      tc_bar_init(bar_gfree + 8 * i, kPrSoftmaxWarps + 3);       // the softmax warps, the MMA, TMA and cleaning warps
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < 2 * 3 * D; i += kPrThreads) lists[i] = kFar;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_base_p;
  allow_next();
  auto wait = [&](unsigned mbar, unsigned parity) { tc_wait(mbar, parity, abort_flag); };   // goes on in either case
  // Segment n, the same for a whole warp; an invalid one behind the last, and once a wait has given up.
  auto segment = [&](int n) {
    const bool there = tc_wait(bar_g + 8 * (n % kPrAhead), (unsigned)(n / kPrAhead) & 1u, abort_flag);
    Segment g = *(const Segment*)(pr_raw + S::kSegmentOffset + 64 * (n % kPrAhead));
    if (__any_sync(0xffffffffu, !there || *abort_flag != 0)) g.valid = 0;
    __syncwarp();
    if (lane == 0) pf_arrive(bar_gfree + 8 * (n % kPrAhead));
    return g;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrIssueRegs));
    if (warp == 11) {
      // ================================================================ deals the segments
      int n = 0;
      auto publish = [&](const Segment& g) {
        if (n >= kPrAhead) wait(bar_gfree + 8 * (n % kPrAhead), (unsigned)(n / kPrAhead - 1) & 1u);
        __syncwarp();
        if (lane == 0) {
          *(Segment*)(pr_raw + S::kSegmentOffset + 64 * (n % kPrAhead)) = g;
          pf_arrive(bar_g + 8 * (n % kPrAhead));
        }
        ++n;
      };
      // the n-th whole item of this CTA; false where there are no more
      auto whole = [&](long long round) {
        const int ctas = gridDim.x;
        const long long unit = round * ctas + ((round & 1) ? ctas - 1 - (int)blockIdx.x : (int)blockIdx.x), rank = unit / P.q_heads;
        Sequence s;
        int index = 0;
        if (rank > 0x3fffffff || find_item(P, (int)rank, (P.k_rows + kPrTile - 1) / kPrTile, s, index) < 0) return false;
        const int cost = ItemSteps(s).cost(index);
        if (cost > 0) publish(Segment{1, s.q0, s.nq, s.k0, s.nk, (int)(unit - rank * P.q_heads), index * kPrRows, 0, cost, 0});
        return true;
      };
      long long round = 0;
      bool more = true, cut = false;
      if (!P.records) {      // nothing is cut: the first item starts before anything else is looked at
        more = whole(round++);
      } else {
        const Deal deal(P, gridDim.x);
        CutItem mark = {};
        cut = deal.ranges > 0;
        if (cut && (int)blockIdx.x < deal.ranges) {
          long long step, end;
          range_begin(P, deal, blockIdx.x + 1, end);
          ItemCursor c = range_begin(P, deal, blockIdx.x, step);
          while (step < end && !__any_sync(0xffffffffu, *abort_flag != 0)) {
            const int steps = (int)min(end - step, (long long)(c.cost - c.step));
            publish(Segment{1, c.s.q0, c.s.nq, c.s.k0, c.s.nk, c.head, c.item * kPrRows, c.step, steps, steps == c.cost ? 0 : c.step ? 1 : 2});
            step += steps;
            if (step == end && c.step + steps < c.cost && c.step == 0) {
              // the item goes on behind this range, and begins in it
              const long long item = step - steps;
              int last = blockIdx.x + 1;
              while (last + 1 < deal.ranges && deal.cut(last + 1) < item + c.cost - deal.slack()) ++last;
              mark = CutItem{1, c.s.q0, c.s.nq, c.s.nk - c.s.nq, c.head, c.item * kPrRows, last, 0};
            }
            if (step < end) next_item(P, c);
          }
        }
        if (lane == 0) P.cuts[blockIdx.x] = mark;
      }
      // offsets that the tensors do not hold, and queries without a key
      for (int b = blockIdx.x; b < P.n_seq; b += gridDim.x) {
        if (lane == 0 && bad_sequence(P, b)) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
        const Sequence s = load_sequence(P, b);
        for (long long i = lane; i < (long long)(s.nq - s.nk) * P.q_heads; i += 32) {
          const int row = s.q0 + (int)(i / P.q_heads), head = (int)(i % P.q_heads);
          for (int c = 0; c < D; c += 8) *(uint4*)((QT*)P.out + head * P.o_sh + row * P.o_st + c) = make_uint4(0u, 0u, 0u, 0u);
          if (P.lse) P.lse[head * P.lse_stride + row] = __int_as_float(0xff800000);
        }
      }
      while (!cut && more && !__any_sync(0xffffffffu, *abort_flag != 0)) more = whole(round++);
      publish(Segment{});
    } else if (warp == 9) {
      // ================================================================ TMA warp
      // Step u of the CTA uses stage u % kStages.  Bits of a stage: the next parity of its plain and dark value barriers and of
      // its barriers of tiles A and B, and whether the step that has it ends with tile B.
      unsigned u = 0, v_parity = 0, d_parity = 0, a_parity = 0, b_parity = 0, ends_b = 0, queries = 0;
      // the last contraction of kind `bar` of the step that had a stage before
      auto stage_done = [&](unsigned bar, unsigned bit, unsigned st) {
        const bool b = (ends_b & bit) != 0;
        return tc_wait(bar + 8 * (b ? kStages + st : st), (b ? b_parity : a_parity) & bit ? 0u : 1u, abort_flag);
      };
      int n = 0;
      for (Segment g = segment(0); g.valid; g = segment(++n)) {
        const SegmentTiles T(g);
        const int kvh = g.head / (P.q_heads / P.kv_heads);
        if (lane == 0) {
          for (int t = 0; t < g.n_t; ++t, ++u) {
            const unsigned st = u % kStages, bit = 1u << st;
            if (u >= kStages && !stage_done(bar_s, bit, st)) break;
            const int y = g.k_base + (g.t_lo + t) * kPrTile;
            pf_expect(bar_k + 8 * st, kTileBytes);
#pragma unroll
            for (int c = 0; c < S::kSlabs; ++c) pf_tma(sKb + st * kTileBytes + c * kPrSlab, &map_k, 64 * c, y, kvh, bar_k + 8 * st);
            if (t == 0) {
              // the query tiles are free once the last score contraction of the segment before is done
              const unsigned before = (u + kStages - 1) % kStages;
              if (u > 0 && !stage_done(bar_s, 1u << before, before)) {
                ++u;      // its K tile is on the way
                break;
              }
              ++queries;
              pf_expect(bar_q, 2 * kTileBytes);
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int c = 0; c < S::kSlabs; ++c)
                  pf_tma(sQ + x * kTileBytes + c * kPrSlab, &map_q, 64 * c, g.q_base + g.q0 + x * kPrTile, g.head, bar_q);
            }
            if (u >= kStages && !stage_done(bar_o, bit, st)) {
              ++u;
              break;
            }
            if (t < T.n_a) a_parity ^= bit;
            if (t < T.n_b) b_parity ^= bit;
            ends_b = t < T.n_b ? ends_b | bit : ends_b & ~bit;
            const unsigned bar = (t < T.t_dark ? bar_v : bar_d) + 8 * st;
            pf_expect(bar, kTileBytes);
#pragma unroll
            for (int c = 0; c < S::kSlabs; ++c) pf_tma(sVb + st * kTileBytes + c * kPrSlab, &map_v, 64 * c, y, kvh, bar);
            if (t < T.t_dark) v_parity ^= bit;
            else d_parity ^= bit;
          }
        }
        __syncwarp();
      }
      if (lane == 0 && *abort_flag) {
        // copies in flight end before the CTA leaves: the last of each barrier that was used (a parity bit is that of the next)
        for (unsigned i = 0; i < kStages; ++i) {
          const unsigned bit = 1u << i, used = (u + kStages - 1 - i) / kStages;      // K tiles of this stage
          if (used) tc_drain(bar_k + 8 * i, (used - 1) & 1u);
          tc_drain(bar_v + 8 * i, v_parity & bit ? 0u : 1u);
          tc_drain(bar_d + 8 * i, d_parity & bit ? 0u : 1u);
        }
        if (queries) tc_drain(bar_q, (queries - 1) & 1u);
      }
    } else if (warp == 8) {
      // ================================================================ MMA warp
      constexpr bool kBf16 = !std::is_same<QT, __half>::value;
      constexpr unsigned idesc_s = tc_idesc<kBf16, 128, 128, false>(), idesc_o = tc_idesc<kBf16, 128, D, true>();
      auto issue_s = [&](int x, unsigned u) {      // S_x = Q_x K^T
        const unsigned q = sQ + x * kTileBytes, k = sKb + (u % kStages) * kTileBytes;
        if (tc_elect()) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const unsigned off = (kk >> 2) * kPrSlab + (kk & 3) * 32;
            tc_mma(tmem + x * kPrTile, tc_desc(q + off, 16, 1024), tc_desc(k + off, 16, 1024), idesc_s, kk > 0);
          }
          tc_commit(bar_s + 8 * (x * kStages + u % kStages));
        }
      };
      auto issue_o = [&](int x, unsigned u, bool first, int half) {      // O_x += P_x V, half a tile of tokens at a time
        const unsigned v = sVb + (u % kStages) * kTileBytes;
        if (tc_elect()) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int kk = 4 * half + k;
            tc_mma_ta(tmem + S::kOutput + x * D, tmem + S::kP + x * S::kPEach + kk * 8, tc_desc(v + kk * 2048, kPrSlab, 1024), idesc_o,
                      (!first || kk > 0) ? 1u : 0u);
          }
          if (half) tc_commit(bar_o + 8 * (x * kStages + u % kStages));
        }
      };
      unsigned count[2] = {0, 0}, v_parity = 0, d_parity = 0, u = 0;
      auto contract_o = [&](int x, bool first) {
        wait(bar_h + 8 * x, count[x] & 1u);     // S_x read where P_x lies over it, the first half of P_x written, the rows of the segment before stored
        tc_fence_after();
        issue_o(x, u, first, 0);
        wait(bar_p + 8 * x, count[x] & 1u);     // the second half
        tc_fence_after();
        issue_o(x, u, first, 1);
        ++count[x];
      };
      int n = 0;
      Segment g = segment(0);
      if (g.valid) {
        SegmentTiles T(g), next = T;
        wait(bar_q, 0);
        wait(bar_k, 0);
        tc_fence_after();
        if (T.n_a > 0) issue_s(0, 0);
        if (T.n_b > 0) issue_s(1, 0);
        int t = 0;
        while (true) {
          const unsigned st = u % kStages, bit = 1u << st;
          const bool dark = t >= T.t_dark, a_now = t < T.n_a, b_now = t < T.n_b, first = t == 0;
          auto wait_v = [&]() {
            if (!dark) {
              wait(bar_v + 8 * st, v_parity & bit ? 1u : 0u);
              v_parity ^= bit;
            } else {
              wait(bar_c + 8 * st, d_parity & bit ? 1u : 0u);
              d_parity ^= bit;
            }
          };
          if constexpr (!S::kApart) {
            wait_v();
            if (a_now) contract_o(0, first);
          }
          // the step behind this one, perhaps of another segment
          bool more = true;
          if (++t == g.n_t) {
            t = 0;
            g = segment(++n);
            more = g.valid;
          }
          if (t == 0) next = SegmentTiles(g);
          if (more) {
            if (t == 0) wait(bar_q, (unsigned)n & 1u);
            wait(bar_k + 8 * ((u + 1) % kStages), ((u + 1) / kStages) & 1u);
            if constexpr (S::kApart)
              if (a_now) wait(bar_r, count[0] & 1u);
            tc_fence_after();
            if (t < next.n_a) issue_s(0, u + 1);
          }
          if constexpr (S::kApart) {
            wait_v();
            if (a_now) contract_o(0, first);
            if (more && b_now) {
              wait(bar_r + 8, count[1] & 1u);
              tc_fence_after();
            }
            if (more && t < next.n_b) issue_s(1, u + 1);
          }
          if (b_now) contract_o(1, first);
          if (!more) break;
          if (!S::kApart && t < next.n_b) issue_s(1, u + 1);
          if (t == 0) T = next;
          ++u;
        }
      }
    } else {
      // ================================================================ the warp that cleans value tiles
      // chunk c of row r lies at chunk c ^ (r & 7) of its slab
      unsigned u = 0, d_parity = 0, held = 0;      // held: sets of lists with something in them
      int n = 0;
      for (Segment g = segment(0); g.valid; g = segment(++n)) {
        const SegmentTiles T(g);
        int* const first_bad = lists + (n & 1) * 3 * D;
        // The lists were those of the segment before the last: nothing changes there before every softmax warp has ended that.
        // A word per warp, because a sum over them does not tell: where tile A (or a tile B without rows) is a segment
        // ahead, its warps would make up for those that still read.  The MMA warp waits for the tile in work meanwhile, and
        // that wait, of a second, raises the abort flag long before this one would run out.  (Raising it here as well costs
        // short prompts 4%, on paths that have nothing to wait for: 301 tokens 13.2 us instead of 12.7.)
        auto others_ended = [&]() {
          for (int it = 0; it < kTcTries && *abort_flag == 0; ++it) {
            int least = ended[0];
#pragma unroll
            for (int i = 1; i < kPrSoftmaxWarps; ++i) least = min(least, ended[i]);
            if (least >= n - 1) break;
            __nanosleep(it < 4096 ? 64 : 16384);
          }
          __threadfence_block();
        };
        if (T.t_dark < g.n_t && (held >> (n & 1)) & 1u) {
          others_ended();
          __syncwarp();
          for (int i = lane; i < 3 * D; i += 32) first_bad[i] = kFar;
          any_bad[n & 1] = 0;
          held &= ~(1u << (n & 1));
          __syncwarp();
        }
        for (int t = T.t_dark; t < g.n_t; ++t) {
          const unsigned st = (u + t) % kStages, bit = 1u << st;
          wait(bar_d + 8 * st, d_parity & bit ? 1u : 0u);
          d_parity ^= bit;
          unsigned char* const tile = pr_raw + (sVb - smem0) + st * kTileBytes;
          const int kv0 = (g.t_lo + t) * kPrTile, rows = min(g.nk - kv0, kPrTile);     // rows of the sequence
          // a first look finds the largest magnitude of every batch, as whole numbers: the second is for what is not finite
          constexpr unsigned kOnes = std::is_same<QT, __half>::value ? 0x7c00u : 0x7f80u;
          bool touched = false;
#pragma unroll 1
          for (int i0 = lane; i0 < kTileBytes / 16; i0 += 32 * 8) {
            uint4 w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = *(const uint4*)(tile + 16 * (i0 + 32 * j));
            unsigned most = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int row = ((i0 + 32 * j) >> 3) & (kPrTile - 1);
              if (row >= rows) {
                *(uint4*)(tile + 16 * (i0 + 32 * j)) = make_uint4(0u, 0u, 0u, 0u);
                touched = true;
              } else {
                most = __vmaxu2(__vmaxu2(__vmaxu2(most, w[j].x & 0x7fff7fffu), w[j].y & 0x7fff7fffu), __vmaxu2(w[j].z & 0x7fff7fffu, w[j].w & 0x7fff7fffu));
              }
            }
            if ((most & 0xffffu) < kOnes && (most >> 16) < kOnes) continue;
            others_ended();
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
              const int i = i0 + 32 * j, row = (i >> 3) & (kPrTile - 1), channel = (i / (kPrTile * 8)) * 64 + (((i & 7) ^ (row & 7)) << 3);
              unsigned short* const values = (unsigned short*)(tile + 16 * i);
#pragma unroll 1
              for (int k = 0; k < 8 && row < rows; ++k) {
                const unsigned bits = values[k];
                if ((bits & 0x7fffu) < kOnes) continue;
                const int kind = (bits & 0x7fffu) > kOnes ? kBadNan : (bits & 0x8000u) ? kBadMinus : kBadPlus;
                atomicMin(first_bad + kind * D + channel + k, kv0 + row);
                values[k] = 0;
                any_bad[n & 1] = 1;
                touched = true;
              }
            }
          }
          if (touched) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (any_bad[n & 1]) held |= 1u << (n & 1);
          if (lane == 0) pf_arrive(bar_c + 8 * st);
        }
        u += g.n_t;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrSoftmaxRegs));
    // ================================================================ softmax warps
    const int x = warp >> 2;                       // 0: tile A, 1: tile B
    const int row = tid & (kPrTile - 1);           // query row inside the tile = TMEM lane
    const unsigned lane_field = (unsigned)((warp & 3) * 32) << 16;
    const unsigned tS = tmem + lane_field + x * kPrTile, tO = tmem + lane_field + S::kOutput + x * D, tP = tmem + lane_field + S::kP + x * S::kPEach;
    const unsigned my_s = bar_s + 8 * x * kStages, my_p = bar_p + 8 * x, my_o = bar_o + 8 * x * kStages;
    unsigned u = 0, parity = 0;                    // the segment's first step; a bit per stage: the next parity of this tile's barriers
    int n = 0;
    for (Segment g = segment(0); g.valid; g = segment(++n)) {
      const SegmentTiles T(g);
      const int n_x = x ? T.n_b : T.n_a;
      const int q_row = g.q0 + x * kPrTile + row;
      const int q_pos = T.hist + q_row;              // keys at positions <= q_pos are visible
      const int diag0 = T.hist + g.q0 + x * kPrTile;     // first row's diagonal: tiles reaching beyond it need masks
      float m_ref = kPrNegBig, l_sum = 0.f;

      for (int t = 0; t < n_x; ++t) {
        const int kv0 = (g.t_lo + t) * kPrTile;
        // S(t) is complete; the contractions run in issue order, so that PV(t-1) is complete as well, if it was issued first:
        // P may be overwritten and O may be rescaled
        const unsigned st = (u + t) % kStages, bit = 1u << st;
        wait(my_s + 8 * st, parity & bit ? 1u : 0u);
        parity ^= bit;
        tc_fence_after();
        unsigned v[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tc_ld32(tS + 32 * q, v[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) tc_wait_ld32(v[q]);
        if constexpr (S::kApart) {
          tc_fence_before();
          pf_arrive(bar_r + 8 * x);
        }
        if (kv0 + kPrTile - 1 > diag0) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (kv0 + 32 * q + c > q_pos) v[q][c] = 0xff800000u;
        }
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = __uint_as_float(v[q][0]);
#pragma unroll
          for (int c = 1; c < 32; ++c) top[q] = fmaxf(top[q], __uint_as_float(v[q][c]));
        }
        const float smax = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (S::kApart && t > 0) {      // S(t) was issued before PV(t-1)
          const unsigned last = (u + t - 1) % kStages;
          wait(my_o + 8 * last, (parity >> last) & 1u ? 0u : 1u);
          tc_fence_after();
        }
        const bool raise = smax * P.scale_log2e > m_ref + kPrSlack;
        if (__any_sync(0xffffffffu, raise)) {
          // rare after the first tile: bring the running sum and the output accumulator to the new reference maximum
          const float m_new = raise ? smax * P.scale_log2e : m_ref;
          const float factor = pf_exp2(m_ref - m_new);
          l_sum *= factor;
          m_ref = m_new;
          if (t > 0) {
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 16) {
              unsigned o[16];
              tc_ld16(tO + c0, o);
              tc_wait_ld16(o);
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * factor);
              tc_st16(tO + c0, o);
            }
          }
        }
        const unsigned long long scale2 = pf_pair(P.scale_log2e, P.scale_log2e), minus_ref2 = pf_pair(-m_ref, -m_ref);
        unsigned long long sum2 = pf_pair(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          unsigned packed[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float e0, e1;
            pf_unpair(pf_fma2(pf_pair(__uint_as_float(v[q][c]), __uint_as_float(v[q][c + 1])), scale2, minus_ref2), e0, e1);
            e0 = pf_exp2(e0);
            e1 = pf_exp2(e1);
            sum2 = pf_add2(sum2, pf_pair(e0, e1));
            packed[c >> 1] = pf_pack2<QT>(e0, e1);
          }
          tc_st16(tP + 16 * q, packed);
          if (q == 1) {   // S has been read, the first half of P is in tensor memory: the contraction with V starts
            tc_wait_st();
            tc_fence_before();
            pf_arrive(bar_h + 8 * x);
          }
        }
        float sum_even, sum_odd;
        pf_unpair(sum2, sum_even, sum_odd);
        l_sum += sum_even + sum_odd;
        tc_wait_st();
        tc_fence_before();
        pf_arrive(my_p);
      }
      if (n_x > 0) {
        const unsigned st = (u + n_x - 1) % kStages;
        wait(my_o + 8 * st, (parity >> st) & 1u ? 0u : 1u);
      }
      u += g.n_t;
      tc_fence_after();
      const bool live = *abort_flag == 0 && q_row < g.nq;
      // complete: the last contraction came after the last cleaned tile
      const int* const first_bad = lists + (n & 1) * 3 * D;
      const bool bad = T.t_dark < g.n_t && any_bad[n & 1] != 0;
      // What cleaning took out, for the rows that see it: the sum of a NaN or of infinities of both signs is NaN.
      auto put_back = [&](float o, int channel) {
        const bool plus = first_bad[kBadPlus * D + channel] <= q_pos, minus = first_bad[kBadMinus * D + channel] <= q_pos;
        if (first_bad[kBadNan * D + channel] <= q_pos || (plus && minus)) return __int_as_float(0x7fc00000);
        return plus ? o + __int_as_float(0x7f800000) : minus ? o + __int_as_float(0xff800000) : o;
      };

      if (g.part == 0) {
        // a row without keys gives zeros; one whose logits are all -infinity divides zero by zero, as its formula does
        const float inv = q_pos < 0 ? 0.f : 1.f / l_sum;
        if (live && P.lse) P.lse[g.head * P.lse_stride + g.q_base + q_row] = q_pos < 0 ? __int_as_float(0xff800000) : (m_ref + log2f(l_sum)) * kLn2;
        QT* orow = (QT*)P.out + (long long)g.head * P.o_sh + (long long)(g.q_base + q_row) * P.o_st;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          unsigned v[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = 0u;
          if (n_x > 0) {
            tc_ld32(tO + c0, v);
            tc_wait_ld32(v);
          }
          if (bad)
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(put_back(__uint_as_float(v[c]), c0 + c));
          if (live) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              uint4 w;
              w.x = pf_pack2<QT>(__uint_as_float(v[8 * q4 + 0]) * inv, __uint_as_float(v[8 * q4 + 1]) * inv);
              w.y = pf_pack2<QT>(__uint_as_float(v[8 * q4 + 2]) * inv, __uint_as_float(v[8 * q4 + 3]) * inv);
              w.z = pf_pack2<QT>(__uint_as_float(v[8 * q4 + 4]) * inv, __uint_as_float(v[8 * q4 + 5]) * inv);
              w.w = pf_pack2<QT>(__uint_as_float(v[8 * q4 + 6]) * inv, __uint_as_float(v[8 * q4 + 7]) * inv);
              *(uint4*)(orow + c0 + 8 * q4) = w;
            }
          }
        }
      } else {
        // partial record of this row: unnormalised output, reference maximum, sum
        float* rec = P.records + (((long long)blockIdx.x * 2 + (g.part == 2)) * kPrRows + x * kPrTile + row) * (D + 2);
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          unsigned v[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = 0u;
          if (n_x > 0) {
            tc_ld32(tO + c0, v);
            tc_wait_ld32(v);
          }
          if (bad)
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __float_as_uint(put_back(__uint_as_float(v[c]), c0 + c));
          if (live)
#pragma unroll
            for (int c = 0; c < 32; c += 2) *(float2*)(rec + c0 + c) = make_float2(__uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        }
        if (live) *(float2*)(rec + D) = make_float2(m_ref, l_sum);
      }
      tc_fence_before();      // O has been read: the arrivals of the next segment let it be overwritten
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();      // the lists have been read
        ended[warp] = n + 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(P.status, INQ_STATUS_WAIT_TIMEOUT);
  if (warp == 8) {
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {
      // contractions may be in flight: they end before tensor memory is freed and the CTA leaves
      if (tc_elect()) tc_commit(bar_e);
      tc_drain(bar_e, 0);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the parts of the items that ranges cut: out = sum_c O_c 2^(m_c - m) / sum_c l_c 2^(m_c - m) over the parts in their
// order.  Block (r, y) takes rows 32 y .. of the item that is cut where range r ends, if it begins in range r; a warp four
// rows at once, a lane D / 32 channels, and the next part is asked for while one is added.
constexpr int kPrMergeRows = 32, kPrMergeEach = 4;
template <typename QT, int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptParams P) {
  follow_stream();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.x;
  const CutItem c = P.cuts[r];
  const int row0 = blockIdx.y * kPrMergeRows + warp * kPrMergeEach;
  if (!c.valid || c.q0 + row0 >= c.nq) return;
  float top[kPrMergeEach], l[kPrMergeEach] = {};
  float2 o[kPrMergeEach][D / 64] = {};
#pragma unroll
  for (int i = 0; i < kPrMergeEach; ++i) top[i] = kPrNegBig;
#pragma unroll 2
  for (int part = r; part <= c.last; ++part) {
    float2 ml[kPrMergeEach], x[kPrMergeEach][D / 64];
#pragma unroll
    for (int i = 0; i < kPrMergeEach; ++i) {      // rows that the item does not have hold whatever memory does, and are not stored
      const float2* const rec = (const float2*)(P.records + ((2LL * part + (part == r)) * kPrRows + row0 + i) * (D + 2));
      ml[i] = __ldcg(rec + D / 2);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) x[i][k] = __ldcg(rec + 32 * k + lane);
    }
#pragma unroll
    for (int i = 0; i < kPrMergeEach; ++i) {
      const float next = fmaxf(top[i], ml[i].x), before = pf_exp2(top[i] - next), w = pf_exp2(ml[i].x - next);
      top[i] = next;
      l[i] = fmaf(ml[i].y, w, l[i] * before);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) o[i][k] = make_float2(fmaf(x[i][k].x, w, o[i][k].x * before), fmaf(x[i][k].y, w, o[i][k].y * before));
    }
  }
#pragma unroll
  for (int i = 0; i < kPrMergeEach; ++i) {
    const int q_row = c.q0 + row0 + i;
    if (q_row >= c.nq) return;
    const bool empty = c.hist + q_row < 0;
    const float inv = empty ? 0.f : 1.f / l[i];
    QT* out = (QT*)P.out + (long long)c.head * P.o_sh + (long long)(c.q_base + q_row) * P.o_st;
#pragma unroll
    for (int k = 0; k < D / 64; ++k) *(unsigned*)(out + 64 * k + 2 * lane) = pf_pack2<QT>(o[i][k].x * inv, o[i][k].y * inv);
    if (lane == 0 && P.lse) P.lse[c.head * P.lse_stride + c.q_base + q_row] = empty ? __int_as_float(0xff800000) : (top[i] + log2f(l[i])) * kLn2;
  }
}

// ---------------------------------------------------------------------------------------- attention weights of keys
// An item is 256 keys (tiles A and B, two softmax warpgroups each, which share out the columns) of one KV head; a step of it
// is 128 columns of queries:
// a tile of 128 queries of one query head of the group or, with a window of at most 64, the windows of 128 / width heads
// side by side.  The steps of all items form one list (request, KV head, keys rising, then query heads and queries), cut
// into equal ranges, one per CTA: what an item costs, 256 keys near the end of a sequence a fraction of the first ones,
// then does not matter.  An item that a range cuts leaves its sums to a second launch; items of few steps are not cut.
// The keys and queries of the steps to come are on their way while this one's are used; score tiles are double
// buffered in tensor memory (x * 256 + 128 * (step % 2)), so that contraction and exponentials run side by side.  The
// exponentials bound it (128 x 128 of them take 1024 cycles of their unit, the contraction 512).
constexpr int kPwColumns = 4;                                 // steps whose columns are described ahead
constexpr int kPwColumnBytes = kPrTile * 4 + 32;              // the exponents of 128 columns, and a StepNote
// What a softmax thread has to know of a step.  Key row r of the item is seen by queries lo + r .. hi - 1 of a window, the
// columns from `columns` on belong to no head.  The last step of a range in an item tells where its sums go: `keys` rows
// of them, at weights + at or, of an item that is cut, at records + at.
struct StepNote {
  int lo, hi, columns, keys;
  long long at;
  int last, cut;
};
static_assert(sizeof(StepNote) == 32, "behind 128 exponents");
template <int D>
struct WeightsShape {
  static constexpr int kSlabs = D / 64;
  static constexpr int kTileBytes = kSlabs * kPrSlab;
  static constexpr int kStages = D == 128 ? 2 : 4;            // query tiles in flight
  static constexpr int kTiles = (4 + kStages) * kTileBytes;   // two items' key tiles A and B, the query tiles
  static constexpr int kBars = 4 + 2 * kStages + 8 + 2 * kPwColumns + 1;
  // after the tiles: TMEM base, abort flag, request counts; the range; barriers; what the columns of the next steps are
  static constexpr int kRangeOffset = kTiles + 16, kBarOffset = kTiles + 128, kColumnsOffset = kBarOffset + 8 * kBars + 8;
  static constexpr int kSumOffset = kColumnsOffset + kPwColumns * kPwColumnBytes;      // sums of the second halves of the columns
  static constexpr int kSmem = kSumOffset + kPrRows * 4;
};
constexpr int kPwThreads = 640;      // 16 softmax warps, then the MMA warp, the TMA warp, one that describes columns, an idle one
constexpr int kPwSoftmaxWarps = 16;
constexpr int kPwLaunchRegs = 96, kPwIssueRegs = 64, kPwSoftmaxRegs = (5 * kPwLaunchRegs - kPwIssueRegs) / 4;
constexpr int kPwWhole = 8;       // items of at most so many steps are not cut

// The steps of one KV head of a sequence.  Key tile t costs `groups` x (tiles - first(t)) steps, first(t) being its first
// tile of queries with one that sees its first key: min(max(2 t - lag, 0), tiles).
struct KeySteps {
  int nw, w0, tiles, lag, items, groups;
  __device__ __forceinline__ KeySteps(const PromptParams& P, const Sequence& s) {
    nw = P.window > 0 ? min(P.window, s.nq) : s.nq;      // queries that count, behind the first w0
    w0 = s.nq - nw;
    tiles = (nw + kPrTile - 1) / kPrTile;
    lag = (s.nk - nw + kPrTile - 1) >> 7;
    items = tiles > 0 ? (s.nk + kPrRows - 1) / kPrRows : 0;      // without queries there are no steps
    groups = (P.q_heads / P.kv_heads * P.width + kPrTile - 1) / kPrTile;
  }
  __device__ __forceinline__ int first(int t) const { return min(max(2 * t - lag, 0), tiles); }
  __device__ __forceinline__ int cost(int t) const { return groups * (tiles - first(t)); }
  __device__ __forceinline__ long long before(int t) const {
    // the sum of first() from 0 to t - 1: zero up to lag / 2, then rising by two, then `tiles`
    const long long full = min(t, max((tiles + lag + 1) >> 1, 0)), start = min((long long)max((lag >> 1) + 1, 0), full);
    const long long sum = full * (full - 1) - start * (start - 1) - (full - start) * lag + (t - full) * tiles;
    return groups * ((long long)t * tiles - sum);
  }
};
// Steps of all items; the whole warp takes part.
__device__ __forceinline__ long long count_steps(const PromptParams& P) {
  long long n = 0;
  for (int b = threadIdx.x & 31; b < P.n_seq; b += 32) {
    const KeySteps k(P, load_sequence(P, b));
    n += k.before(k.items);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) n += (long long)__shfl_xor_sync(0xffffffffu, (unsigned long long)n, d);
  return n * P.kv_heads;
}
// A place in the list of steps.
struct StepCursor {
  int b, kvh, tile, step, cost;      // step: inside the item, of `cost`
  Sequence s;
};
// The place of step u, which exists; the whole warp takes part.
__device__ __forceinline__ StepCursor seek_step(const PromptParams& P, long long u) {
  const int lane = threadIdx.x & 31;
  StepCursor c = {};
  for (int b0 = 0; b0 < P.n_seq; b0 += 32) {
    const Sequence s = b0 + lane < P.n_seq ? load_sequence(P, b0 + lane) : Sequence{0, 0, 0, 0};
    const KeySteps k(P, s);
    const long long mine = k.before(k.items) * P.kv_heads;
    long long sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = (long long)__shfl_up_sync(0xffffffffu, (unsigned long long)sum, d);
      if (lane >= d) sum += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, sum > u);
    if (found) {
      const int who = __ffs(found) - 1;
      c.b = b0 + who;
      c.s.q0 = __shfl_sync(0xffffffffu, s.q0, who);
      c.s.nq = __shfl_sync(0xffffffffu, s.nq, who);
      c.s.k0 = __shfl_sync(0xffffffffu, s.k0, who);
      c.s.nk = __shfl_sync(0xffffffffu, s.nk, who);
      u -= shuffle64(sum - mine, who);
      break;
    }
    u -= shuffle64(sum, 31);
  }
  const KeySteps k(P, c.s);
  const long long per_head = k.before(k.items);
  c.kvh = (int)(u / per_head);
  u -= c.kvh * per_head;
  int lo = 0, hi = k.items;      // before(lo) <= u < before(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (k.before(mid) <= u) lo = mid;
    else hi = mid;
  }
  c.tile = lo;
  c.step = (int)(u - k.before(lo));
  c.cost = k.cost(lo);
  return c;
}
// The first step of the item behind the one of `c`.
__device__ __forceinline__ void next_item(const PromptParams& P, StepCursor& c) {
  c.step = 0;
  if (++c.tile == KeySteps(P, c.s).items) {
    c.tile = 0;
    if (++c.kvh == P.kv_heads) {
      c.kvh = 0;
      do {
        if (++c.b >= P.n_seq) return;      // behind the last step
        c.s = load_sequence(P, c.b);
      } while (KeySteps(P, c.s).items == 0);
    }
  }
  c.cost = KeySteps(P, c.s).cost(c.tile);
}
// The ranges: as equal as whole steps and uncut small items allow.
__device__ __forceinline__ int range_count(long long total, int ctas) { return (int)min(total, (long long)ctas); }
__device__ __forceinline__ long long range_start(long long total, int range, int ranges) { return (long long)((double)total / ranges * range); }
__device__ __forceinline__ int range_of(long long total, long long step, int ranges) {
  int r = (int)min((long long)((double)step / ((double)total / ranges)), (long long)ranges - 1);
  while (r > 0 && range_start(total, r, ranges) > step) --r;
  while (r + 1 < ranges && range_start(total, r + 1, ranges) <= step) ++r;
  return r;
}
__device__ __forceinline__ StepCursor range_cursor(const PromptParams& P, long long total, int range, int ranges, long long& step) {
  step = range_start(total, range, ranges);
  StepCursor c = seek_step(P, step);
  if (c.cost <= kPwWhole) {
    step -= c.step;
    c.step = 0;
  }
  return c;
}

template <typename QT, int D>
__global__ void __launch_bounds__(kPwThreads, 1) prompt_weights_kernel(const PromptParams P, const __grid_constant__ CUtensorMap map_q,
                                                                       const __grid_constant__ CUtensorMap map_k) {
  using S = WeightsShape<D>;
  constexpr int kStages = S::kStages, kTileBytes = S::kTileBytes;
  extern __shared__ __align__(1024) unsigned char pr_raw[];
  const unsigned smem0 = tc_smem(pr_raw);
  const unsigned sKb = smem0, sQb = smem0 + 4 * kTileBytes;
  unsigned* const tmem_base_p = (unsigned*)(pr_raw + S::kTiles);
  volatile int* const abort_flag = (volatile int*)(pr_raw + S::kTiles + 4);
  volatile int* const requested = abort_flag + 1;       // key pairs and query tiles that the TMA warp asked for in all
  const unsigned bars = smem0 + S::kBarOffset;
  const unsigned bar_k = bars /* two items */, bar_kfree = bars + 16, bar_q = bars + 32, bar_qfree = bar_q + 8 * kStages;
  const unsigned bar_s = bar_qfree + 8 * kStages /* [x][buffer] */, bar_f = bar_s + 32 /* [x][buffer] */;
  const unsigned bar_c = bar_f + 32 /* columns described */, bar_cfree = bar_c + 8 * kPwColumns, bar_e = bar_cfree + 8 * kPwColumns;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  follow_stream();
  if (smem0 & 1023u) {
    if (tid == 0) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
    return;
  }
  // One warp each finds the first step of the range and the one behind it, while others set up.
  struct Range {
    StepCursor at;
    long long first, end;
  };
  static_assert(sizeof(Range) <= 96, "between the flags and the barriers");
  Range* const range = (Range*)(pr_raw + S::kRangeOffset);
  if (warp < 2) {
    const long long total = count_steps(P);
    const int ranges = range_count(total, gridDim.x);
    long long step = 0;
    StepCursor c = {};
    const int r = blockIdx.x + warp;
    if (r < ranges) c = range_cursor(P, total, r, ranges, step);
    else step = total;
    if (lane == 0) {
      if (warp == 0) {
        range->at = c;
        range->first = step;
      } else {
        range->end = step;
      }
    }
  } else if (warp == 2) {
    if (lane == 0) {
      *abort_flag = requested[0] = requested[1] = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tc_bar_init(bar_k + 8 * i, 1);
        tc_bar_init(bar_kfree + 8 * i, 1);
      }
#pragma unroll
      for (int i = 0; i < kStages; ++i) {
        tc_bar_init(bar_q + 8 * i, 1);
        tc_bar_init(bar_qfree + 8 * i, 1);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        tc_bar_init(bar_s + 8 * i, 1);
        tc_bar_init(bar_f + 8 * i, 2 * kPrTile);
      }
#pragma unroll
      for (int i = 0; i < kPwColumns; ++i) {
        tc_bar_init(bar_c + 8 * i, 32);
        tc_bar_init(bar_cfree + 8 * i, kPwSoftmaxWarps);
      }
      tc_bar_init(bar_e, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  } else if (warp < kPwSoftmaxWarps) {
    // offsets that the tensors do not hold, and keys of a sequence without queries
    constexpr int kThreads = 32 * (kPwSoftmaxWarps - 3);
    const int t = tid - 96;
    for (int b = blockIdx.x; b < P.n_seq; b += gridDim.x) {
      if (t == 0 && bad_sequence(P, b)) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
      const Sequence s = load_sequence(P, b);
      if (s.nq == 0)
        for (int h = 0; h < P.kv_heads; ++h)
          for (int i = t; i < s.nk; i += kThreads) P.weights[h * P.weights_stride + s.k0 + i] = 0.f;
    }
  } else if (warp == kPwSoftmaxWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_base_p)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_base_p;
  allow_next();
  const int group = P.q_heads / P.kv_heads, heads_per_step = kPrTile / P.width;
  int left = (int)(range->end - range->first);           // steps of this range

  if (warp >= kPwSoftmaxWarps) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPwIssueRegs));
  StepCursor at = range->at;
  if (warp == kPwSoftmaxWarps + 1) {
    // ================================================================ TMA warp
    int pairs = 0, tiles = 0;      // key pairs and query tiles requested so far
    bool go = true;
    while (go && left > 0) {
      const KeySteps k(P, at.s);
      const int kb = pairs & 1, steps = min(left, at.cost - at.step);
      if (pairs >= 2) tc_wait(bar_kfree + 8 * kb, (unsigned)((pairs >> 1) - 1) & 1u, abort_flag);
      if (__any_sync(0xffffffffu, *abort_flag != 0)) break;      // nothing more is asked for; the others run through
      if (lane == 0) {
        requested[0] = pairs + 1;
        pf_expect(bar_k + 8 * kb, 2 * kTileBytes);
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int c = 0; c < S::kSlabs; ++c)
            pf_tma(sKb + (2 * kb + x) * kTileBytes + c * kPrSlab, &map_k, 64 * c, at.s.k0 + at.tile * kPrRows + x * kPrTile, at.kvh, bar_k + 8 * kb);
      }
      ++pairs;
      const int qt0 = k.first(at.tile), per_group = k.tiles - qt0;
      for (int i = 0; i < steps; ++i, ++tiles) {
        const int st = tiles % kStages, step = at.step + i, g = step / per_group, qt = qt0 + step - g * per_group;
        const bool free = tiles < kStages || tc_wait(bar_qfree + 8 * st, (unsigned)(tiles / kStages - 1) & 1u, abort_flag);
        if (__any_sync(0xffffffffu, !free)) {
          go = false;
          break;
        }
        if (lane == 0) {
          requested[1] = tiles + 1;
          const int heads = min(heads_per_step, group - g * heads_per_step);
          pf_expect(bar_q + 8 * st, heads * P.width * 2 * D);
          for (int j = 0; j < heads; ++j)
#pragma unroll
            for (int c = 0; c < S::kSlabs; ++c)
              pf_tma(sQb + st * kTileBytes + c * kPrSlab + j * P.width * 128, &map_q, 64 * c, at.s.q0 + k.w0 + qt * kPrTile,
                     at.kvh * group + g * heads_per_step + j, bar_q + 8 * st);
        }
      }
      left -= steps;
      if (left > 0) next_item(P, at);
    }
  } else if (warp == kPwSoftmaxWarps) {
    // ================================================================ MMA warp
    constexpr bool kBf16 = !std::is_same<QT, __half>::value;
    constexpr unsigned idesc = tc_idesc<kBf16, 128, 128, false>();
    int pairs = 0, step = 0;
    while (left > 0) {
      const int kb = pairs & 1, steps = min(left, at.cost - at.step);
      tc_wait(bar_k + 8 * kb, (unsigned)(pairs >> 1) & 1u, abort_flag);
      ++pairs;
      for (int i = 0; i < steps; ++i, ++step) {
        const int st = step % kStages, buffer = step & 1;
        tc_wait(bar_q + 8 * st, (unsigned)(step / kStages) & 1u, abort_flag);
        for (int x = 0; x < 2; ++x) {
          if (step >= 2) tc_wait(bar_f + 16 * x + 8 * buffer, (unsigned)((step >> 1) - 1) & 1u, abort_flag);
          __syncwarp();
          tc_fence_after();
          if (tc_elect()) {
            const unsigned k = sKb + (2 * kb + x) * kTileBytes, q = sQb + st * kTileBytes;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const unsigned off = (kk >> 2) * kPrSlab + (kk & 3) * 32;
              tc_mma(tmem + 256 * x + 128 * buffer, tc_desc(k + off, 16, 1024), tc_desc(q + off, 16, 1024), idesc, kk > 0);
            }
            tc_commit(bar_s + 16 * x + 8 * buffer);
            if (x == 1) {
              tc_commit(bar_qfree + 8 * st);
              if (i + 1 == steps) tc_commit(bar_kfree + 8 * kb);
            }
          }
          __syncwarp();
        }
      }
      left -= steps;
      if (left > 0) next_item(P, at);
    }
    // the CTA does not leave before the last commits have arrived
    if (step > 0) {
      tc_wait(bar_qfree + 8 * ((step - 1) % kStages), (unsigned)((step - 1) / kStages) & 1u, abort_flag);
      tc_wait(bar_kfree + 8 * ((pairs - 1) & 1), (unsigned)((pairs - 1) >> 1) & 1u, abort_flag);
    }
  } else if (warp == kPwSoftmaxWarps + 2) {
    // ================================================================ describes the columns, four to a lane
    const int width = P.width, column = 4 * lane, column_head = column / width, column_q = column & (width - 1);
    int step = 0;
    while (left > 0) {
      const KeySteps k(P, at.s);
      const int steps = min(left, at.cost - at.step), qt0 = k.first(at.tile), per_group = k.tiles - qt0, hist = at.s.nk - k.nw;
      int g = at.step / per_group, qt = qt0 + at.step - g * per_group;
      for (int i = 0; i < steps; ++i, ++step) {
        const int c = step % kPwColumns, head = g * heads_per_step + column_head, q = qt * kPrTile + column_q;
        const float* const lse = P.lse + (long long)(at.kvh * group + head) * P.lse_stride + at.s.q0 + k.w0 + q;
        float l[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // a column without a query, or of one without a key, weighs nothing: -infinity in the place of its exponent
          const float x = head < group && q + j < k.nw ? __ldg(lse + j) : __int_as_float(0xff800000);
          l[j] = x == __int_as_float(0xff800000) ? x : -kLog2e * x;
        }
        if (step >= kPwColumns) tc_wait(bar_cfree + 8 * c, (unsigned)(step / kPwColumns - 1) & 1u, abort_flag);
        __syncwarp();
        unsigned char* const to = pr_raw + S::kColumnsOffset + c * kPwColumnBytes;
        *(float4*)(to + 4 * column) = make_float4(l[0], l[1], l[2], l[3]);
        if (lane == 0) {
          StepNote* const note = (StepNote*)(to + 4 * kPrTile);
          note->lo = at.tile * kPrRows - (hist + qt * kPrTile);
          note->hi = k.nw - qt * kPrTile;
          note->columns = min(group - g * heads_per_step, heads_per_step) * width;
          note->last = i + 1 == steps;
          note->cut = steps < at.cost;
          note->keys = note->cut ? kPrRows : at.s.nk - at.tile * kPrRows;
          // of a cut item: the range that it begins in, and the ranges behind it
          note->at = note->cut ? ((long long)blockIdx.x * 2 + (at.step == 0)) * kPrRows : at.kvh * P.weights_stride + at.s.k0 + at.tile * kPrRows;
        }
        pf_arrive(bar_c + 8 * c);
        if (++qt == k.tiles) {
          qt = qt0;
          ++g;
        }
      }
      left -= steps;
      if (left > 0) next_item(P, at);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPwSoftmaxRegs));
    // ================================================================ two threads per key row, 64 columns each
    const int x = (warp >> 2) & 1, half = warp >> 3, row = tid & (kPrTile - 1), width = P.width;
    float* const second = (float*)(pr_raw + S::kSumOffset) + x * kPrTile + row;
    const unsigned tS = tmem + ((unsigned)((warp & 3) * 32) << 16) + 256 * x;
    const unsigned long long scale2 = pf_pair(P.scale_log2e, P.scale_log2e);
    float sum = 0.f;
    for (int step = 0; step < left; ++step) {
      const int buffer = step & 1, described = step % kPwColumns;
      const unsigned char* const about = pr_raw + S::kColumnsOffset + described * kPwColumnBytes;
      const float* const exponents = (const float*)about;
      const StepNote* const note = (const StepNote*)(about + 4 * kPrTile);
      tc_wait(bar_c + 8 * described, (unsigned)(step / kPwColumns) & 1u, abort_flag);
      const int lo = note->lo + x * kPrTile + row, hi = note->hi, columns = note->columns;
      // the last key of the tile is not seen by the first query, or a column stands for no query
      const bool masked = note->lo + x * kPrTile + kPrTile - 1 > 0 || hi < width || columns < kPrTile;
      tc_wait(bar_s + 16 * x + 8 * buffer, (unsigned)(step >> 1) & 1u, abort_flag);
      __syncwarp();
      tc_fence_after();
      unsigned v[2][32];
      tc_ld32(tS + 128 * buffer + 64 * half, v[0]);
      tc_ld32(tS + 128 * buffer + 64 * half + 32, v[1]);
      tc_wait_ld32(v[0]);
      tc_wait_ld32(v[1]);
      tc_fence_before();
      pf_arrive(bar_f + 16 * x + 8 * buffer);
      unsigned long long sums[2] = {pf_pair(0.f, 0.f), pf_pair(0.f, 0.f)};
      // Columns 32 q .. 32 q + 31 of this half; bit c of `seen`: column 32 q + c counts.  (A polynomial on the FMA units in the
      // place of a quarter or three eighths of the exponentials changed nothing, with eight softmax warps: 87 to 90 us for
      // 4096 tokens either way.)
      auto add = [&](int q, auto some, unsigned seen) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 l4 = *(const float4*)(exponents + 64 * half + 32 * q + c);
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int i = c + 2 * p;
            const unsigned long long e2 = pf_fma2(pf_pair(__uint_as_float(v[q][i]), __uint_as_float(v[q][i + 1])), scale2,
                                                  p ? pf_pair(l4.z, l4.w) : pf_pair(l4.x, l4.y));
            float e0, e1;
            pf_unpair(e2, e0, e1);
            e0 = pf_exp2(e0);
            e1 = pf_exp2(e1);
            if (decltype(some)::value) {      // whatever a column that does not count holds
              e0 = seen & (1u << i) ? e0 : 0.f;
              e1 = seen & (2u << i) ? e1 : 0.f;
            }
            sums[p] = pf_add2(sums[p], pf_pair(e0, e1));
          }
        }
      };
      if (!masked) {
#pragma unroll
        for (int q = 0; q < 2; ++q) add(q, std::false_type{}, 0u);
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int column = 64 * half + 32 * q;
          if (column < columns) {
            // columns of queries lo .. hi - 1 of a window, of one head, of half a window, or of two heads
            const int base = column & (width - 1), from = min(max(lo - base, 0), 32), to = min(max(hi - base, 0), 32);
            unsigned seen = (unsigned)((1ull << to) - 1ull) & ~(unsigned)((1ull << from) - 1ull);
            if (width == 16) seen = (seen & 0xffffu) | (column + 16 < columns ? seen << 16 : 0u);
            if (__any_sync(0xffffffffu, seen != 0u)) add(q, std::true_type{}, seen);
          }
        }
      }
      float even, odd;
      pf_unpair(pf_add2(sums[0], sums[1]), even, odd);
      sum += even + odd;
      if (note->last) {
        // the halves' sums, always in this order; the second barrier frees the place
        if (half) *second = sum;
        asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");
        if (!half && x * kPrTile + row < note->keys && *abort_flag == 0)
          (note->cut ? P.records : P.weights)[note->at + x * kPrTile + row] = sum + *second;
        asm volatile("bar.sync %0, 256;" ::"r"(1 + x) : "memory");
        sum = 0.f;
      }
      __syncwarp();
      if (lane == 0) pf_arrive(bar_cfree + 8 * described);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(P.status, INQ_STATUS_WAIT_TIMEOUT);
  if (warp == kPwSoftmaxWarps) {
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {
      if (tc_elect()) tc_commit(bar_e);
      tc_drain(bar_e, 0);
#pragma unroll 1
      for (int back = 2; back > 0; --back)
        if (requested[0] >= back) tc_drain(bar_k + 8 * ((requested[0] - back) & 1), (unsigned)((requested[0] - back) >> 1) & 1u);
#pragma unroll 1
      for (int back = kStages; back > 0; --back)
        if (requested[1] >= back)
          tc_drain(bar_q + 8 * ((requested[1] - back) % kStages), (unsigned)((requested[1] - back) / kStages) & 1u);
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Adds the parts of the items that ranges cut, in their order: block r takes the item that is cut where range r ends, if
// it begins in range r.
__global__ void __launch_bounds__(kPrRows) prompt_weights_sum_kernel(const PromptParams P, int ctas) {
  follow_stream();
  const long long total = count_steps(P);
  const int ranges = range_count(total, ctas), r = blockIdx.x;
  if (r + 1 >= ranges) return;
  const long long cut = range_start(total, r + 1, ranges);
  const StepCursor c = seek_step(P, cut);
  if (c.step == 0 || c.cost <= kPwWhole || range_of(total, cut - c.step, ranges) != r) return;
  const int last = range_of(total, cut - c.step + c.cost - 1, ranges);
  float sum = __ldcg(P.records + (2LL * r + 1) * kPrRows + threadIdx.x);
  for (int i = r + 1; i <= last; ++i) sum += __ldcg(P.records + 2LL * i * kPrRows + threadIdx.x);
  const int key = c.tile * kPrRows + threadIdx.x;
  if (key < c.s.nk) P.weights[c.kvh * P.weights_stride + c.s.k0 + key] = sum;
}

}  // namespace inq

using namespace inq;

namespace {
// The shares that setmaxnreg hands out must not exceed what the kernel is launched with (as in csrc/prefill.cu).
int prompt_registers_fit(const void* kernel, int launched) {
  cudaFuncAttributes attributes;
  INQ_CUDA_CHECK(cudaFuncGetAttributes(&attributes, kernel));
  return attributes.numRegs < launched ? INQ_ERR_UNSUPPORTED : INQ_OK;
}
int check_args(const inq_prompt_args_t* a) {
  if (!a || !a->q || !a->k || !a->cu_q || !a->cu_k || !a->status) return INQ_ERR_ARGUMENT;
  if (a->q_heads < 1 || a->kv_heads < 1 || a->q_heads % a->kv_heads || a->n_seq < 1) return INQ_ERR_ARGUMENT;
  if (a->q_rows < 1 || a->k_rows < 1 || !(a->scale > 0.f)) return INQ_ERR_ARGUMENT;
  if (a->q_rows > 0x3fffffff || a->k_rows > 0x3fffffff) return INQ_ERR_CAPACITY;
  if (a->dtype != INQ_F16 && a->dtype != INQ_BF16) return INQ_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return INQ_ERR_UNSUPPORTED;
  // rows are read and written as 16-byte vectors
  if ((a->q_stride_t | a->k_stride_t | a->q_stride_h | a->k_stride_h) & 7) return INQ_ERR_ARGUMENT;
  if (((uintptr_t)a->q | (uintptr_t)a->k) & 15) return INQ_ERR_ARGUMENT;
  if (a->q_stride_h <= 0 || a->k_stride_h <= 0 || a->q_stride_t <= 0 || a->k_stride_t <= 0) return INQ_ERR_ARGUMENT;
  return INQ_OK;
}
PromptParams base_params(const inq_prompt_args_t* a) {
  PromptParams P = {};
  P.cu_q = a->cu_q; P.cu_k = a->cu_k;
  P.n_seq = a->n_seq; P.q_rows = (int)a->q_rows; P.k_rows = (int)a->k_rows;
  P.q_heads = a->q_heads; P.kv_heads = a->kv_heads;
  P.scale_log2e = a->scale * kLog2e;
  P.status = a->status;
  P.records = (float*)a->workspace;
  return P;
}
int sm_count(int* n) {
  int device = 0;   // asked per call: the answer belongs to the current device
  INQ_CUDA_CHECK(cudaGetDevice(&device));
  INQ_CUDA_CHECK(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device));
  return INQ_OK;
}
// Items that `rows` rows of `n_seq` sequences make at most.
long long most_tiles(long long rows, int n_seq) { return rows / kPrRows + std::min<long long>(rows, n_seq); }

// Whether the kernel may find that cutting items pays (see Deal): not where even the dearest item that the tensors allow costs
// no more than a cut, nor where the items are many rounds of whole ones.
bool attention_may_cut(int q_heads, long long q_rows, long long k_rows, int n_seq, int n_sm) {
  const long long least = std::max<long long>(1, q_rows / kPrRows) * q_heads;
  return k_rows > 8 * kPrTile && least < 3LL * n_sm;
}
// Columns of a step per query head: windows of at most 64 queries lie side by side, as many as the group has heads for.
int weights_width(int group, int window) {
  int width = kPrTile;
  while (window > 0 && width > 16 && window <= width / 2 && kPrTile / width < group) width /= 2;
  return width;
}
// Whether an item of inq_prompt_weights may be cut.
bool weights_cut(int group, long long q_rows, int window) {
  const int width = weights_width(group, window);
  const long long tiles = (std::min<long long>(q_rows, window > 0 ? window : q_rows) + kPrTile - 1) / kPrTile;
  return tiles * ((group * width + kPrTile - 1) / kPrTile) > kPwWhole;
}
long long attention_record_bytes(int head_dim, int n_sm) {
  return n_sm * (2LL * kPrRows * (head_dim + 2) * (long long)sizeof(float) + (long long)sizeof(CutItem));
}

template <typename QT, int D>
int launch_attention(const PromptParams& P, unsigned ctas, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v) {
  const int fit = prompt_registers_fit((const void*)prompt_kernel<QT, D>, kPrLaunchRegs);
  if (fit != INQ_OK) return fit;
  INQ_CUDA_CHECK(cudaFuncSetAttribute(prompt_kernel<QT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<D>::kSmem));
  INQ_CUDA_CHECK(launch_following(prompt_kernel<QT, D>, ctas, kPrThreads, PromptShape<D>::kSmem, stream, P, q, k, v));
  if (P.records) INQ_CUDA_CHECK(launch_following(prompt_merge_kernel<QT, D>, dim3(ctas, kPrRows / kPrMergeRows), 256, 0, stream, P));
  return INQ_OK;
}
template <typename QT, int D>
int launch_weights(const PromptParams& P, unsigned ctas, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& k) {
  const int fit = prompt_registers_fit((const void*)prompt_weights_kernel<QT, D>, kPwLaunchRegs);
  if (fit != INQ_OK) return fit;
  INQ_CUDA_CHECK(cudaFuncSetAttribute(prompt_weights_kernel<QT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightsShape<D>::kSmem));
  INQ_CUDA_CHECK(launch_following(prompt_weights_kernel<QT, D>, ctas, kPwThreads, WeightsShape<D>::kSmem, stream, P, q, k));
  if (P.records) INQ_CUDA_CHECK(launch_following(prompt_weights_sum_kernel, ctas, kPrRows, 0, stream, P, (int)ctas));
  return INQ_OK;
}
}  // namespace

extern "C" int64_t inq_prompt_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int64_t q_rows, int64_t k_rows,
                                              int32_t n_seq, int32_t weights, int32_t window) {
  int n_sm = 0;
  if (q_heads < 1 || kv_heads < 1 || n_seq < 1 || q_rows < 0 || k_rows < 0 || sm_count(&n_sm) != INQ_OK) return 0;
  return weights ? weights_cut(q_heads / kv_heads, q_rows, window) ? 2LL * n_sm * kPrRows * (int64_t)sizeof(float) : 0
                 : attention_may_cut(q_heads, q_rows, k_rows, n_seq, n_sm) ? attention_record_bytes(head_dim, n_sm) : 0;
}

extern "C" int inq_prompt_attention(const inq_prompt_args_t* a, inq_stream_t stream_) {
  const int rc = check_args(a);
  if (rc != INQ_OK) return rc;
  if (!a->v || !a->out || ((uintptr_t)a->v & 15) || ((uintptr_t)a->out & 15)) return INQ_ERR_ARGUMENT;
  if (((a->v_stride_t | a->v_stride_h | a->o_stride_t | a->o_stride_h) & 7) || a->v_stride_h <= 0 || a->v_stride_t <= 0) return INQ_ERR_ARGUMENT;
  PromptParams P = base_params(a);
  P.out = a->out; P.lse = a->lse;
  P.o_sh = a->o_stride_h; P.o_st = a->o_stride_t; P.lse_stride = a->lse_stride;
  int n_sm = 0;
  const int sm_rc = sm_count(&n_sm);
  if (sm_rc != INQ_OK) return sm_rc;
  if (!attention_may_cut(a->q_heads, a->q_rows, a->k_rows, a->n_seq, n_sm) || !a->workspace ||
      a->workspace_bytes < attention_record_bytes(a->head_dim, n_sm))
    P.records = nullptr;
  P.cuts = P.records ? (CutItem*)(P.records + 2LL * n_sm * kPrRows * (a->head_dim + 2)) : nullptr;
  CUtensorMap map_q, map_k, map_v;
  if (!make_map(&map_q, a->q, a->dtype, a->head_dim, a->q_rows, a->q_heads, a->q_stride_t, a->q_stride_h, kPrTile) ||
      !make_map(&map_k, a->k, a->dtype, a->head_dim, a->k_rows, a->kv_heads, a->k_stride_t, a->k_stride_h, kPrTile) ||
      !make_map(&map_v, a->v, a->dtype, a->head_dim, a->k_rows, a->kv_heads, a->v_stride_t, a->v_stride_h, kPrTile))
    return INQ_ERR_ARGUMENT;
  const unsigned ctas = (unsigned)(P.records ? n_sm : std::min<long long>(n_sm, most_tiles(a->q_rows, a->n_seq) * a->q_heads));
  cudaStream_t stream = (cudaStream_t)stream_;
  if (a->dtype == INQ_F16)
    return a->head_dim == 64 ? launch_attention<__half, 64>(P, ctas, stream, map_q, map_k, map_v)
                             : launch_attention<__half, 128>(P, ctas, stream, map_q, map_k, map_v);
  return a->head_dim == 64 ? launch_attention<__nv_bfloat16, 64>(P, ctas, stream, map_q, map_k, map_v)
                           : launch_attention<__nv_bfloat16, 128>(P, ctas, stream, map_q, map_k, map_v);
}

extern "C" int inq_prompt_weights(const inq_prompt_args_t* a, inq_stream_t stream_) {
  const int rc = check_args(a);
  if (rc != INQ_OK) return rc;
  if (!a->lse || !a->weights || a->window < 0) return INQ_ERR_ARGUMENT;
  PromptParams P = base_params(a);
  P.lse = a->lse; P.lse_stride = a->lse_stride;
  P.weights = a->weights; P.weights_stride = a->weights_stride;
  P.window = a->window;
  int n_sm = 0;
  const int sm_rc = sm_count(&n_sm);
  if (sm_rc != INQ_OK) return sm_rc;
  P.width = weights_width(a->q_heads / a->kv_heads, a->window);
  if (!weights_cut(a->q_heads / a->kv_heads, a->q_rows, a->window)) P.records = nullptr;
  else if (!a->workspace || a->workspace_bytes < 2LL * n_sm * kPrRows * (long long)sizeof(float)) return INQ_ERR_CAPACITY;
  CUtensorMap map_q, map_k;
  if (!make_map(&map_q, a->q, a->dtype, a->head_dim, a->q_rows, a->q_heads, a->q_stride_t, a->q_stride_h, P.width) ||
      !make_map(&map_k, a->k, a->dtype, a->head_dim, a->k_rows, a->kv_heads, a->k_stride_t, a->k_stride_h, kPrTile))
    return INQ_ERR_ARGUMENT;
  const unsigned ctas = (unsigned)n_sm;
  cudaStream_t stream = (cudaStream_t)stream_;
  if (a->dtype == INQ_F16)
    return a->head_dim == 64 ? launch_weights<__half, 64>(P, ctas, stream, map_q, map_k) : launch_weights<__half, 128>(P, ctas, stream, map_q, map_k);
  return a->head_dim == 64 ? launch_weights<__nv_bfloat16, 64>(P, ctas, stream, map_q, map_k)
                           : launch_weights<__nv_bfloat16, 128>(P, ctas, stream, map_q, map_k);
}
