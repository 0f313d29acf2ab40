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
//   * an item (256 query rows of one head) finds its sequence by its rank in the order of falling cost, so
//     that the longest items start first whatever the mix of lengths (find_item);
//   * two more warps clean the value tiles that hold rows some query must not see.  The contraction multiplies
//     such rows by probability zero, which is no help against infinities and NaN: rows behind the sequence (those
//     of its neighbour, or memory that nothing has written) are set to zero, non-finite values at the positions that
//     only later queries see are set to zero and put back, by position, into the rows that do see them.
//
// prompt_weights_kernel.  w_j = sum over the group's heads and the last `window` queries of 2^(s_ij - lse_i).  The
// contraction is transposed, S^T = K Q^T: a thread owns a KEY row and adds over columns, so that a sum never
// leaves its thread and no atomics order it.
#include <algorithm>

#include "attention.cuh"

namespace inq {

constexpr int kPrThreads = 384;              // 8 softmax warps, the MMA warp, the TMA warp, two that clean value tiles
constexpr int kPrLaunchRegs = 168, kPrIssueRegs = 72, kPrSoftmaxRegs = (3 * kPrLaunchRegs - kPrIssueRegs) / 2;
constexpr int kPrTile = 128;                 // rows per tile
constexpr int kPrRows = 2 * kPrTile;         // rows per item (tiles A and B)
constexpr int kPrSlab = kPrTile * 128;       // 128 rows x 128 bytes
constexpr float kPrNegBig = -3.0e38f;        // stands for the maximum of nothing: below every finite logit that matters
constexpr float kPrSlack = 8.f;              // the reference maximum may lag the true one by 2^8
constexpr int kPrMaxSplits = 8;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct PromptParams {
  void* out;
  float* lse;                       // attention: written, weights: read; [q_heads][lse_stride]
  float* weights;                   // [kv_heads][weights_stride]
  long long o_sh, o_st, lse_stride, weights_stride;
  const int *cu_q, *cu_k;
  int n_seq, q_rows, k_rows, q_heads, kv_heads;
  int splits;
  int window;                       // weights: queries per sequence that count, 0 = all
  int width;                        // weights: columns of a step per query head
  float* records;                   // partial results of cut items
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
// every turn.  Returns the sequence, or -1 where there are fewer items.
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
  int lo = 0, hi = max_cost + 1;      // count(lo) > rank >= count(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) > rank) lo = mid;
    else hi = mid;
  }
  int left = rank - count(lo + 1);
  for (int b0 = 0; b0 < P.n_seq; b0 += 32) {
    const Sequence s = b0 == 0 ? mine : b0 + lane < P.n_seq ? load_sequence(P, b0 + lane) : Sequence{0, 0, 0, 0};
    const int ge = items_at_least(s, lo), equal = ge - items_at_least(s, lo + 1);
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

template <int D>
struct PromptShape {
  static constexpr int kSlabs = D / 64;                       // column slabs of an operand tile
  static constexpr int kTileBytes = kSlabs * kPrSlab;
  static constexpr int kStages = D == 128 ? 2 : 4;            // K and V tiles in flight
  static constexpr int kTiles = (2 + 2 * kStages) * kTileBytes;
  static constexpr int kBars = 2 + 4 * kStages + 8;
  // then: TMEM base, abort flag, two request counts, the item (8 words), a flag, barriers, three lists of D positions
  static constexpr int kBarOffset = kTiles + 64, kListOffset = kBarOffset + 8 * kBars;
  static constexpr int kSmem = kListOffset + 3 * D * 4;
};

constexpr int kFar = 0x7fffffff;
// positions of the first +infinity, -infinity and NaN of each channel among the cleaned values
enum { kBadPlus = 0, kBadMinus = 1, kBadNan = 2 };

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
  volatile int* const requested = abort_flag + 1;             // K and V tiles that the TMA warp asked for in all
  volatile int* const item_p = abort_flag + 3;                // found, index, q0, nq, k0, nk
  volatile int* const any_bad = abort_flag + 10;
  int* const first_bad = (int*)(pr_raw + S::kListOffset);     // [3][D]
  const unsigned bars = smem0 + S::kBarOffset;
  // per stage: K and V tiles, V tiles that want cleaning, such tiles cleaned
  const unsigned bar_q = bars, bar_e = bars + 8, bar_k = bars + 16, bar_v = bar_k + 8 * kStages, bar_d = bar_v + 8 * kStages;
  const unsigned bar_c = bar_d + 8 * kStages, bar_s = bar_c + 8 * kStages /* A, B */, bar_p = bar_s + 16 /* A, B */, bar_o = bar_p + 16, bar_h = bar_o + 16;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  follow_stream();       // cu_q and cu_k may come from the launch before this one
  if (smem0 & 1023u) {
    if (tid == 0) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
    return;
  }
  const int unit = (int)(blockIdx.x / P.splits), seg = (int)(blockIdx.x % P.splits);
  const int head = unit % P.q_heads;
  if (warp == 8) {
    Sequence s;
    int index = 0;
    const int b = find_item(P, unit / P.q_heads, (P.k_rows + kPrTile - 1) / kPrTile, s, index);
    if (lane == 0) {
      item_p[0] = b;
      item_p[1] = index;
      item_p[2] = s.q0;
      item_p[3] = s.nq;
      item_p[4] = s.k0;
      item_p[5] = s.nk;
    }
  } else if (warp == 9 && lane == 0) {
    *abort_flag = requested[0] = requested[1] = 0;
    *any_bad = 0;
    tc_bar_init(bar_q, 1);
    tc_bar_init(bar_e, 1);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      tc_bar_init(bar_k + 8 * i, 1);
      tc_bar_init(bar_v + 8 * i, 1);
      tc_bar_init(bar_d + 8 * i, 1);
      tc_bar_init(bar_c + 8 * i, 2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      tc_bar_init(bar_s + 8 * i, 1);
      tc_bar_init(bar_p + 8 * i, kPrTile);
      tc_bar_init(bar_o + 8 * i, 1);
      tc_bar_init(bar_h + 8 * i, kPrTile);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int i = tid; i < 3 * D; i += kPrThreads) first_bad[i] = kFar;
  if (blockIdx.x == 0)
    for (int b = tid; b < P.n_seq; b += kPrThreads)
      if (bad_sequence(P, b)) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
  __syncthreads();
  if (item_p[0] < 0) return;       // fewer items than the sizes of the tensors allow
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc_smem(tmem_base_p)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const unsigned tmem = *tmem_base_p;      // S_A 0..127, S_B 128..255 (P over their first 64), O_A 256.., O_B 384..
  allow_next();
  auto wait = [&](unsigned mbar, unsigned parity) { tc_wait(mbar, parity, abort_flag); };   // goes on in either case

  const int kvh = head / (P.q_heads / P.kv_heads);
  const int q0 = item_p[1] * kPrRows, q_base = item_p[2], nq = item_p[3], k_base = item_p[4], nk = item_p[5];
  const int hist = nk - nq;       // negative where the first queries have no key at all
  // tiles that A and B walk; B may hold no query at all, and a tile no key
  const int all_a = (max(min(nk, hist + q0 + kPrTile), 0) + kPrTile - 1) / kPrTile;
  const int all_b = q0 + kPrTile < nq ? (max(min(nk, hist + q0 + kPrRows), 0) + kPrTile - 1) / kPrTile : 0;
  const int all = max(all_a, all_b);
  const int t_lo = (int)((long long)all * seg / P.splits), t_hi = (int)((long long)all * (seg + 1) / P.splits);
  const int n_t = t_hi - t_lo;
  const int n_a = max(0, min(all_a, t_hi) - t_lo), n_b = max(0, min(all_b, t_hi) - t_lo);
  const int last = n_b > 0 ? 1 : 0;      // the tile that takes part in every step
  // Tiles from t_dark on hold rows that some query of this item must not see.  Their values arrive at barriers of
  // their own: the warps that clean them look at no earlier tile, and a parity alone does not tell phases apart.
  const int t_dark = max(0, (max(hist + q0 + 1, 0) >> 7) - t_lo);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrIssueRegs));
    if (warp == 9) {
      // ================================================================ TMA warp
      if (lane == 0 && n_t > 0) {
        auto request = [&](int what, int t) {
          requested[what] = t + 1;
          const unsigned bar = (what == 0 ? bar_k : t < t_dark ? bar_v : bar_d) + 8 * (t % kStages), dst = (what ? sVb : sKb) + (t % kStages) * kTileBytes;
          pf_expect(bar, kTileBytes);
#pragma unroll
          for (int c = 0; c < S::kSlabs; ++c)
            pf_tma(dst + c * kPrSlab, what ? &map_v : &map_k, 64 * c, k_base + (t_lo + t) * kPrTile, kvh, bar);
        };
        pf_expect(bar_q, 2 * kTileBytes);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int c = 0; c < S::kSlabs; ++c)
            pf_tma(sQ + x * kTileBytes + c * kPrSlab, &map_q, 64 * c, q_base + q0 + x * kPrTile, head, bar_q);
        for (int t = 0; t < kStages && t < n_t; ++t) {
          request(0, t);
          request(1, t);
        }
        for (int t = 0; t + kStages < n_t; ++t) {
          // K(t) is free once the last score contraction of step t is done, V(t) once the last output contraction is
          if (!tc_wait(bar_s + 8 * last, (unsigned)t & 1u, abort_flag)) break;
          request(0, t + kStages);
          if (!tc_wait(bar_o + 8 * last, (unsigned)t & 1u, abort_flag)) break;
          request(1, t + kStages);
        }
      }
    } else if (warp == 8) {
      // ================================================================ MMA warp
      if (n_t > 0) {
        constexpr bool kBf16 = !std::is_same<QT, __half>::value;
        constexpr unsigned idesc_s = tc_idesc<kBf16, 128, 128, false>(), idesc_o = tc_idesc<kBf16, 128, D, true>();
        auto issue_s = [&](int x, int t) {      // S_x = Q_x K(t)^T
          const unsigned q = sQ + x * kTileBytes, k = sKb + (t % kStages) * kTileBytes;
          if (tc_elect()) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const unsigned off = (kk >> 2) * kPrSlab + (kk & 3) * 32;
              tc_mma(tmem + x * kPrTile, tc_desc(q + off, 16, 1024), tc_desc(k + off, 16, 1024), idesc_s, kk > 0);
            }
            tc_commit(bar_s + 8 * x);
          }
        };
        auto issue_o = [&](int x, int t, int half) {      // O_x += P_x V(t), half a tile of tokens at a time
          const unsigned v = sVb + (t % kStages) * kTileBytes;
          if (tc_elect()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int kk = 4 * half + k;
              tc_mma_ta(tmem + 2 * kPrTile + x * kPrTile, tmem + x * kPrTile + kk * 8, tc_desc(v + kk * 2048, kPrSlab, 1024), idesc_o,
                        (t > 0 || kk > 0) ? 1u : 0u);
            }
            if (half) tc_commit(bar_o + 8 * x);
          }
        };
        auto contract_o = [&](int x, int t) {
          wait(bar_h + 8 * x, (unsigned)t & 1u);     // S_x(t) read, the first half of P_x(t) written
          tc_fence_after();
          issue_o(x, t, 0);
          wait(bar_p + 8 * x, (unsigned)t & 1u);     // the second half
          tc_fence_after();
          issue_o(x, t, 1);
        };
        wait(bar_q, 0);
        wait(bar_k, 0);
        tc_fence_after();
        if (n_a > 0) issue_s(0, 0);
        if (n_b > 0) issue_s(1, 0);
        for (int t = 0; t < n_t; ++t) {
          if (t < t_dark) wait(bar_v + 8 * (t % kStages), (unsigned)(t / kStages) & 1u);
          else wait(bar_c + 8 * (t % kStages), (unsigned)((t - t_dark) / kStages) & 1u);
          if (t < n_a) contract_o(0, t);
          if (t + 1 < n_t) {
            wait(bar_k + 8 * ((t + 1) % kStages), (unsigned)((t + 1) / kStages) & 1u);
            if (t + 1 < n_a) issue_s(0, t + 1);
          }
          if (t < n_b) contract_o(1, t);
          if (t + 1 < n_b) issue_s(1, t + 1);
        }
      }
    } else {
      // ================================================================ two warps that clean value tiles
      // a lane owns two chunks of 16 bytes per slab and row group; chunk c of row r lies at chunk c ^ (r & 7)
      for (int t = t_dark; t < n_t; ++t) {
        wait(bar_d + 8 * (t % kStages), (unsigned)((t - t_dark) / kStages) & 1u);
        unsigned char* const tile = pr_raw + (sVb - smem0) + (t % kStages) * kTileBytes;
        const int kv0 = (t_lo + t) * kPrTile, rows = min(nk - kv0, kPrTile);     // rows of the sequence
        const int first = (warp - 10) * 32 + lane;
        bool touched = false;
#pragma unroll 1
        for (int i0 = first; i0 < kTileBytes / 16; i0 += 64 * 8) {
          uint4 w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = *(const uint4*)(tile + 16 * (i0 + 64 * j));
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int i = i0 + 64 * j, row = (i >> 3) & (kPrTile - 1);
            if (row >= rows) {
              *(uint4*)(tile + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
              touched = true;
              continue;
            }
            // all ones in the exponent of either half of a word: the mask of the type, compared half by half
            constexpr unsigned kOnes = std::is_same<QT, __half>::value ? 0x7c007c00u : 0x7f807f80u;
            const unsigned words[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const unsigned e = ~words[k] & kOnes;
              bad |= (e & 0xffffu) == 0u || (e >> 16) == 0u;
            }
            if (bad) {
              const int channel = (i / (kPrTile * 8)) * 64 + (((i & 7) ^ (row & 7)) << 3);
              unsigned clean[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                clean[k] = words[k];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const unsigned bits = (words[k] >> (16 * half)) & 0xffffu;
                  if ((~bits & (kOnes & 0xffffu)) == 0u) {
                    const int kind = (bits & ~kOnes & 0x7fffu) ? kBadNan : (bits & 0x8000u) ? kBadMinus : kBadPlus;
                    atomicMin(first_bad + kind * D + channel + 2 * k + half, kv0 + row);
                    clean[k] &= ~(0xffffu << (16 * half));
                  }
                }
              }
              *(uint4*)(tile + 16 * i) = make_uint4(clean[0], clean[1], clean[2], clean[3]);
              *any_bad = 1;
              touched = true;
            }
          }
        }
        if (touched) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) pf_arrive(bar_c + 8 * (t % kStages));
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrSoftmaxRegs));
    // ================================================================ softmax warps
    const int x = warp >> 2;                       // 0: tile A, 1: tile B
    const int row = tid & (kPrTile - 1);           // query row inside the tile = TMEM lane
    const int n_x = x ? n_b : n_a;
    const int q_row = q0 + x * kPrTile + row;
    const int q_pos = hist + q_row;                // keys at positions <= q_pos are visible
    const int diag0 = hist + q0 + x * kPrTile;     // first row's diagonal: tiles reaching beyond it need masks
    const unsigned lane_field = (unsigned)((warp & 3) * 32) << 16;
    const unsigned tS = tmem + lane_field + x * kPrTile, tO = tmem + lane_field + 2 * kPrTile + x * kPrTile;
    const unsigned my_s = bar_s + 8 * x, my_p = bar_p + 8 * x, my_o = bar_o + 8 * x;
    float m_ref = kPrNegBig, l_sum = 0.f;

    for (int t = 0; t < n_x; ++t) {
      const int kv0 = (t_lo + t) * kPrTile;
      // S(t) is complete; the contractions run in issue order, so PV(t-1) is complete as well:
      // the columns of P may be overwritten by S and O may be rescaled
      wait(my_s, (unsigned)t & 1u);
      tc_fence_after();
      unsigned v[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tc_ld32(tS + 32 * q, v[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) tc_wait_ld32(v[q]);
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
        tc_st16(tS + 16 * q, packed);
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
    if (n_x > 0) wait(my_o, (unsigned)(n_x - 1) & 1u);
    tc_fence_after();
    const bool ok = *abort_flag == 0;
    const bool live = ok && q_row < nq;
    const bool bad = *any_bad != 0;     // complete: the last contraction came after the last cleaned tile
    // What cleaning took out, for the rows that see it: the sum of a NaN or of infinities of both signs is NaN.
    auto put_back = [&](float o, int channel) {
      const bool plus = first_bad[kBadPlus * D + channel] <= q_pos, minus = first_bad[kBadMinus * D + channel] <= q_pos;
      if (first_bad[kBadNan * D + channel] <= q_pos || (plus && minus)) return __int_as_float(0x7fc00000);
      return plus ? o + __int_as_float(0x7f800000) : minus ? o + __int_as_float(0xff800000) : o;
    };

    if (P.splits == 1) {
      // a row without keys gives zeros; one whose logits are all -infinity divides zero by zero, as its formula does
      const float inv = q_pos < 0 ? 0.f : 1.f / l_sum;
      if (live && P.lse) P.lse[head * P.lse_stride + q_base + q_row] = q_pos < 0 ? __int_as_float(0xff800000) : (m_ref + log2f(l_sum)) * kLn2;
      QT* orow = (QT*)P.out + (long long)head * P.o_sh + (long long)(q_base + q_row) * P.o_st;
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
      float* rec = P.records + (((long long)unit * P.splits + seg) * kPrRows + x * kPrTile + row) * (D + 2);
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
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(P.status, INQ_STATUS_WAIT_TIMEOUT);
  if (warp == 8) {
    __syncwarp();
    if (__any_sync(0xffffffffu, *abort_flag != 0)) {
      // contractions and copies may be in flight: they end before tensor memory is freed and the CTA leaves
      if (tc_elect()) tc_commit(bar_e);
      tc_drain(bar_e, 0);
      if (requested[1] > 0) tc_drain(bar_q, 0);
#pragma unroll 1
      for (int back = kStages; back > 0; --back) {
        const int k = requested[0] - back, v = requested[1] - back;
        if (k >= 0) tc_drain(bar_k + 8 * (k % kStages), (unsigned)(k / kStages) & 1u);
        if (v >= t_dark) tc_drain(bar_d + 8 * (v % kStages), (unsigned)((v - t_dark) / kStages) & 1u);
        else if (v >= 0) tc_drain(bar_v + 8 * (v % kStages), (unsigned)(v / kStages) & 1u);
      }
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the KV segments of every item: out = sum_s O_s 2^(m_s - m) / sum_s l_s 2^(m_s - m).  A block takes 64 rows of
// an item, a warp eight of them in turn, a lane D / 32 neighbouring channels; the loads of all segments of a row are
// issued before the first is used.
constexpr int kPrMergeRows = 64;
template <typename QT, int D>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const PromptParams P) {
  follow_stream();
  const int unit = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = unit % P.q_heads;
  Sequence s;
  int index = 0;
  if (find_item(P, unit / P.q_heads, (P.k_rows + kPrTile - 1) / kPrTile, s, index) < 0) return;
#pragma unroll 1
  for (int r = warp; r < kPrMergeRows; r += 8) {
    const int row = blockIdx.y * kPrMergeRows + r, q_row = index * kPrRows + row;
    if (q_row >= s.nq) return;
    const float* base = P.records + ((long long)unit * P.splits * kPrRows + row) * (D + 2);
    float2 ml[kPrMaxSplits], va[kPrMaxSplits][D / 64];
#pragma unroll
    for (int g = 0; g < kPrMaxSplits; ++g) {
      if (g < P.splits) {
        const float2* rec = (const float2*)(base + (long long)g * kPrRows * (D + 2));
        ml[g] = __ldcg(rec + D / 2);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) va[g][c] = __ldcg(rec + 32 * c + lane);
      }
    }
    float top = kPrNegBig;
#pragma unroll
    for (int g = 0; g < kPrMaxSplits; ++g)
      if (g < P.splits) top = fmaxf(top, ml[g].x);
    float l = 0.f;
    float2 o[D / 64] = {};
#pragma unroll
    for (int g = 0; g < kPrMaxSplits; ++g) {
      if (g < P.splits) {
        const float w = pf_exp2(ml[g].x - top);
        l = fmaf(ml[g].y, w, l);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          o[c].x = fmaf(va[g][c].x, w, o[c].x);
          o[c].y = fmaf(va[g][c].y, w, o[c].y);
        }
      }
    }
    const bool empty = s.nk - s.nq + q_row < 0;
    const float inv = empty ? 0.f : 1.f / l;
    QT* out = (QT*)P.out + (long long)head * P.o_sh + (long long)(s.q0 + q_row) * P.o_st;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) *(unsigned*)(out + 64 * c + 2 * lane) = pf_pack2<QT>(o[c].x * inv, o[c].y * inv);
    if (lane == 0 && P.lse)
      P.lse[head * P.lse_stride + s.q0 + q_row] = empty ? __int_as_float(0xff800000) : (top + log2f(l)) * kLn2;
  }
}

// ---------------------------------------------------------------------------------------- attention weights of keys
// An item is 256 keys (tiles A and B, one softmax warpgroup each) of one KV head; a step of it is 128 columns of queries:
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
  static constexpr int kSmem = kColumnsOffset + kPwColumns * kPwColumnBytes;
};
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
__device__ __forceinline__ long long shuffle64(long long v, int lane) {
  return (long long)__shfl_sync(0xffffffffu, (unsigned long long)v, lane);
}
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
__global__ void __launch_bounds__(kPrThreads, 1) prompt_weights_kernel(const PromptParams P, const __grid_constant__ CUtensorMap map_q,
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
        tc_bar_init(bar_f + 8 * i, kPrTile);
      }
#pragma unroll
      for (int i = 0; i < kPwColumns; ++i) {
        tc_bar_init(bar_c + 8 * i, 32);
        tc_bar_init(bar_cfree + 8 * i, 8);
      }
      tc_bar_init(bar_e, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
  } else if (warp < 8) {
    // offsets that the tensors do not hold, and keys of a sequence without queries
    const int t = tid - 96;
    for (int b = blockIdx.x; b < P.n_seq; b += gridDim.x) {
      if (t == 0 && bad_sequence(P, b)) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
      const Sequence s = load_sequence(P, b);
      if (s.nq == 0)
        for (int h = 0; h < P.kv_heads; ++h)
          for (int i = t; i < s.nk; i += 160) P.weights[h * P.weights_stride + s.k0 + i] = 0.f;
    }
  } else if (warp == 8) {
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

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrIssueRegs));
  StepCursor at = range->at;
  if (warp == 9) {
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
  } else if (warp == 8) {
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
  } else if (warp == 10) {
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
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrSoftmaxRegs));
    // ================================================================ one thread per key row
    const int x = warp >> 2, row = tid & (kPrTile - 1), width = P.width;
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
      unsigned v[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tc_ld32(tS + 128 * buffer + 32 * q, v[q]);
#pragma unroll
      for (int q = 0; q < 4; ++q) tc_wait_ld32(v[q]);
      tc_fence_before();
      pf_arrive(bar_f + 16 * x + 8 * buffer);
      unsigned long long sums[2] = {pf_pair(0.f, 0.f), pf_pair(0.f, 0.f)};
      // Columns 32 q .. 32 q + 31; bit c of `seen`: column 32 q + c counts.  (A polynomial on the FMA units in the place of a
      // quarter or three eighths of the exponentials changed nothing: 87 to 90 us for 4096 tokens either way.)
      auto add = [&](int q, auto some, unsigned seen) {
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 l4 = *(const float4*)(exponents + 32 * q + c);
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
        for (int q = 0; q < 4; ++q) add(q, std::false_type{}, 0u);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (32 * q < columns) {
            // columns of queries lo .. hi - 1 of a window, of one head, of half a window, or of two heads
            const int base = 32 * q & (width - 1), from = min(max(lo - base, 0), 32), to = min(max(hi - base, 0), 32);
            unsigned seen = (unsigned)((1ull << to) - 1ull) & ~(unsigned)((1ull << from) - 1ull);
            if (width == 16) seen = (seen & 0xffffu) | (32 * q + 16 < columns ? seen << 16 : 0u);
            if (__any_sync(0xffffffffu, seen != 0u)) add(q, std::true_type{}, seen);
          }
        }
      }
      float even, odd;
      pf_unpair(pf_add2(sums[0], sums[1]), even, odd);
      sum += even + odd;
      if (note->last) {
        if (x * kPrTile + row < note->keys && *abort_flag == 0) (note->cut ? P.records : P.weights)[note->at + x * kPrTile + row] = sum;
        sum = 0.f;
      }
      __syncwarp();
      if (lane == 0) pf_arrive(bar_cfree + 8 * described);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(P.status, INQ_STATUS_WAIT_TIMEOUT);
  if (warp == 8) {
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
int prompt_registers_fit(const void* kernel) {
  cudaFuncAttributes attributes;
  INQ_CUDA_CHECK(cudaFuncGetAttributes(&attributes, kernel));
  return attributes.numRegs < kPrLaunchRegs ? INQ_ERR_UNSUPPORTED : INQ_OK;
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
  P.splits = 1;
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

// KV segments per item of inq_prompt_attention.  Cuts only pay while the items are few compared with the SMs: at most 2048
// segments in all.  The lengths are not known here, a mean sequence stands for all: rounds of CTAs over the SMs, each
// as long as a mean segment, six tile times per cut (the model of inq_prefill_attention, with its figures).
int attention_cuts(int q_heads, long long q_rows, long long k_rows, int n_seq, int n_sm) {
  const long long items = most_tiles(q_rows, n_seq) * q_heads;
  const int most = (int)std::max<long long>(1, std::min<long long>(kPrMaxSplits, 2048 / std::max<long long>(items, 1)));
  const double keys = (double)k_rows / n_seq, queries = (double)q_rows / n_seq;
  const double tiles = std::max(1.0, (keys - 0.5 * std::min(queries, keys)) / kPrTile);
  const long long likely = std::max<long long>(1, (q_rows / kPrRows + (n_seq + 1) / 2) * q_heads);
  double best = 1e30;
  int cuts = 1;
  for (int sp = 1; sp <= most; ++sp) {
    if (sp > 1 && tiles / sp < 2) break;
    const double rounds = (double)((likely * sp + n_sm - 1) / n_sm);
    const double cost = rounds * (tiles / sp + (sp > 1 ? 6.0 : 0.0));
    if (cost < best - 1e-9) {
      best = cost;
      cuts = sp;
    }
  }
  return cuts;
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
long long attention_record_bytes(int q_heads, int head_dim, long long q_rows, int n_seq, int cuts) {
  return cuts > 1 ? most_tiles(q_rows, n_seq) * q_heads * cuts * kPrRows * (head_dim + 2) * (long long)sizeof(float) : 0;
}
template <typename QT, int D>
int launch_attention(const PromptParams& P, unsigned ctas, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v) {
  const int fit = prompt_registers_fit((const void*)prompt_kernel<QT, D>);
  if (fit != INQ_OK) return fit;
  INQ_CUDA_CHECK(cudaFuncSetAttribute(prompt_kernel<QT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<D>::kSmem));
  INQ_CUDA_CHECK(launch_following(prompt_kernel<QT, D>, ctas, kPrThreads, PromptShape<D>::kSmem, stream, P, q, k, v));
  if (P.splits > 1)
    INQ_CUDA_CHECK(launch_following(prompt_merge_kernel<QT, D>, dim3(ctas / P.splits, kPrRows / kPrMergeRows), 256, 0, stream, P));
  return INQ_OK;
}
template <typename QT, int D>
int launch_weights(const PromptParams& P, unsigned ctas, cudaStream_t stream, const CUtensorMap& q, const CUtensorMap& k) {
  const int fit = prompt_registers_fit((const void*)prompt_weights_kernel<QT, D>);
  if (fit != INQ_OK) return fit;
  INQ_CUDA_CHECK(cudaFuncSetAttribute(prompt_weights_kernel<QT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, WeightsShape<D>::kSmem));
  INQ_CUDA_CHECK(launch_following(prompt_weights_kernel<QT, D>, ctas, kPrThreads, WeightsShape<D>::kSmem, stream, P, q, k));
  if (P.records) INQ_CUDA_CHECK(launch_following(prompt_weights_sum_kernel, ctas, kPrRows, 0, stream, P, (int)ctas));
  return INQ_OK;
}
}  // namespace

extern "C" int64_t inq_prompt_workspace_bytes(int32_t q_heads, int32_t kv_heads, int32_t head_dim, int64_t q_rows, int64_t k_rows,
                                              int32_t n_seq, int32_t weights, int32_t window) {
  int n_sm = 0;
  if (q_heads < 1 || kv_heads < 1 || n_seq < 1 || q_rows < 0 || k_rows < 0 || sm_count(&n_sm) != INQ_OK) return 0;
  return weights ? weights_cut(q_heads / kv_heads, q_rows, window) ? 2LL * n_sm * kPrRows * (int64_t)sizeof(float) : 0
                 : attention_record_bytes(q_heads, head_dim, q_rows, n_seq, attention_cuts(q_heads, q_rows, k_rows, n_seq, n_sm));
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
  const long long items = most_tiles(a->q_rows, a->n_seq) * a->q_heads;
  P.splits = attention_cuts(a->q_heads, a->q_rows, a->k_rows, a->n_seq, n_sm);
  if (!a->workspace || a->workspace_bytes < attention_record_bytes(a->q_heads, a->head_dim, a->q_rows, a->n_seq, P.splits)) P.splits = 1;
  if (items * P.splits > 0x7fffffffLL) return INQ_ERR_CAPACITY;
  CUtensorMap map_q, map_k, map_v;
  if (!make_map(&map_q, a->q, a->dtype, a->head_dim, a->q_rows, a->q_heads, a->q_stride_t, a->q_stride_h, kPrTile) ||
      !make_map(&map_k, a->k, a->dtype, a->head_dim, a->k_rows, a->kv_heads, a->k_stride_t, a->k_stride_h, kPrTile) ||
      !make_map(&map_v, a->v, a->dtype, a->head_dim, a->k_rows, a->kv_heads, a->v_stride_t, a->v_stride_h, kPrTile))
    return INQ_ERR_ARGUMENT;
  const unsigned ctas = (unsigned)(items * P.splits);
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
