// Attention of one new token per request over an uncompressed paged cache, split over the cache's length and
// joined, with the store of the new token's key and value and the accumulated attention weights.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m): one pass over the cache, bound by its bytes (2 D elements
// a token and KV head).  What counts is that loads never pause, so the shape is built around them:
//   * a unit is 64 tokens of one pair (request, KV head, up to 16 of its query heads); the units of all pairs form
//     one list, cut into ranges, one per CTA and two CTAs per SM (one streams while the other starts or joins).  The lengths
//     are read on the device, so that a captured step serves every later length; a pair that no range cuts is finished
//     by its CTA.
//   * a warp owns 16 tokens of every unit and everything about them: its own ring of asynchronous copies, both
//     contractions (mma.sync m16n8k16), its own running maximum, sum and output.  Warps meet only where their CTA's
//     range of a pair ends; until then no barrier keeps a load waiting.
// mma.sync suffices: per 512 bytes of a token it computes 8192 operations, a tenth of what the SM could do meanwhile.
// The parts of a pair that ranges cut are joined, in their order, by the CTA that hands in the last one, or by a launch.
// 131072 tokens of one request, 4 KV heads: 51 us, of them 45 of streaming (5.9 TB/s); 64 requests of up to 8192 tokens, 8 KV
// heads, 156 to 162 us (5.9 TB/s); 700 tokens 8.9 us, launch and four dependent trips to memory (11 with the host's call).
//
// Where weights are asked for, a further launch turns the logits that the first one left into them:
// out_w_j = w_j + sum_g 2^(s_gj - lse_g).
#include <algorithm>
#include <atomic>

#include "attention.cuh"

namespace inq {

constexpr int kDpWarps = 4, kDpThreads = 32 * kDpWarps, kDpPerSm = 2;
constexpr int kDpSlice = 16;                       // tokens of a unit per warp
constexpr int kDpUnit = kDpWarps * kDpSlice;
constexpr float kDpNothing = -3.3e38f;             // the maximum of no token at all
constexpr float kDpNegBig = -3.0e38f;              // where there are tokens, the maximum is this at least: their logits may all be -infinity
constexpr float kDpSlack = 8.f;                    // the reference maximum may lag the true one by 2^8

struct DensePagedParams {
  const void *q, *new_k, *new_v;
  void *k, *v, *out;
  long long q_sb, q_sh, o_sb, o_sh, n_sb, n_sh, m_sb, m_sh;       // n: new key, m: new value
  long long k_sp, k_sh, k_st, v_sp, v_sh, v_st;
  const int *table, *lengths;
  long long table_stride;
  long long pages;
  int requests, q_heads, kv_heads, group, chunks, page_tokens, page_shift, table_columns;
  int even_ctas;       // CTAs that run at a time: the ranges of an even cut
  int late_join;       // whether a launch of its own joins the parts
  const float* weights;
  float* out_weights;
  long long w_sb, w_sh, ow_sb, ow_sh;
  float* records;      // [part + pair][rows][D + 2]: unnormalised output, maximum, sum
  float* logits;       // [request][query head][capacity], base 2
  float* lse;          // [request][query head], base 2, where weights are asked for
  int* counters;       // [pair]: parts handed in, zero between launches
  long long capacity;
  float scale_log2e;
  int* status;
};

// Tokens that a request attends to, and whether its new token has a place.
struct Request {
  int tokens;          // cached ones and the new one
  int fresh;           // position of the new token, -1: none
  int units;
};
__device__ __forceinline__ Request load_request(const DensePagedParams& P, int b, bool report = false) {
  Request r = {0, -1, 0};
  const int held = __ldg(P.lengths + b);
  const long long room = P.capacity;
  if (held >= 0) {
    r.tokens = (int)min((long long)held, room);
    bool bad = held > room;
    if (P.new_k) {
      if (held < room) r.fresh = r.tokens++;
      else bad = true;
    }
    if (bad && report) atomicOr(P.status, INQ_STATUS_BAD_INDEX);
  }
  r.units = (r.tokens + kDpUnit - 1) / kDpUnit;
  return r;
}
// Units of all pairs, and those in front of request `upto`.  The whole warp takes part.
__device__ __forceinline__ unsigned count_units(const DensePagedParams& P, int upto, unsigned& before) {
  const int lane = threadIdx.x & 31;
  unsigned all = 0, front = 0;
  for (int b = lane; b < P.requests; b += 32) {
    const unsigned n = load_request(P, b).units;
    all += n;
    if (b < upto) front += n;
  }
  const unsigned per = P.kv_heads * P.chunks;
  before = __reduce_add_sync(0xffffffffu, front) * per;
  return __reduce_add_sync(0xffffffffu, all) * per;
}

// How the list of units is cut into ranges, one CTA each.  CTAs do not stream alike (64 requests in equal ranges: half of
// them had finished after 135 us, the last after 160), so the first CTAs get three quarters of an even share and those that
// take their places an eighth each.  Few units are cut evenly: what joins the parts costs more (16 requests, an even share
// of 29 units: 70 us, 81 with smaller ranges behind).
constexpr unsigned kDpEven = 48;         // an even share of fewer units than this is not cut further
constexpr int kDpMostRanges = 3;         // ranges per CTA of an even cut, at most
struct Ranges {
  unsigned total, ctas, size0, extra;    // the first `ctas` ranges: size0 units, the first `extra` of them one more
  unsigned size1, count;                 // then ranges of size1; count: all
  __host__ __device__ __forceinline__ Ranges(unsigned units, unsigned most) : total(units) {
    ctas = units < most ? units : most;
    count = ctas;
    size0 = size1 = extra = 0;
    if (ctas == 0) return;
    const unsigned even = units / ctas;
    size0 = even < kDpEven ? even : even - even / 4;
    const unsigned rest = units - size0 * ctas;
    if (even < kDpEven) {
      extra = rest;
    } else {
      size1 = (rest + 2 * ctas - 1) / (2 * ctas);
      count = ctas + (rest + size1 - 1) / size1;
    }
  }
  __device__ __forceinline__ unsigned start(unsigned range) const {
    return range < ctas ? range * size0 + min(range, extra) : min(ctas * size0 + extra + (range - ctas) * size1, total);
  }
  // The range that holds a unit
  __device__ __forceinline__ unsigned of(unsigned unit) const {
    const unsigned longer = extra * (size0 + 1), behind = ctas * size0 + extra;
    if (unit < longer) return unit / (size0 + 1);
    return unit < behind ? extra + (unit - longer) / size0 : ctas + (unit - behind) / size1;
  }
};

// A place in the list of units: request, pair inside the request, unit inside the pair.
struct Cursor {
  int b, pair, unit;
  Request r;
};
__device__ __forceinline__ void skip_empty(const DensePagedParams& P, Cursor& c) {
  while (c.r.units == 0 && ++c.b < P.requests) c.r = load_request(P, c.b);
}
// The place of unit `unit`, which exists.  The whole warp takes part.
__device__ __forceinline__ Cursor seek(const DensePagedParams& P, unsigned unit) {
  const int lane = threadIdx.x & 31;
  const unsigned per = P.kv_heads * P.chunks;
  Cursor c = {0, 0, 0, {0, -1, 0}};
  for (int b0 = 0; b0 < P.requests; b0 += 32) {
    Request r = {0, -1, 0};
    if (b0 + lane < P.requests) r = load_request(P, b0 + lane);
    unsigned sum = r.units * per;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, sum > unit);
    if (found) {
      const int who = __ffs(found) - 1;
      c.r.tokens = __shfl_sync(0xffffffffu, r.tokens, who);
      c.r.fresh = __shfl_sync(0xffffffffu, r.fresh, who);
      c.r.units = __shfl_sync(0xffffffffu, r.units, who);
      const unsigned inside = unit - (__shfl_sync(0xffffffffu, sum, who) - c.r.units * per);
      c.b = b0 + who;
      c.pair = (int)(inside / c.r.units);
      c.unit = (int)(inside - c.pair * c.r.units);
      return c;
    }
    unit -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return c;
}
__device__ __forceinline__ void advance(const DensePagedParams& P, Cursor& c) {
  if (++c.unit < c.r.units) return;
  c.unit = 0;
  if (++c.pair < P.kv_heads * P.chunks) return;
  c.pair = 0;
  c.r.units = 0;
  skip_empty(P, c);
}

__device__ __forceinline__ void dp_copy16(unsigned dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void dp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void dp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void dp_ldm4(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dp_ldm4t(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename QT>
__device__ __forceinline__ void dp_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  if (std::is_same<QT, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ unsigned dp_transpose(unsigned x) {
  unsigned y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <int D>
struct DensePagedShape {
  static constexpr int kRowBytes = 2 * D, kChunks = D / 8;              // 16-byte chunks of a row
  static constexpr int kSliceBytes = 2 * kDpSlice * kRowBytes;          // K rows, then V rows
  static constexpr int kStages = D == 128 ? 3 : 4;
  static constexpr int kRing = kDpWarps * kStages * kSliceBytes;
  static constexpr int kExchange = kDpWarps * 4 * D * 4;                // four rows of every warp's output
  static constexpr int kSmem = kRing + kExchange + kDpWarps * 16 * 2 * 4;
};

// Log-sum-exp of a row to base 2 (+infinity without a token, for what divides by it), and the reciprocal of its sum (zero without
// a token).  A row whose logits are all -infinity divides zero by zero, as its formula does.
__device__ __forceinline__ float join_lse(float top, float sum) { return top < kDpNegBig ? __int_as_float(0x7f800000) : top + log2f(sum); }
__device__ __forceinline__ float join_inverse(float top, float sum) { return top < kDpNegBig ? 0.f : 1.f / sum; }
// Parts c0 .. c1 - 1 of a row in their order: reference maximum, sum and, D / 32 channels a lane, unnormalised output.  A warp;
// all it reads of 16 parts is asked for at once, since a trip to memory is what this costs.
template <int D>
struct Joined {
  static constexpr int kPairs = D / 64, kAtOnce = 16;
  float top = kDpNothing, sum = 0.f;
  float2 out[kPairs] = {};
  __device__ __forceinline__ void add(const float* rec, long long stride, int c0, int c1) {
    const int lane = threadIdx.x & 31;
    for (int c = c0; c < c1; c += kAtOnce) {
      const float2 ml = lane < kAtOnce && c + lane < c1 ? __ldcg((const float2*)(rec + (c + lane) * stride + D)) : make_float2(kDpNothing, 0.f);
      float2 x[kAtOnce][kPairs];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int k = 0; k < kPairs; ++k) x[i][k] = c + i < c1 ? __ldcg((const float2*)(rec + (c + i) * stride) + 32 * k + lane) : make_float2(0.f, 0.f);
      float next = ml.x;
#pragma unroll
      for (int d = 8; d; d >>= 1) next = fmaxf(next, __shfl_xor_sync(0xffffffffu, next, d));
      next = fmaxf(top, __shfl_sync(0xffffffffu, next, 0));
      const float before = pf_exp2(top - next), factor = pf_exp2(ml.x - next);
      top = next;
      sum *= before;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) out[k] = make_float2(out[k].x * before, out[k].y * before);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const float f = __shfl_sync(0xffffffffu, factor, i);
        sum = fmaf(__shfl_sync(0xffffffffu, ml.y, i), f, sum);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          out[k].x = fmaf(x[i][k].x, f, out[k].x);
          out[k].y = fmaf(x[i][k].y, f, out[k].y);
        }
      }
    }
  }
  template <typename QT>
  __device__ __forceinline__ void store(QT* to, float* lse) const {
    const int lane = threadIdx.x & 31;
    const float inv = join_inverse(top, sum);
#pragma unroll
    for (int k = 0; k < kPairs; ++k) *(unsigned*)(to + 64 * k + 2 * lane) = pf_pack2<QT>(out[k].x * inv, out[k].y * inv);
    if (lse && lane == 0) *lse = join_lse(top, sum);
  }
};

// TILES: query heads of a pair that the kernel holds, in eights.  Both contractions take the cache as their left operand,
// S^T = K Q^T (16 tokens x 8 heads) and O^T = V^T P^T (16 channels x 8 heads): the query heads of one KV head are few, and as
// rows of a 16-row operand half of them would be empty.  The probabilities change places between the two by movmatrix.
template <typename QT, int D, int TILES, bool WEIGHTS>
__global__ void __launch_bounds__(kDpThreads, kDpPerSm) paged_kernel(const DensePagedParams P) {
  using S = DensePagedShape<D>;
  constexpr int kStages = S::kStages, kCopies = kDpSlice * S::kChunks / 32;      // 16-byte copies of a lane per K or V slice
  constexpr int kRowsAtOnce = 32 / S::kChunks;
  extern __shared__ __align__(1024) unsigned char dp_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned ring = tc_smem(dp_raw) + warp * kStages * S::kSliceBytes;
  float* const exchange = (float*)(dp_raw + S::kRing);                           // [warp][4][D], columns swizzled
  float* const ml = (float*)(dp_raw + S::kRing + S::kExchange);                  // [warp][16][maximum, sum]
  follow_stream();
  unsigned unused;
  const Ranges ranges(count_units(P, 0, unused), P.even_ctas);
  allow_next();
  const bool whole = P.page_tokens % kDpSlice == 0;     // a slice lies in one page

  // Physical page of the row that lane & 15 stands for, or -1.
  auto look_up = [&](const Cursor& c) {
    const int t = c.unit * kDpUnit + warp * kDpSlice + (lane & 15);
    if (t >= c.r.tokens) return -1;
    const int column = P.page_shift >= 0 ? t >> P.page_shift : t / P.page_tokens;
    const int page = __ldg(P.table + c.b * P.table_stride + column);
    if (page >= 0 && page < P.pages) return page;
    atomicOr(P.status, INQ_STATUS_BAD_INDEX);
    return -1;
  };
  const int chunk = lane % S::kChunks, row0 = lane / S::kChunks;       // this lane copies chunk `chunk` of rows row0 + kRowsAtOnce i
  // Asks for the slice of unit `c` into a stage; returns the rows that it holds.  Rows that there are not, and those of a
  // page outside the pool, are filled with zeros: a masked token's weight is zero, which is no help against what
  // memory may hold there.
  auto request = [&](const Cursor& c, int page, int stage) {
    const int t0 = c.unit * kDpUnit + warp * kDpSlice, kvh = c.pair / P.chunks;
    const unsigned dst = ring + stage * S::kSliceBytes;
    unsigned valid = 0;
    if (whole && t0 + kDpSlice <= c.r.tokens && (c.r.fresh < t0 || c.r.fresh >= t0 + kDpSlice)) {
      // 16 tokens of one page
      const long long p = max(page, 0);
      const int o = (P.page_shift >= 0 ? t0 & (P.page_tokens - 1) : t0 % P.page_tokens) + row0;
      const char* ks = (const char*)P.k + 2 * (p * P.k_sp + kvh * P.k_sh + o * P.k_st + 8 * chunk);
      const char* vs = (const char*)P.v + 2 * (p * P.v_sp + kvh * P.v_sh + o * P.v_st + 8 * chunk);
      const long long kstep = 2 * kRowsAtOnce * P.k_st, vstep = 2 * kRowsAtOnce * P.v_st;
      const bool have = page >= 0;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const unsigned to = dst + (row0 + i * kRowsAtOnce) * S::kRowBytes + ((chunk ^ ((row0 + i * kRowsAtOnce) & 7)) << 4);
        dp_copy16(to, ks, have);
        dp_copy16(to + kDpSlice * S::kRowBytes, vs, have);
        ks += kstep;
        vs += vstep;
      }
      valid = have ? 0xffffu : 0u;
    } else if (t0 < c.r.tokens) {
      // any row may lie in a page of its own, or be the new token's
      const int t = t0 + (lane & 15);
      const bool is_new = t == c.r.fresh;
      valid = __ballot_sync(0xffffffffu, page >= 0) & 0xffffu;      // a new token without a page is not stored, and not attended to
      const long long p = max(page, 0);
      const int o = P.page_shift >= 0 ? t & (P.page_tokens - 1) : t % P.page_tokens;
      const QT* const kr = is_new ? (const QT*)P.new_k + c.b * P.n_sb + kvh * P.n_sh : (const QT*)P.k + p * P.k_sp + kvh * P.k_sh + o * P.k_st;
      const QT* const vr = is_new ? (const QT*)P.new_v + c.b * P.m_sb + kvh * P.m_sh : (const QT*)P.v + p * P.v_sp + kvh * P.v_sh + o * P.v_st;
#pragma unroll 1
      for (int i = 0; i < kCopies; ++i) {
        const int r = row0 + i * kRowsAtOnce;
        const QT* const ks = (const QT*)__shfl_sync(0xffffffffu, (unsigned long long)kr, r);
        const QT* const vs = (const QT*)__shfl_sync(0xffffffffu, (unsigned long long)vr, r);
        const unsigned to = dst + r * S::kRowBytes + ((chunk ^ (r & 7)) << 4);
        const bool have = (valid >> r) & 1u;
        dp_copy16(to, ks + 8 * chunk, have);
        dp_copy16(to + kDpSlice * S::kRowBytes, vs + 8 * chunk, have);
      }
      // the new token is stored by the warp that reads it, once per KV head
      const unsigned news = __ballot_sync(0xffffffffu, is_new && page >= 0) & 0xffffu;
      if (news && c.pair % P.chunks == 0) {
        const int who = __ffs(news) - 1;
        const long long np = __shfl_sync(0xffffffffu, page, who);
        const int no = __shfl_sync(0xffffffffu, o, who);
        if (lane < 2 * S::kChunks) {
          const bool value = lane >= S::kChunks;
          const QT* const src = value ? (const QT*)P.new_v + c.b * P.m_sb + kvh * P.m_sh : (const QT*)P.new_k + c.b * P.n_sb + kvh * P.n_sh;
          QT* const to = value ? (QT*)P.v + np * P.v_sp + kvh * P.v_sh + no * P.v_st : (QT*)P.k + np * P.k_sp + kvh * P.k_sh + no * P.k_st;
          *(uint4*)(to + 8 * (lane % S::kChunks)) = *(const uint4*)(src + 8 * (lane % S::kChunks));
        }
      }
    }
    dp_commit();
    return valid;
  };

  // requests with nothing to attend to: zeros; lengths that the table cannot hold are reported
  auto settle = [&]() {
    for (int b = blockIdx.x; b < P.requests; b += gridDim.x)
      if (load_request(P, b, tid == 0).units == 0)
        for (int i = tid; i < P.q_heads * S::kChunks; i += kDpThreads)
          *(uint4*)((QT*)P.out + b * P.o_sb + (long long)(i / S::kChunks) * P.o_sh + i % S::kChunks * 8) = make_uint4(0u, 0u, 0u, 0u);
  };
  const unsigned range = blockIdx.x;
  if (range >= ranges.count) {
    settle();
    return;
  }
  const unsigned begin = ranges.start(range);
  const int count = (int)(ranges.start(range + 1) - begin);

  unsigned long long rows_ahead = 0;        // 16 bits per requested slice, the oldest lowest
  constexpr int kAhead = kStages - 1;      // slices requested in front of the one in work
  static_assert(kAhead <= 3, "16 bits per slice, and the one in work");
  Cursor at = seek(P, begin), ahead = at;         // the unit in work and the one to ask for next
  int page = look_up(ahead), asked = 0, ask_stage = 0, stage = 0;
  auto ask = [&]() {
    if (asked < count) {
      const unsigned valid = request(ahead, page, ask_stage);
      ask_stage = ask_stage + 1 == kStages ? 0 : ask_stage + 1;
      rows_ahead |= (unsigned long long)valid << (16 * kAhead);
      if (++asked < count) {
        advance(P, ahead);
        page = look_up(ahead);
      }
    } else {
      dp_commit();
    }
  };
  for (int i = 0; i < kAhead; ++i) {
    ask();
    rows_ahead >>= 16;
  }
  settle();

  unsigned qf[TILES][D / 16][2];                // query heads as right operands
  float o[TILES][D / 16][4], m[TILES][2], l[TILES][2];      // heads 8 i + 2 (lane & 3) (+ 1)
  const int c0 = 2 * (lane & 3), g = lane >> 2;
  unsigned some = 0;          // whether this warp has met a token of the pair
  bool first = true;
  for (int done = 1; done <= count; ++done) {
    const int h0 = at.pair / P.chunks * P.group + at.pair % P.chunks * 16, rows = min(P.group - at.pair % P.chunks * 16, 16);
    if (first) {
      // a new pair: its query rows (those beyond the group are zero), an empty state
      first = false;
      some = 0;
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const int r = g + 8 * i;
        const QT* const src = (const QT*)P.q + at.b * P.q_sb + (long long)(h0 + min(r, rows - 1)) * P.q_sh + c0;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[i][kk][0] = r < rows ? *(const unsigned*)(src + 16 * kk) : 0u;
          qf[i][kk][1] = r < rows ? *(const unsigned*)(src + 16 * kk + 8) : 0u;
          o[i][kk][0] = o[i][kk][1] = o[i][kk][2] = o[i][kk][3] = 0.f;
        }
        m[i][0] = m[i][1] = kDpNothing;
        l[i][0] = l[i][1] = 0.f;
      }
    }
    ask();
    const unsigned valid = (unsigned)rows_ahead & 0xffffu;
    rows_ahead >>= 16;
    some |= valid;
    dp_wait<kAhead>();
    __syncwarp();
    if (at.unit * kDpUnit + warp * kDpSlice < at.r.tokens) {
      const unsigned kbase = ring + stage * S::kSliceBytes, vbase = kbase + kDpSlice * S::kRowBytes;
      // two chains per tile of heads, so that a contraction does not wait for the one before it
      float s[TILES][2][4] = {};
      const int krow = lane & 15, kc = lane >> 4;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        unsigned a[4];
        dp_ldm4(a, kbase + krow * S::kRowBytes + (((2 * kk + kc) ^ (krow & 7)) << 4));
#pragma unroll
        for (int i = 0; i < TILES; ++i) dp_mma<QT>(s[i][kk & 1], a[0], a[1], a[2], a[3], qf[i][kk][0], qf[i][kk][1]);
      }
      unsigned p[TILES][2];
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        float x[4];       // tokens g (0, 1) and g + 8 (2, 3)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (s[i][0][e] + s[i][1][e]) * P.scale_log2e;
        if (valid != 0xffffu) {
          if (!((valid >> g) & 1u)) x[0] = x[1] = __int_as_float(0xff800000);
          if (!((valid >> (g + 8)) & 1u)) x[2] = x[3] = __int_as_float(0xff800000);
        }
        if (WEIGHTS) {
          const int t = at.unit * kDpUnit + warp * kDpSlice + g;
          float* const to = P.logits + ((long long)at.b * P.q_heads + h0 + 8 * i + c0) * P.capacity + t;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (8 * i + c0 + (e & 1) < rows && t + 4 * (e & 2) < at.r.tokens) to[(e & 1) * P.capacity + 4 * (e & 2)] = x[e];
        }
        float top[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[e] = fmaxf(x[e], x[e + 2]);
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
          top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16));
        }
        if (__any_sync(0xffffffffu, top[0] > m[i][0] + kDpSlack || top[1] > m[i][1] + kDpSlack)) {
          float factor[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float next = top[e] > m[i][e] + kDpSlack ? top[e] : m[i][e];
            factor[e] = pf_exp2(m[i][e] - next);
            m[i][e] = next;
            l[i][e] *= factor[e];
          }
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            o[i][kk][0] *= factor[0];
            o[i][kk][1] *= factor[1];
            o[i][kk][2] *= factor[0];
            o[i][kk][3] *= factor[1];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = pf_exp2(x[e] - m[i][e & 1]);
        l[i][0] += x[0] + x[2];
        l[i][1] += x[1] + x[3];
        // rounded once, the sums are not; tokens change from rows to columns
        p[i][0] = dp_transpose(pf_pack2<QT>(x[0], x[1]));
        p[i][1] = dp_transpose(pf_pack2<QT>(x[2], x[3]));
      }
      // matrices of a transposed load: channels 16 kk .. and 16 kk + 8 .. of tokens 0-7, then of tokens 8-15
      const int vrow = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        unsigned a[4];
        dp_ldm4t(a, vbase + vrow * S::kRowBytes + (((2 * kk + vc) ^ (vrow & 7)) << 4));
#pragma unroll
        for (int i = 0; i < TILES; ++i) dp_mma<QT>(o[i][kk], a[0], a[1], a[2], a[3], p[i][0], p[i][1]);
      }
    }
    __syncwarp();        // the stage may be asked for again
    stage = stage + 1 == kStages ? 0 : stage + 1;
    const bool pair_ends = at.unit + 1 == at.r.units;
    if (pair_ends || done == count) {
      // ---- this CTA's part of the pair: the warps' states joined, a record or, where it is the whole pair, the output
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 4);
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 8);
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 16);
          if (lane < 4) *(float2*)(ml + 2 * (warp * 16 + 8 * i + c0 + e)) = make_float2(some ? fmaxf(m[i][e], kDpNegBig) : m[i][e], l[i][e]);
        }
      const bool alone = pair_ends && done > at.unit;      // every unit of the pair was in this range
      const long long pair = (long long)at.b * P.kv_heads * P.chunks + at.pair;
#pragma unroll
      for (int four = 0; four < 2 * TILES; ++four) {      // rows 4 four .. of the pair, which half of the lanes hold
        if ((lane & 2) == 2 * (four & 1)) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = (c0 & 2) + (e & 1);
              exchange[(warp * 4 + r) * D + ((16 * kk + g + 4 * (e & 2)) ^ (8 * r))] = o[four >> 1][kk][e];
            }
        }
        __syncthreads();
        const int r = tid / (D / 4), c = 4 * (tid % (D / 4)), row = r + 4 * four;
        if (r < 4 && row < rows) {
          float2 each[kDpWarps];
          float top = kDpNothing;
#pragma unroll
          for (int w = 0; w < kDpWarps; ++w) {
            each[w] = *(const float2*)(ml + 2 * (w * 16 + row));
            top = fmaxf(top, each[w].x);
          }
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          float weight = 0.f;
#pragma unroll
          for (int w = 0; w < kDpWarps; ++w) {
            const float f = pf_exp2(each[w].x - top);
            const float4 x = *(const float4*)(exchange + (w * 4 + r) * D + (c ^ (8 * r)));
            weight = fmaf(each[w].y, f, weight);
            sum.x = fmaf(x.x, f, sum.x);
            sum.y = fmaf(x.y, f, sum.y);
            sum.z = fmaf(x.z, f, sum.z);
            sum.w = fmaf(x.w, f, sum.w);
          }
          float* const rec = P.records + ((range + pair) * 16 + row) * (D + 2);
          if (c == 0) *(float2*)(rec + D) = make_float2(top, weight);
          if (alone) {
            if (WEIGHTS && c == 0) P.lse[at.b * P.q_heads + h0 + row] = join_lse(top, weight);
            const float inv = join_inverse(top, weight);
            *(uint2*)((QT*)P.out + at.b * P.o_sb + (long long)(h0 + row) * P.o_sh + c) =
                make_uint2(pf_pack2<QT>(sum.x * inv, sum.y * inv), pf_pack2<QT>(sum.z * inv, sum.w * inv));
          } else {
            *(float2*)(rec + c) = make_float2(sum.x, sum.y);
            *(float2*)(rec + c + 2) = make_float2(sum.z, sum.w);
          }
        }
        __syncthreads();
      }
      if (!alone && !P.late_join) {
        // the CTA that hands in the last part joins them all, in their order, and leaves the counter as it found it
        const unsigned u0 = begin + done - 1 - at.unit;
        const int part0 = (int)ranges.of(u0), parts = (int)ranges.of(u0 + at.r.units - 1) - part0 + 1;
        __threadfence();
        __syncthreads();
        int* const last = (int*)ml;
        if (tid == 0) {
          const bool is_last = atomicAdd(P.counters + pair, 1) == parts - 1;
          if (is_last) P.counters[pair] = 0;
          *last = is_last;
        }
        __syncthreads();
        const bool joins = *last != 0;
        if (joins) {
          __threadfence();
          for (int row = warp; row < rows; row += kDpWarps) {
            Joined<D> all;
            all.add(P.records + ((part0 + pair) * 16 + row) * (D + 2), 16 * (D + 2), 0, parts);
            all.template store<QT>((QT*)P.out + at.b * P.o_sb + (long long)(h0 + row) * P.o_sh, WEIGHTS ? P.lse + at.b * P.q_heads + h0 + row : nullptr);
          }
        }
        __syncthreads();
      }
      first = true;
    }
    if (done < count) advance(P, at);
  }
}

// Joins the parts of all pairs, a block per row, its warps neighbouring parts each: where a pair has many parts, one CTA of the
// launch above would take longer over its rows than this launch does.
constexpr int kDpJoinWarps = 8;
template <typename QT, int D>
__global__ void __launch_bounds__(32 * kDpJoinWarps) paged_join_kernel(const DensePagedParams P) {
  __shared__ float2 ml[kDpJoinWarps], outs[kDpJoinWarps][D / 2];
  follow_stream();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x / P.q_heads, head = blockIdx.x % P.q_heads;
  const Request r = load_request(P, b);
  if (r.units == 0) return;
  unsigned before;
  const Ranges ranges(count_units(P, b, before), P.even_ctas);
  const int g = head % P.group, pair = head / P.group * P.chunks + g / 16;
  const unsigned u0 = before + pair * r.units;
  const int part0 = (int)ranges.of(u0), parts = (int)ranges.of(u0 + r.units - 1) - part0 + 1;
  if (parts == 1) return;       // written by the CTA that had the whole pair
  Joined<D> mine;
  mine.add(P.records + ((part0 + (long long)b * P.kv_heads * P.chunks + pair) * 16 + g % 16) * (D + 2), 16 * (D + 2), parts * warp / kDpJoinWarps,
           parts * (warp + 1) / kDpJoinWarps);
  if (lane == 0) ml[warp] = make_float2(mine.top, mine.sum);
#pragma unroll
  for (int k = 0; k < D / 64; ++k) outs[warp][32 * k + lane] = mine.out[k];
  __syncthreads();
  if (warp) return;
  Joined<D> all;
#pragma unroll
  for (int w = 0; w < kDpJoinWarps; ++w) all.top = fmaxf(all.top, ml[w].x);
#pragma unroll
  for (int w = 0; w < kDpJoinWarps; ++w) {
    const float f = pf_exp2(ml[w].x - all.top);
    all.sum = fmaf(ml[w].y, f, all.sum);
#pragma unroll
    for (int k = 0; k < D / 64; ++k) {
      const float2 x = outs[w][32 * k + lane];
      all.out[k] = make_float2(fmaf(x.x, f, all.out[k].x), fmaf(x.y, f, all.out[k].y));
    }
  }
  all.template store<QT>((QT*)P.out + b * P.o_sb + (long long)head * P.o_sh, P.out_weights ? P.lse + blockIdx.x : nullptr);
}

// Accumulated weights: out_w_t = w_t + sum_g 2^(s_gt - lse_g), from the logits and log-sum-exps that the launches before this
// one left.  A block takes 512 tokens of a KV head.
constexpr int kDpWeightThreads = 128, kDpWeightEach = 4, kDpWeightTokens = kDpWeightThreads * kDpWeightEach;
__global__ void __launch_bounds__(kDpWeightThreads) paged_weights_kernel(const DensePagedParams P, int blocks) {
  follow_stream();
  const int tid = threadIdx.x, kvh = blockIdx.x / blocks % P.kv_heads, b = blockIdx.x / (blocks * P.kv_heads);
  const int t0 = blockIdx.x % blocks * kDpWeightTokens;
  const Request r = load_request(P, b);
  if (t0 >= r.tokens) return;
  float sums[kDpWeightEach];
#pragma unroll
  for (int i = 0; i < kDpWeightEach; ++i) {
    const int t = t0 + tid + i * kDpWeightThreads;
    sums[i] = P.weights && t < r.tokens && t != r.fresh ? P.weights[b * P.w_sb + kvh * P.w_sh + t] : 0.f;
  }
  const float* const lse = P.lse + b * P.q_heads + kvh * P.group;
  const float* const logits = P.logits + ((long long)b * P.q_heads + kvh * P.group) * P.capacity;
#pragma unroll 4
  for (int g = 0; g < P.group; ++g) {
    const float minus = __ldcg(lse + g);
#pragma unroll
    for (int i = 0; i < kDpWeightEach; ++i) {
      const int t = t0 + tid + i * kDpWeightThreads;
      if (t < r.tokens) sums[i] += pf_exp2(__ldcg(logits + g * P.capacity + t) - minus);
    }
  }
#pragma unroll
  for (int i = 0; i < kDpWeightEach; ++i) {
    const int t = t0 + tid + i * kDpWeightThreads;
    if (t < r.tokens) P.out_weights[b * P.ow_sb + kvh * P.ow_sh + t] = sums[i];
  }
}

}  // namespace inq

using namespace inq;

namespace {
int ranges(int* n) {
  int device = 0;   // asked per call: the answer belongs to the current device
  INQ_CUDA_CHECK(cudaGetDevice(&device));
  INQ_CUDA_CHECK(cudaDeviceGetAttribute(n, cudaDevAttrMultiProcessorCount, device));
  return INQ_OK;
}
long long record_floats(const inq_paged_attention_args_t* a, int ctas) {
  const long long chunks = (a->q_heads / a->kv_heads + 15) / 16;
  return ((long long)a->requests * a->kv_heads * chunks + (long long)ctas * kDpPerSm * kDpMostRanges) * 16 * (a->head_dim + 2);
}
long long logit_floats(const inq_paged_attention_args_t* a) {
  return a->out_weights ? (long long)a->requests * a->q_heads * ((long long)a->table_columns * a->page_tokens + 1) : 0;      // and lse
}
int check_args(const inq_paged_attention_args_t* a) {
  if (!a || !a->q || !a->k || !a->v || !a->out || !a->table || !a->lengths || !a->counters || !a->status) return INQ_ERR_ARGUMENT;
  if (a->requests < 1 || a->kv_heads < 1 || a->q_heads < 1 || a->q_heads % a->kv_heads || !(a->scale > 0.f)) return INQ_ERR_ARGUMENT;
  if (a->pages < 1 || a->page_tokens < 1 || a->table_columns < 1) return INQ_ERR_ARGUMENT;
  if ((a->new_k == nullptr) != (a->new_v == nullptr) || (a->weights && !a->out_weights)) return INQ_ERR_ARGUMENT;
  if (a->dtype != INQ_F16 && a->dtype != INQ_BF16) return INQ_ERR_UNSUPPORTED;
  if (a->head_dim != 64 && a->head_dim != 128) return INQ_ERR_UNSUPPORTED;
  if ((long long)a->table_columns * a->page_tokens > 0x3fffffffLL || a->pages > 0x7fffffffLL) return INQ_ERR_CAPACITY;
  // rows are moved as 16-byte vectors
  if ((a->q_stride_b | a->q_stride_h | a->o_stride_b | a->o_stride_h | a->k_stride_p | a->k_stride_h | a->k_stride_t | a->v_stride_p |
       a->v_stride_h | a->v_stride_t | a->new_k_stride_b | a->new_k_stride_h | a->new_v_stride_b | a->new_v_stride_h) & 7)
    return INQ_ERR_ARGUMENT;
  if (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)a->new_k | (uintptr_t)a->new_v) & 15) return INQ_ERR_ARGUMENT;
  return INQ_OK;
}
// The limit belongs to a kernel on a device; a device that has it is not asked again.
int allow_shared(const void* kernel, std::atomic<unsigned long long>& known, int bytes) {
  int device = 0;
  INQ_CUDA_CHECK(cudaGetDevice(&device));
  const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
  if (known.load(std::memory_order_relaxed) & bit) return INQ_OK;
  INQ_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  known.fetch_or(bit, std::memory_order_relaxed);
  return INQ_OK;
}
template <typename QT, int D, int TILES, bool WEIGHTS>
int launch_kernel(const DensePagedParams& P, int ctas, cudaStream_t stream) {
  static std::atomic<unsigned long long> known{0};
  const int rc = allow_shared((const void*)paged_kernel<QT, D, TILES, WEIGHTS>, known, DensePagedShape<D>::kSmem);
  if (rc != INQ_OK) return rc;
  INQ_CUDA_CHECK(launch_following(paged_kernel<QT, D, TILES, WEIGHTS>, ctas, kDpThreads, DensePagedShape<D>::kSmem, stream, P));
  return INQ_OK;
}
template <typename QT, int D>
int launch(const DensePagedParams& P, int ctas, cudaStream_t stream) {
  const int rc = P.out_weights ? P.group <= 8 ? launch_kernel<QT, D, 1, true>(P, ctas, stream) : launch_kernel<QT, D, 2, true>(P, ctas, stream)
                 : P.group <= 8 ? launch_kernel<QT, D, 1, false>(P, ctas, stream) : launch_kernel<QT, D, 2, false>(P, ctas, stream);
  if (rc != INQ_OK) return rc;
  if (P.late_join) INQ_CUDA_CHECK(launch_following(paged_join_kernel<QT, D>, dim3(P.requests * P.q_heads), 32 * kDpJoinWarps, 0, stream, P));
  if (P.out_weights) {
    const int blocks = (int)((P.capacity + kDpWeightTokens - 1) / kDpWeightTokens);
    INQ_CUDA_CHECK(launch_following(paged_weights_kernel, dim3((unsigned)(P.requests * P.kv_heads * blocks)), kDpWeightThreads, 0, stream, P, blocks));
  }
  return INQ_OK;
}
}  // namespace

extern "C" int64_t inq_paged_attention_workspace_bytes(const inq_paged_attention_args_t* a) {
  int n_sm = 0;
  if (!a || a->kv_heads < 1 || a->q_heads < 1 || ranges(&n_sm) != INQ_OK) return 0;
  return 4 * (record_floats(a, n_sm) + logit_floats(a));
}

extern "C" int inq_paged_attention(const inq_paged_attention_args_t* a, inq_stream_t stream_) {
  int rc = check_args(a);
  if (rc != INQ_OK) return rc;
  int n_sm = 0;
  rc = ranges(&n_sm);
  if (rc != INQ_OK) return rc;
  const long long records = record_floats(a, n_sm);
  const long long most_units = (long long)a->requests * a->kv_heads * ((a->q_heads / a->kv_heads + 15) / 16) *
                               (((long long)a->table_columns * a->page_tokens + kDpUnit - 1) / kDpUnit);
  if ((long long)a->requests * a->kv_heads * (((long long)a->table_columns * a->page_tokens + kDpWeightTokens - 1) / kDpWeightTokens) > 0x7fffffffLL)
    return INQ_ERR_CAPACITY;
  if (most_units > 0x7fffffffLL) return INQ_ERR_CAPACITY;      // units are counted in 32 bits
  if (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < 4 * (records + logit_floats(a))) return INQ_ERR_CAPACITY;
  DensePagedParams P = {};
  P.q = a->q; P.k = a->k; P.v = a->v; P.out = a->out; P.new_k = a->new_k; P.new_v = a->new_v;
  P.q_sb = a->q_stride_b; P.q_sh = a->q_stride_h; P.o_sb = a->o_stride_b; P.o_sh = a->o_stride_h;
  P.k_sp = a->k_stride_p; P.k_sh = a->k_stride_h; P.k_st = a->k_stride_t;
  P.v_sp = a->v_stride_p; P.v_sh = a->v_stride_h; P.v_st = a->v_stride_t;
  P.n_sb = a->new_k_stride_b; P.n_sh = a->new_k_stride_h; P.m_sb = a->new_v_stride_b; P.m_sh = a->new_v_stride_h;
  P.table = a->table; P.lengths = a->lengths; P.table_stride = a->table_stride; P.pages = a->pages;
  P.requests = a->requests; P.q_heads = a->q_heads; P.kv_heads = a->kv_heads; P.group = a->q_heads / a->kv_heads;
  P.chunks = (P.group + 15) / 16;
  P.page_tokens = a->page_tokens; P.table_columns = a->table_columns;
  P.page_shift = -1;
  for (int i = 0; i < 30; ++i)
    if (a->page_tokens == 1 << i) P.page_shift = i;
  P.capacity = (long long)a->table_columns * a->page_tokens;
  P.weights = a->weights; P.out_weights = a->out_weights;
  P.w_sb = a->w_stride_b; P.w_sh = a->w_stride_h; P.ow_sb = a->ow_stride_b; P.ow_sh = a->ow_stride_h;
  P.records = (float*)a->workspace;
  P.logits = P.records + records;
  P.lse = P.logits + (long long)a->requests * a->q_heads * P.capacity;
  P.counters = a->counters;
  P.even_ctas = kDpPerSm * n_sm;
  // parts of a pair if all are alike: a CTA joins up to sixteen in one trip to memory
  P.late_join = P.even_ctas > 16LL * a->requests * a->kv_heads * P.chunks && most_units > 16LL * a->requests * a->kv_heads * P.chunks;
  P.scale_log2e = a->scale * 1.4426950408889634f;
  P.status = a->status;
  // the lengths are not known here: as many CTAs as any would need
  const long long even = most_units / P.even_ctas;
  const int ctas = (int)std::max<long long>(1, std::min<long long>(most_units, even < kDpEven ? P.even_ctas : (long long)P.even_ctas * kDpMostRanges));
  cudaStream_t stream = (cudaStream_t)stream_;
  if (a->dtype == INQ_F16) return a->head_dim == 64 ? launch<__half, 64>(P, ctas, stream) : launch<__half, 128>(P, ctas, stream);
  return a->head_dim == 64 ? launch<__nv_bfloat16, 64>(P, ctas, stream) : launch<__nv_bfloat16, 128>(P, ctas, stream);
}
