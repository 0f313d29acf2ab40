// Attention of one new token per request over an uncompressed paged cache, split over the cache's length and
// joined, with the store of the new token's key and value and the accumulated attention weights.
//
// out = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m): one pass over the cache, bound by its bytes (2 D elements
// a token and KV head).  What counts is that loads never pause, so the shape is built around them:
//   * a unit is 128 tokens of one pair (request, KV head, up to 16 of its query heads); the units of all pairs form
//     one list, cut into equal ranges, one per CTA and one CTA per SM.  The lengths are read on the device, so that a
//     captured step serves every later length; a pair that no range cuts is finished by its CTA.
//   * a warp owns 16 tokens of every unit and everything about them: its own ring of asynchronous copies, both
//     contractions (mma.sync m16n8k16), its own running maximum, sum and output.  Warps meet only where their CTA's
//     range of a pair ends; until then no barrier keeps a load waiting.
// mma.sync suffices: per 512 bytes of a token it computes 8192 operations, a tenth of what the SM could do meanwhile.
// The parts of a pair that ranges cut are joined, in their order, by the CTA that hands in the last one.
//
// Where weights are asked for, a second launch turns the logits that the first one left into them:
// out_w_j = w_j + sum_g 2^(s_gj - lse_g).
#include <algorithm>
#include <atomic>

#include "attention.cuh"

namespace inq {

constexpr int kDpWarps = 8, kDpThreads = 32 * kDpWarps;
constexpr int kDpSlice = 16;                       // tokens of a unit per warp
constexpr int kDpUnit = kDpWarps * kDpSlice;
constexpr float kDpNegBig = -3.0e38f;              // the maximum of nothing
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
  const float* weights;
  float* out_weights;
  long long w_sb, w_sh, ow_sb, ow_sh;
  float* records;      // [part + pair][rows][D + 2]: unnormalised output, maximum, sum
  float* logits;       // [request][query head][capacity], base 2
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
__device__ __forceinline__ long long count_units(const DensePagedParams& P, int upto, long long& before) {
  const int lane = threadIdx.x & 31;
  long long all = 0, front = 0;
  for (int b = lane; b < P.requests; b += 32) {
    const int n = load_request(P, b).units;
    all += n;
    if (b < upto) front += n;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, d);
    front += __shfl_xor_sync(0xffffffffu, front, d);
  }
  const long long per = (long long)P.kv_heads * P.chunks;
  before = front * per;
  return all * per;
}
// Range c of `ctas` is [range_start(c), range_start(c + 1)); there are no more ranges than units, so that none is empty.
__device__ __forceinline__ int range_count(long long total, int most) { return (int)min(total, (long long)most); }
__device__ __forceinline__ long long range_start(long long total, int cta, int ctas) { return total * cta / ctas; }
__device__ __forceinline__ int range_of(long long total, long long unit, int ctas) { return (int)(((unit + 1) * ctas - 1) / total); }

// A place in the list of units: request, pair inside the request, unit inside the pair.
struct Cursor {
  int b, pair, unit;
  Request r;
};
__device__ __forceinline__ void skip_empty(const DensePagedParams& P, Cursor& c) {
  while (c.r.units == 0 && ++c.b < P.requests) c.r = load_request(P, c.b);
}
// The place of unit `unit`, which exists.  The whole warp takes part.
__device__ __forceinline__ Cursor seek(const DensePagedParams& P, long long unit) {
  const int lane = threadIdx.x & 31, per = P.kv_heads * P.chunks;
  Cursor c = {0, 0, 0, {0, -1, 0}};
  for (int b0 = 0; b0 < P.requests; b0 += 32) {
    Request r = {0, -1, 0};
    if (b0 + lane < P.requests) r = load_request(P, b0 + lane);
    long long sum = (long long)r.units * per;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += other;
    }
    const unsigned found = __ballot_sync(0xffffffffu, sum > unit);
    if (found) {
      const int who = __ffs(found) - 1;
      c.r.tokens = __shfl_sync(0xffffffffu, r.tokens, who);
      c.r.fresh = __shfl_sync(0xffffffffu, r.fresh, who);
      c.r.units = __shfl_sync(0xffffffffu, r.units, who);
      const long long inside = unit - (__shfl_sync(0xffffffffu, sum, who) - (long long)c.r.units * per);
      c.b = b0 + who;
      c.pair = (int)(inside / c.r.units);
      c.unit = (int)(inside % c.r.units);
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
  static constexpr int kExchange = kDpWarps * 8 * D * 4;                // eight rows of every warp's output
  static constexpr int kSmem = kRing + kExchange + kDpWarps * 16 * 2 * 4;
};

// Reference maximum and sum of a row over n parts, the same in every lane; the whole warp takes part.
__device__ __forceinline__ float2 join_sums(const float* first, long long stride, int n) {
  const int lane = threadIdx.x & 31;
  float top = kDpNegBig, sum = 0.f;
  for (int c = lane; c < n; c += 32) {
    const float2 ml = __ldcg((const float2*)(first + c * stride));
    const float next = fmaxf(top, ml.x);
    sum = sum * pf_exp2(top - next) + ml.y * pf_exp2(ml.x - next);
    top = next;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float other_top = __shfl_xor_sync(0xffffffffu, top, d), other = __shfl_xor_sync(0xffffffffu, sum, d);
    const float next = fmaxf(top, other_top);
    sum = sum * pf_exp2(top - next) + other * pf_exp2(other_top - next);
    top = next;
  }
  return make_float2(top, sum);
}
// A row of a cut pair: out = sum_c O_c 2^(m_c - m) / sum_c l_c 2^(m_c - m) over its n parts.  A warp, D / 32 channels a lane.
template <typename QT, int D>
__device__ __forceinline__ void join_row(const float* rec, long long stride, int n, QT* out) {
  constexpr int kEach = D / 32;
  const int lane = threadIdx.x & 31;
  const float2 whole = join_sums(rec + D, stride, n);
  float sum[kEach] = {};
#pragma unroll 8
  for (int c = 0; c < n; ++c) {
    const float f = pf_exp2(__ldcg(rec + c * stride + D) - whole.x);
#pragma unroll
    for (int i = 0; i < kEach; i += 2) {
      const float2 x = __ldcg((const float2*)(rec + c * stride + kEach * lane + i));
      sum[i] = fmaf(x.x, f, sum[i]);
      sum[i + 1] = fmaf(x.y, f, sum[i + 1]);
    }
  }
  const float inv = whole.y == 0.f ? 0.f : 1.f / whole.y;
#pragma unroll
  for (int i = 0; i < kEach; i += 2) *(unsigned*)(out + kEach * lane + i) = pf_pack2<QT>(sum[i] * inv, sum[i + 1] * inv);
}

// TILES: query heads of a pair that the kernel holds, in eights.  Both contractions take the cache as their left operand,
// S^T = K Q^T (16 tokens x 8 heads) and O^T = V^T P^T (16 channels x 8 heads): the query heads of one KV head are few, and as
// rows of a 16-row operand half of them would be empty.  The probabilities change places between the two by movmatrix.
template <typename QT, int D, int TILES, bool WEIGHTS>
__global__ void __launch_bounds__(kDpThreads, 1) paged_kernel(const DensePagedParams P) {
  using S = DensePagedShape<D>;
  constexpr int kStages = S::kStages, kCopies = kDpSlice * S::kChunks / 32;      // 16-byte copies of a lane per K or V slice
  constexpr int kRowsAtOnce = 32 / S::kChunks;
  extern __shared__ __align__(1024) unsigned char dp_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const unsigned ring = tc_smem(dp_raw) + warp * kStages * S::kSliceBytes;
  float* const exchange = (float*)(dp_raw + S::kRing);                           // [warp][8][D], columns swizzled
  float* const ml = (float*)(dp_raw + S::kRing + S::kExchange);                  // [warp][16][maximum, sum]
  follow_stream();
  if (blockIdx.x == 0 && tid < 32)
    for (int b = tid; b < P.requests; b += 32) load_request(P, b, true);
  // requests with nothing to attend to: zeros
  for (int b = blockIdx.x; b < P.requests; b += gridDim.x)
    if (load_request(P, b).units == 0)
      for (int i = tid; i < P.q_heads * S::kChunks; i += kDpThreads)
        *(uint4*)((QT*)P.out + b * P.o_sb + (long long)(i / S::kChunks) * P.o_sh + i % S::kChunks * 8) = make_uint4(0u, 0u, 0u, 0u);
  long long unused;
  const long long total = count_units(P, 0, unused);
  const int ctas = range_count(total, gridDim.x);
  allow_next();
  if ((int)blockIdx.x >= ctas) return;
  const long long w0 = range_start(total, blockIdx.x, ctas), w1 = range_start(total, blockIdx.x + 1, ctas);
  Cursor at = seek(P, w0), ahead = at;         // the unit in work and the one to ask for next
  const int count = (int)(w1 - w0);
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
      valid = __ballot_sync(0xffffffffu, page >= 0 || (is_new && t < c.r.tokens)) & 0xffffu;
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

  unsigned long long rows_ahead = 0;        // 16 bits per requested slice, the oldest lowest
  constexpr int kAhead = kStages - 1;      // slices requested in front of the one in work
  static_assert(kAhead <= 3, "16 bits per slice, and the one in work");
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

  unsigned qf[TILES][D / 16][2];                // query heads as right operands
  float o[TILES][D / 16][4], m[TILES][2], l[TILES][2];      // heads 8 i + 2 (lane & 3) (+ 1)
  const int c0 = 2 * (lane & 3), g = lane >> 2;
  bool first = true;
  for (int done = 0; done < count; ++done) {
    const int h0 = at.pair / P.chunks * P.group + at.pair % P.chunks * 16, rows = min(P.group - at.pair % P.chunks * 16, 16);
    if (first) {
      // a new pair: its query rows (those beyond the group are zero), an empty state
      first = false;
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
        m[i][0] = m[i][1] = kDpNegBig;
        l[i][0] = l[i][1] = 0.f;
      }
    }
    ask();
    const unsigned valid = (unsigned)rows_ahead & 0xffffu;
    rows_ahead >>= 16;
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
    if (pair_ends || done + 1 == count) {
      // ---- this CTA's part of the pair: the warps' states joined, a record or, where it is the whole pair, the output
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 4);
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 8);
          l[i][e] += __shfl_xor_sync(0xffffffffu, l[i][e], 16);
          if (lane < 4) *(float2*)(ml + 2 * (warp * 16 + 8 * i + c0 + e)) = make_float2(m[i][e], l[i][e]);
        }
      const bool alone = pair_ends && done >= at.unit;      // every unit of the pair was in this range
      const long long pair = (long long)at.b * P.kv_heads * P.chunks + at.pair;
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = c0 + (e & 1);
            exchange[(warp * 8 + r) * D + ((16 * kk + g + 4 * (e & 2)) ^ (4 * r))] = o[i][kk][e];
          }
        __syncthreads();
        const int r = tid / (D / 4), c = 4 * (tid % (D / 4)), row = r + 8 * i;
        if (r < 8 && row < rows) {
          float2 each[kDpWarps];
          float top = kDpNegBig;
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
            const float4 x = *(const float4*)(exchange + (w * 8 + r) * D + (c ^ (4 * r)));
            weight = fmaf(each[w].y, f, weight);
            sum.x = fmaf(x.x, f, sum.x);
            sum.y = fmaf(x.y, f, sum.y);
            sum.z = fmaf(x.z, f, sum.z);
            sum.w = fmaf(x.w, f, sum.w);
          }
          float* const rec = P.records + ((blockIdx.x + pair) * 16 + row) * (D + 2);
          if (c == 0) *(float2*)(rec + D) = make_float2(top, weight);
          if (alone) {
            const float inv = weight == 0.f ? 0.f : 1.f / weight;
            *(uint2*)((QT*)P.out + at.b * P.o_sb + (long long)(h0 + row) * P.o_sh + c) =
                make_uint2(pf_pack2<QT>(sum.x * inv, sum.y * inv), pf_pack2<QT>(sum.z * inv, sum.w * inv));
          } else {
            *(float2*)(rec + c) = make_float2(sum.x, sum.y);
            *(float2*)(rec + c + 2) = make_float2(sum.z, sum.w);
          }
        }
        __syncthreads();
      }
      if (!alone) {
        // the CTA that hands in the last part joins them all, in their order, and leaves the counter as it found it
        const long long u0 = w0 + done - at.unit;
        const int part0 = range_of(total, u0, ctas), parts = range_of(total, u0 + at.r.units - 1, ctas) - part0 + 1;
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
          for (int row = warp; row < rows; row += kDpWarps)
            join_row<QT, D>(P.records + ((part0 + pair) * 16 + row) * (D + 2), 16 * (D + 2), parts,
                            (QT*)P.out + at.b * P.o_sb + (long long)(h0 + row) * P.o_sh);
        }
        __syncthreads();
      }
      first = true;
    }
    if (done + 1 < count) advance(P, at);
  }
}

// Accumulated weights: out_w_t = w_t + sum_g 2^(s_gt - lse_g), from the logits that the launch before this one left and the
// maxima and sums of its parts.  A block takes 512 tokens of a KV head.
constexpr int kDpWeightThreads = 128, kDpWeightEach = 4, kDpWeightTokens = kDpWeightThreads * kDpWeightEach;
template <int D>
__global__ void __launch_bounds__(kDpWeightThreads) paged_weights_kernel(const DensePagedParams P, int most_ctas, int blocks) {
  constexpr int kStride = 16 * (D + 2);
  __shared__ float lse_s[64];
  follow_stream();
  const int tid = threadIdx.x, warp = tid >> 5, kvh = blockIdx.x / blocks % P.kv_heads, b = blockIdx.x / (blocks * P.kv_heads);
  const int t0 = blockIdx.x % blocks * kDpWeightTokens;
  const Request r = load_request(P, b);
  if (t0 >= r.tokens) return;
  float sums[kDpWeightEach];
#pragma unroll
  for (int i = 0; i < kDpWeightEach; ++i) {
    const int t = t0 + tid + i * kDpWeightThreads;
    sums[i] = P.weights && t < r.tokens && t != r.fresh ? P.weights[b * P.w_sb + kvh * P.w_sh + t] : 0.f;
  }
  long long before;
  const long long total = count_units(P, b, before);
  const int ctas = range_count(total, most_ctas);
  const float* const logits = P.logits + ((long long)b * P.q_heads + kvh * P.group) * P.capacity;
  for (int g0 = 0; g0 < P.group; g0 += 64) {
    const int g1 = min(g0 + 64, P.group);
    __syncthreads();
    for (int g = g0 + warp; g < g1; g += kDpWeightThreads / 32) {
      const int pair = kvh * P.chunks + g / 16;
      const long long u0 = before + (long long)pair * r.units;
      const int c0 = range_of(total, u0, ctas), n = range_of(total, u0 + r.units - 1, ctas) - c0 + 1;
      const float2 whole = join_sums(P.records + ((c0 + (long long)b * P.kv_heads * P.chunks + pair) * 16 + g % 16) * (D + 2) + D, kStride, n);
      if ((tid & 31) == 0) lse_s[g - g0] = whole.y == 0.f ? __int_as_float(0x7f800000) : whole.x + log2f(whole.y);
    }
    __syncthreads();
#pragma unroll 4
    for (int g = g0; g < g1; ++g) {
      const float lse = lse_s[g - g0];
#pragma unroll
      for (int i = 0; i < kDpWeightEach; ++i) {
        const int t = t0 + tid + i * kDpWeightThreads;
        if (t < r.tokens) sums[i] += pf_exp2(__ldcg(logits + g * P.capacity + t) - lse);
      }
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
  return ((long long)a->requests * a->kv_heads * chunks + ctas) * 16 * (a->head_dim + 2);
}
long long logit_floats(const inq_paged_attention_args_t* a) {
  return a->out_weights ? (long long)a->requests * a->q_heads * a->table_columns * a->page_tokens : 0;
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
  if (!P.out_weights) return P.group <= 8 ? launch_kernel<QT, D, 1, false>(P, ctas, stream) : launch_kernel<QT, D, 2, false>(P, ctas, stream);
  const int rc = P.group <= 8 ? launch_kernel<QT, D, 1, true>(P, ctas, stream) : launch_kernel<QT, D, 2, true>(P, ctas, stream);
  if (rc != INQ_OK) return rc;
  const int blocks = (int)((P.capacity + kDpWeightTokens - 1) / kDpWeightTokens);
  INQ_CUDA_CHECK(launch_following(paged_weights_kernel<D>, dim3((unsigned)(P.requests * P.kv_heads * blocks)), kDpWeightThreads, 0, stream, P, ctas, blocks));
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
  if ((long long)a->requests * a->kv_heads * (((long long)a->table_columns * a->page_tokens + kDpWeightTokens - 1) / kDpWeightTokens) > 0x7fffffffLL)
    return INQ_ERR_CAPACITY;
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
  P.counters = a->counters;
  P.scale_log2e = a->scale * 1.4426950408889634f;
  P.status = a->status;
  cudaStream_t stream = (cudaStream_t)stream_;
  if (a->dtype == INQ_F16) return a->head_dim == 64 ? launch<__half, 64>(P, n_sm, stream) : launch<__half, 128>(P, n_sm, stream);
  return a->head_dim == 64 ? launch<__nv_bfloat16, 64>(P, n_sm, stream) : launch<__nv_bfloat16, 128>(P, n_sm, stream);
}
