// page_select.hip - which pages a query's attention reads: bounds of each page's keys,
// and the pages that promise most.
//
// bounds[page][KV head] = the lowest and the highest key of the page, channel by channel.
// No key k of the page has a larger q . k than (values of 8-bit pools: but for the bounds' rounding to bf16, 2^-9)
//     score = sum_d max(q_d low_d, q_d high_d) = q+ . high + q- . low
// (q+ = max(q, 0), q- = min(q, 0)), a product of length 128 on the matrix cores. The
// queries of one block of the chunk (they see the same keys) and the heads of a KV
// head choose together, by the largest score among them: columns of the page table that
// the block sees, `top` of them, the first ones and those around the block's own
// tokens always, equals by the lowest column.
//
// The order is that of the exact scores: bf16 products are exact in fp32, and their fp32
// sum is off by at most 2^-17 sum |q_d b_d| whatever the matrix cores' order and rounding.
// Where the border between taken and left pages is nearer than that, the scores in doubt are
// summed again in 64 bits, where bf16 products of any but extreme ratios add without a rounding.
#include "paged_seq.h"

namespace bd3 {
namespace {

// Bounds of the pages that hold tokens of the chunks: a wave a page and head. Latency: the lengths, the table's entry
// and the keys are three round trips, one after the other; 1 page x 4 heads 2.6 us, 64 pages of 32 rows x 12 heads 4.6.
template <int POOL>
__global__ __launch_bounds__(256) void page_bounds_kernel(SelectArgs s) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63;
  const int w = wave_uniform(wg_x() * 4 + (wi_x() >> 6));
  const int j = fast_div(w, a.kv_heads_div);
  const int h = w - j * a.kv_heads;
  const auto first = [&](const PagedSeq& q) { return (q.kv > q.n ? q.kv - q.n : 0) >> a.page_shift; };
  const SeqPiece<PagedSeq> it(
      a.seqs, j, [&](int b) { return PagedSeq(a, b); },
      [&](const PagedSeq& q) { return q.n > 0 && q.kv > 0 ? ((q.kv - 1) >> a.page_shift) - first(q) + 1 : 0; });
  if (!it.found) return;
  const int col = first(it.sq) + it.at;
  const int page = wave_uniform(a.table[(int64_t)it.b * a.table_s + col]);
  if ((unsigned)page >= (unsigned)a.pages) return;
  const int rest = it.sq.kv - (col << a.page_shift);
  const int keys = rest < a.page ? rest : a.page;

  constexpr int kParts = POOL == kPoolBf16 ? 8 : 4;  // 16-byte parts of a row
  constexpr int kCh = kHeadDim / kParts;             // channels of a lane
  constexpr int kRows = 64 / kParts;                 // rows of a load
  const int part = lane % kParts, row = lane / kParts;
  float lo[kCh], hi[kCh];
#pragma unroll
  for (int i = 0; i < kCh; ++i) {
    lo[i] = INFINITY;
    hi[i] = -INFINITY;
  }
  const char* src = static_cast<const char*>(a.k) + (POOL == kPoolBf16 ? 2 : 1) * (page * a.sk_p + h * a.sk_h) + 16 * part;
  const int64_t row_bytes = (POOL == kPoolBf16 ? 2 : 1) * a.sk_s;
  const float* scales = POOL == kPoolBf16 ? nullptr : a.k_scales + ((int64_t)page * a.kv_heads + h) * (a.page >> 4);
#pragma unroll 4
  for (int r0 = 0; r0 < keys; r0 += kRows) {
    const int r = r0 + row < keys ? r0 + row : keys - 1;  // the last one again
    const u32x4 x = ld16(src + r * row_bytes);
    if constexpr (POOL == kPoolBf16) {
      const bf16x8 v = __builtin_bit_cast(bf16x8, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = fminf(lo[i], (float)v[i]);
        hi[i] = fmaxf(hi[i], (float)v[i]);
      }
    } else {
      const float scale = scales[r >> 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 v = codes_f32<POOL>(x[i]) * scale;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          lo[4 * i + k] = fminf(lo[4 * i + k], v[k]);
          hi[4 * i + k] = fmaxf(hi[4 * i + k], v[k]);
        }
      }
    }
  }
  // Over the lanes of one part: rotations by 4 and 8 within 16 lanes, then across these.
  const auto over_rows = [](float x) {
    if constexpr (kParts == 4) x = fmaxf(x, dpp_move<0x124>(x));
    return max_xor16_32(fmaxf(x, dpp_move<0x128>(x)));
  };
#pragma unroll
  for (int i = 0; i < kCh; ++i) {
    lo[i] = -over_rows(-lo[i]);
    hi[i] = over_rows(hi[i]);
  }
  if (lane >= kParts) return;
  uint16_t* out = s.bounds + ((int64_t)page * a.kv_heads + h) * (2 * kHeadDim) + kCh * part;
#pragma unroll
  for (int i = 0; i < kCh; i += 8) {
    *reinterpret_cast<bf16x8*>(out + i) =
        to_bf16x8(lo[i], lo[i + 1], lo[i + 2], lo[i + 3], lo[i + 4], lo[i + 5], lo[i + 6], lo[i + 7]);
    *reinterpret_cast<bf16x8*>(out + kHeadDim + i) =
        to_bf16x8(hi[i], hi[i + 1], hi[i + 2], hi[i + 3], hi[i + 4], hi[i + 5], hi[i + 6], hi[i + 7]);
  }
}

// One block of a chunk's queries.
struct QueryBlock {
  int lo, hi;          // its tokens of the chunk
  int cols;            // columns that hold keys it sees
  int own;             // the first that holds a position of the block
  __device__ __forceinline__ QueryBlock(const PagedArgs& a, const PagedSeq& q, int g) {
    q.block_tokens(a, g, lo, hi);
    const int end = hi > lo ? q.key_end(a, hi - 1) : 0;
    cols = (int)(((int64_t)end + a.page - 1) >> a.page_shift);
    const int64_t at = ((int64_t)PagedSeq::block_of(a, q.kv - q.n) + g) * a.bs;
    own = at > 0 ? (int)(at >> a.page_shift) : 0;
  }
};

// Halves of a bf16 pair by sign: the other sign's become 0.
typedef short i16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 positive(u32x4 x) {
  const i16x8 v = __builtin_bit_cast(i16x8, x);
  return __builtin_bit_cast(bf16x8, __builtin_elementwise_max(v, (i16x8)(short)0));
}
__device__ __forceinline__ bf16x8 negative(u32x4 x) {
  const i16x8 v = __builtin_bit_cast(i16x8, x);
  return __builtin_bit_cast(bf16x8, __builtin_elementwise_min(v, (i16x8)(short)0));
}

// Scores of 16 columns: S (16 rows x 16 columns) = [q+ q-] . bounds^T on v_mfma_f32_16x16x32_bf16, the largest of
// each column over the rows, and the same product of the absolute values. Lane (l16, hq): a row's and a column's
// channels; then, in all four quarters, column l16. The first 16 rows stay in registers. (With the columns as rows of the
// product the maximum took 32 more instructions, and a call on one token over 1000 pages 2 us.)
struct ColumnScores {
  int h, rows, row0;      // the block's rows, the first one's place in the chunk
  const uint16_t* q;      // the chunk's first token, the KV head's first query head
  const uint16_t* bounds;  // the KV head's of page 0
  int64_t sq_t, sq_h, page_step;
  int pages, group;
  FastDiv group_div;
  int lane;
  u32x4 q0, q1;           // of row l16, channels 8 hq .. + 7 and 32 + 8 hq .. + 7
  struct Box {
    bf16x8 x[4];          // high, low: the same channels
  };
  int ranked_from, ranked_to;  // columns that are not always taken
  float most;             // largest sum of absolute values so far (of the lane's ranked columns)

  __device__ __forceinline__ ColumnScores(const SelectArgs& s, const PagedSeq& sq, const QueryBlock& blk, int h_)
      : h(h_), rows((blk.hi - blk.lo) * s.p.group), row0(blk.lo * s.p.group),
        q(s.p.q + (int64_t)sq.q0 * s.p.sq_t + (int64_t)(h_ * s.p.group) * s.p.sq_h),
        bounds(s.bounds + (int64_t)h_ * (2 * kHeadDim)), sq_t(s.p.sq_t), sq_h(s.p.sq_h),
        page_step((int64_t)s.p.kv_heads * (2 * kHeadDim)), pages(s.p.pages), group(s.p.group), group_div(s.p.group_div),
        lane(wi_x() & 63), ranked_from(s.first), ranked_to(blk.own - s.recent), most(0.f) {
    const uint16_t* qp = row(0);
    q0 = ld16(qp);
    q1 = ld16(qp + 32);
  }
  __device__ __forceinline__ const uint16_t* row(int r0) const {
    const int r = row0 + (r0 + (lane & 15) < rows ? r0 + (lane & 15) : rows - 1);
    const int tok = fast_div(r, group_div);
    return q + tok * sq_t + (r - tok * group) * sq_h + 8 * (lane >> 4);
  }
  __device__ __forceinline__ const uint16_t* bounds_of(int page) const {
    return bounds + page * page_step + 8 * (lane >> 4);
  }
  __device__ __forceinline__ Box load(int page) const {
    // no page: left out by the selection
    const uint16_t* bp = bounds_of((unsigned)page < (unsigned)pages ? page : 0);
    Box b;
#pragma unroll
    for (int c = 0; c < 4; ++c) b.x[c] = __builtin_bit_cast(bf16x8, ld16(bp + (c < 2 ? kHeadDim : 0) + 32 * (c & 1)));
    return b;
  }
  __device__ __forceinline__ static bf16x8 size(bf16x8 x, uint32_t bits = 0x7fff7fffu) {
    return __builtin_bit_cast(bf16x8, __builtin_bit_cast(u32x4, x) & bits);
  }
  // The bounds of a column that is not ranked (always taken, or without a page) count as zeros in the sums of absolute
  // values: they are no part of any error, and may be anything (a large first page, bounds not formed yet, page 0).
  // Those past the last column are not ranked either.
  __device__ __forceinline__ float scores(const Box& box, int col, int page) {
    float best = -INFINITY;
    const bool ranked = col >= ranked_from && col < ranked_to && (unsigned)page < (unsigned)pages;
    const uint32_t bits = ranked ? 0x7fff7fffu : 0u;
    const auto add = [&](u32x4 x0, u32x4 x1) {
      const bf16x8 part[4] = {positive(x0), positive(x1), negative(x0), negative(x1)};
      f32x4 acc = {}, sum = {};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc = mfma16(part[c], box.x[c], acc);
        sum = mfma16(c < 2 ? part[c] : size(part[c]), size(box.x[c], bits), sum);
      }
      best = fmaxf(fmaxf(best, fmaxf(acc[0], acc[1])), fmaxf(acc[2], acc[3]));
      most = fmaxf(fmaxf(most, fmaxf(sum[0], sum[1])), fmaxf(sum[2], sum[3]));
    };
    add(q0, q1);  // before the loop, whose waits are for the next columns' bounds as well
    for (int r0 = 16; r0 < rows; r0 += 16) {
      const uint16_t* qp = row(r0);
      add(ld16(qp), ld16(qp + 32));
    }
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(best), __float_as_uint(best), false, false);
    return max_xor32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  }
  // Bound of the ranked scores' distance from the exact sums: 64 additions of terms that are not zeros, each off by at most
  // 2^-23 of the terms' absolute sum whatever their order and rounding; 2^-16 for 2^-17, which covers that sum's own.
  // And twice 128 terms and sums that may have lost 2^-126 each: below it numbers may lose their bits.
  __device__ __forceinline__ float error() const { return fmaf(wave_max(most), 0x1p-16f, 0x1p-118f); }
};

// Floats in the order of unsigned integers; 0 is below all, kForced above.
constexpr uint32_t kForced = 0xffffffffu;
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return k < 1u ? 1u : (k > kForced - 1 ? kForced - 1 : k);
}
__device__ __forceinline__ uint64_t order_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return u >> 63 ? ~u : u | (uint64_t)1 << 63;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {  // as wave_max
  const auto least = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
  v = least(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = least(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = least(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = least(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = least(r[0], r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return least(q[0], q[1]);
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) { return ~wave_min_u32(~v); }

// The exact score of a page: 16 rows at a time, 16 channels to a lane, in 64 bits. (Every lane's sums run in one
// order, so equal bounds have equal scores.)
__device__ __forceinline__ double exact_score(const ColumnScores& c, int page) {
  const ColumnScores::Box box = c.load(page);
  double best = -__builtin_huge_val();
  u32x4 x[2] = {c.q0, c.q1};
  for (int r0 = 0;;) {
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bf16x8 q = __builtin_bit_cast(bf16x8, x[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (double)(float)q[i] * (double)((float)q[i] > 0.f ? (float)box.x[k][i] : (float)box.x[2 + k][i]);
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    best = sum > best ? sum : best;
    r0 += 16;
    if (r0 >= c.rows) break;
    const uint16_t* qp = c.row(r0);
    x[0] = ld16(qp);
    x[1] = ld16(qp + 32);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    const double o = __shfl_xor(best, m, 64);
    best = o > best ? o : best;
  }
  return best;
}

constexpr int kPickWaves = 4;

// What the waves of a workgroup tell each other.
constexpr int kBins = 512;
constexpr int kPasses = 4;  // of 9 bits of a key's 32
constexpr int kFew = 64;    // columns in doubt that are ranked in registers
template <int NW>
struct TeamLds {
  uint32_t words[2][5][NW];
  uint32_t bins[kPasses][kBins];
  double sums[kFew];  // of the columns in doubt
  int cols[kFew];
  int doubtful;
};
enum Merge { kSum, kLeast, kMost };
template <int NW>
struct Team {
  TeamLds<NW>& lds;
  int wave, turn = 0;
  // Each number merged over the waves.
  template <Merge... M>
  __device__ __forceinline__ void join(uint32_t (&v)[sizeof...(M)]) {
    constexpr Merge how[] = {M...};
    auto& x = lds.words[turn++ & 1];
    if ((wi_x() & 63) == 0)
#pragma unroll
      for (int k = 0; k < (int)sizeof...(M); ++k) x[k][wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < (int)sizeof...(M); ++k) {  // a lane a wave, the same in every NW lanes; then lanes i ^ 1, 2, 4, 8
      uint32_t r = x[k][wi_x() & (NW - 1)];
      const auto with = [&](uint32_t o) { r = how[k] == kSum ? r + o : how[k] == kLeast ? (r < o ? r : o) : (r > o ? r : o); };
      with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)r, 0xB1, 0xF, 0xF, false));
      with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)r, 0x4E, 0xF, 0xF, false));
      if constexpr (NW > 4) with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)r, 0x141, 0xF, 0xF, false));
      if constexpr (NW > 8) with((uint32_t)__builtin_amdgcn_update_dpp(0, (int)r, 0x140, 0xF, 0xF, false));
      v[k] = wave_uniform_u32(r);
    }
  }
  // Sum over the earlier waves, and over all.
  __device__ __forceinline__ int before(int v, int& all) {
    auto& x = lds.words[turn++ & 1];
    if ((wi_x() & 63) == 0) x[0][wave] = (uint32_t)v;
    __syncthreads();
    int r = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      r += w < wave ? (int)x[0][w] : 0;
      all += (int)x[0][w];
    }
    all = wave_uniform(all);
    return wave_uniform(r);
  }
};

// What a wave knows of its columns' keys, in every lane: candidates, those always taken, the least and
// the largest key of the others, a bound of the scores' errors (positive floats are ordered as their bits).
struct Known {
  uint32_t v[5] = {0, 0, kForced, 0, 0};
  __device__ __forceinline__ void add(uint32_t k) {
    v[0] += __popcll(__ballot(k > 0));
    v[1] += __popcll(__ballot(k == kForced));
    if (k > 0 && k != kForced) {
      v[2] = k < v[2] ? k : v[2];
      v[3] = k > v[3] ? k : v[3];
    }
  }
  __device__ __forceinline__ void done(float err) {
    v[2] = wave_min_u32(v[2]);
    v[3] = wave_max_u32(v[3]);
    v[4] = __float_as_uint(err);
  }
};

// The selection of one block and KV head by NW waves: wave w has the groups of 64 columns from w * per on, `per` to
// a wave; their keys stay in registers (per <= R) or, R = 0, are asked for again each time. key(g) is the
// lane's of group g: 0 no candidate, kForced always taken. Where the wave has them already (OWN) they come in `kept`,
// else they are there after a barrier here. sums: a double for each column.
//
// The threshold is found by histograms of 512 bins over the range of keys that it is known to be in (a bit search
// took 20 passes over the keys and 27 of the then 39 us of a call on one token over 1000 pages).
template <int NW, int R, bool OWN, class Key>
__device__ __forceinline__ void choose(const SelectArgs& s, const ColumnScores& c, const PagedSeq& sq, const QueryBlock& blk,
                                       const int32_t* table, int per, uint32_t (&kept)[R > 0 ? R : 1], Known known, Key key,
                                       double* sums, Team<NW> team) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63;
  const int groups = (blk.cols + 63) >> 6;
  const int g0 = team.wave * per;
  const int n = g0 < groups ? (g0 + per < groups ? per : groups - g0) : 0;
#pragma unroll
  for (int b = 0; b < kPasses * kBins; b += 64 * NW) (&team.lds.bins[0][0])[b + wi_x()] = 0;
  static_assert(kPasses * kBins % (64 * NW) == 0, "whole turns");
  if (wi_x() == 0) team.lds.doubtful = 0;
  team.template join<kSum, kSum, kLeast, kMost, kMost>(known.v);
  const auto reread = [&](auto f) {
    for (int i = 0; i < n; ++i) f(g0 + i, key(g0 + i));
  };
  const auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i) f(g0 + i, kept[i]);  // keys of groups past the last one are 0
    } else {
      reread(f);
    }
  };
  if constexpr (R > 0 && !OWN) {
#pragma unroll
    for (int i = 0; i < R; ++i) kept[i] = i < n ? key(g0 + i) : 0;
  }
  const int there = (int)known.v[0];
  const float err = __uint_as_float(known.v[4]);
  int need = a.top - (int)known.v[1];  // of the others

  // Taken: keys from `sure` on and the best `open` of those from `doubt` on.
  uint32_t sure = 1, doubt = 1;
  int open = 0;
  uint64_t level = 0;  // sums above it are taken, of those equal to it the first `room` columns
  int room = 0, equal_before = 0;
  if (there > a.top && need <= 0) {
    sure = doubt = kForced;  // the first of those always taken
  } else if (there > a.top) {
    uint32_t lo = known.v[2], hi = known.v[3];  // the need-th largest key of the others is in [lo, hi]
    int in_range = there - (int)known.v[1];     // as are these many
    for (int pass = 0; in_range > need && lo < hi; ++pass) {
      const int wide = 32 - __builtin_clz((hi - lo) | 1u);
      const int shift = wide > 9 ? wide - 9 : 0;
      uint32_t* bins = team.lds.bins[pass];
      each([&](int, uint32_t k) {
        if (k >= lo && k <= hi) atomicAdd(&bins[(k - lo) >> shift], 1u);
      });
      __syncthreads();
      // Lane l: bins 511 - 8 l downwards.
      uint32_t mine[8], total = 0;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        mine[b] = bins[kBins - 1 - 8 * lane - b];
        total += mine[b];
      }
      const int upto = wave_scan((int)total);
      const int at = __builtin_ctzll(__ballot(upto >= need));
      int above = __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane((int)total, at);
      int bin = 0, count = 0;
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const int m = __builtin_amdgcn_readlane((int)mine[b], at);
        if (count == 0 && above + m >= need) {
          bin = kBins - 1 - 8 * at - b;
          count = m;
        }
        above += count == 0 ? m : 0;
      }
      need -= above;
      in_range = count;
      const uint32_t last = lo + ((uint32_t)(bin + 1) << shift) - 1;
      hi = last < hi && last >= lo ? last : hi;
      lo += (uint32_t)bin << shift;
    }
    // Keys from lo on: exactly `top` with those always taken, unless equal ones are left. The next one has
    // to be further below than their errors; else the doubtful ones are those around lo.
    uint32_t border[2] = {kForced, 0};  // the least taken, the largest left
    each([&](int, uint32_t k) {
      if (k >= lo) border[0] = k < border[0] ? k : border[0];
      if (k < lo) border[1] = k > border[1] ? k : border[1];
    });
    border[0] = wave_min_u32(border[0]);
    border[1] = wave_max_u32(border[1]);
    team.template join<kLeast, kMost>(border);
    sure = doubt = lo;
    const float v = key_value(border[0]);
    const bool bounded = (__float_as_uint(err) & 0x7f800000u) != 0x7f800000u;
    if (in_range > need || !(bounded && (border[1] == 0 || v - key_value(border[1]) > 2.01f * err))) {
      // 2.01: these sums round as well, by 2^-24 |v| < 2^-8 err
      sure = bounded ? order_key(v + 2.01f * err) + 1 : kForced;
      doubt = bounded ? order_key(v - 2.01f * err) : 1;
      uint32_t count[2] = {0, 0};  // sure ones, doubtful ones
      each([&](int g, uint32_t k) {
        const bool maybe = k >= doubt && k < sure;
        const uint64_t in = __ballot(maybe);
        count[0] += __popcll(__ballot(k >= sure));
        count[1] += __popcll(in);
        if (R == 0 || in == 0) return;
        int at = 0;
        if (lane == 0) at = atomicAdd(&team.lds.doubtful, (int)__popcll(in));
        at = wave_uniform(at) + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
        if (maybe && at < kFew) team.lds.cols[at] = 64 * g + lane;
      });
      team.template join<kSum, kSum>(count);  // its barrier also shows the columns
      open = a.top - (int)count[0];
      const int few = (int)count[1];
      if (R > 0 && few <= kFew) {  // a lane each
        for (int i = team.wave; i < few; i += NW) {
          const double e = exact_score(c, wave_uniform(table[wave_uniform(team.lds.cols[i])]));
          if (lane == 0) team.lds.sums[i] = e;
        }
        __syncthreads();
        const int col = lane < few ? team.lds.cols[lane] : -1;
        const double mine = lane < few ? team.lds.sums[lane] : 0.0;
        int ahead = 0;
        for (int i = 0; i < few; ++i) {
          const double e = team.lds.sums[i];
          ahead += e > mine || (e == mine && __builtin_amdgcn_readlane(col, i) < col);
        }
        uint64_t in = __ballot(lane < few && ahead < open);
        while (in != 0) {
          const int at = __builtin_amdgcn_readlane(col, __builtin_ctzll(in));
          in &= in - 1;
#pragma unroll
          for (int i = 0; i < R; ++i) kept[i] = i < n && 64 * (g0 + i) + lane == at ? kForced : kept[i];
        }
        open = 0;
      } else {
        reread([&](int g, uint32_t k) {
          uint64_t in = __ballot(k >= doubt && k < sure);
          while (in != 0) {
            const int col = 64 * g + __builtin_ctzll(in);
            in &= in - 1;
            const double e = exact_score(c, wave_uniform(table[col]));
            if (lane == 0) sums[col] = e;
          }
        });
        __syncthreads();
        // The open-th largest of the sums, bit by bit (pages that are all alike: 30000 of them 3.6 ms, each one
        // against each 124).
        const auto count_sums = [&](auto of) {
          uint32_t m = 0;
          reread([&](int g, uint32_t k) {
            m += __popcll(__ballot(k >= doubt && k < sure && of(order_key(sums[64 * g + lane]))));
          });
          return m;
        };
        for (int bit = 63; bit >= 0; --bit) {
          const uint64_t from = level | (uint64_t)1 << bit;
          uint32_t m[1] = {count_sums([&](uint64_t x) { return x >= from; })};
          team.template join<kSum>(m);
          if ((int)m[0] >= open) level = from;
          if ((int)m[0] == open) break;
        }
        uint32_t m[1] = {count_sums([&](uint64_t x) { return x > level; })};
        team.template join<kSum>(m);
        room = open - (int)m[0];
        int all;
        equal_before = team.before((int)count_sums([&](uint64_t x) { return x == level; }), all);
      }
    }
  }
  const auto taken = [&](int g, uint32_t k, int& equal) {
    bool take = k >= sure;
    if (open > 0) {
      const bool maybe = k >= doubt && k < sure;
      const uint64_t x = maybe ? order_key(sums[64 * g + lane]) : 0;
      const uint64_t at = __ballot(maybe && x == level);
      const int nth = equal + __builtin_amdgcn_mbcnt_hi((uint32_t)(at >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)at, 0));
      take = take || (maybe && (x > level || (x == level && nth < room)));
      equal += __popcll(at);
    }
    return take;
  };
  // The columns taken, in ascending order, for each token of the block.
  int mine = 0, all;
  int equal = equal_before;
  if (open > 0)
    reread([&](int g, uint32_t k) { mine += __popcll(__ballot(taken(g, k, equal))); });
  else
    each([&](int, uint32_t k) { mine += __popcll(__ballot(k >= sure)); });
  int base = team.before(mine, all);
  int32_t* out = s.out + (int64_t)(sq.q0 + blk.lo) * a.kv_heads * a.top + (int64_t)c.h * a.top;
  const int64_t step = (int64_t)a.kv_heads * a.top;
  const int tokens = blk.hi - blk.lo;
  const auto emit = [&](int g, bool take) {
    const uint64_t in = __ballot(take);
    const int at = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
    if (take && at < a.top)
      for (int tok = 0; tok < tokens; ++tok) out[tok * step + at] = 64 * g + lane;
    base += __popcll(in);
  };
  equal = equal_before;
  if (open > 0)
    reread([&](int g, uint32_t k) { emit(g, taken(g, k, equal)); });
  else
    each([&](int g, uint32_t k) { emit(g, k >= sure); });
  for (int at = all + wi_x(); at < a.top; at += 64 * NW)
    for (int tok = 0; tok < tokens; ++tok) out[tok * step + at] = -1;
}

__device__ __forceinline__ uint32_t column_key(const SelectArgs& s, const QueryBlock& blk, int col, int page, float score) {
  if (col >= blk.cols || (unsigned)page >= (unsigned)s.p.pages) return 0;
  return col < s.first || col >= blk.own - s.recent ? kForced : order_key(score);
}

struct BlockPiece : SeqPiece<PagedSeq> {
  int h;
  __device__ __forceinline__ BlockPiece(const PagedArgs& a, int jh)
      : BlockPiece(a, jh, wave_uniform(fast_div(jh, a.kv_heads_div))) {}
  __device__ __forceinline__ BlockPiece(const PagedArgs& a, int jh, int j)
      : SeqPiece<PagedSeq>(a.seqs, j, [&](int b) { return PagedSeq(a, b); }, [&](const PagedSeq& q) { return q.blocks(a); }),
        h(jh - j * a.kv_heads) {}
};

// Up to kPickColumns: the waves of a workgroup score them into LDS, 16 a wave and turn, the next two turns' bounds
// on their way, and choose. A CU's fetches bound it (1875 columns, 480 KB, 22 us; 1000 18.6; 500 15; 187 11; eight waves
// were as fast within 3%). 32 sequences of 2000-16000 keys, pages of 32, 12 heads, two blocks each: 17.5 us, of
// which 5 are the first bounds' queue, 4-6 the rest of them, 3 the choice and 2 more that of an item with
// columns in doubt.
__global__ __launch_bounds__(64 * kPickWaves, 4) void page_pick_kernel(SelectArgs s) {
  constexpr int NW = kPickWaves;
  const PagedArgs& a = s.p;
  __shared__ uint32_t keys[kPickColumns];
  __shared__ double sums[kPickColumns];
  __shared__ TeamLds<NW> team;
  const int lane = wi_x() & 63, l16 = lane & 15;
  const int wave = wave_uniform(wi_x() >> 6);
  const BlockPiece it(a, wg_x());
  if (!it.found) return;
  const QueryBlock blk(a, it.sq, it.at);
  if (blk.lo >= blk.hi) return;
  const int32_t* table = a.table + (int64_t)it.b * a.table_s;
  const int tiles = (blk.cols + 15) >> 4;
  // The wave's pages, by way of LDS, where their keys will lie: looked up in the loop they would be
  // waited for behind the bounds on their way.
  constexpr int kTurns = kPickColumns / 64 / NW;
  const auto column = [&](int i) { return 16 * (wave + NW * i) + l16; };  // the lane's of the wave's i-th tile
  int pages[kTurns];
#pragma unroll
  for (int j = 0; j < kTurns; ++j) {
    const int col = column(4 * j + (lane >> 4));
    pages[j] = col < blk.cols ? table[col] : -1;
  }
  ColumnScores c(s, it.sq, blk, it.h);
#pragma unroll
  for (int j = 0; j < kTurns; ++j) keys[column(4 * j + (lane >> 4))] = (uint32_t)pages[j];
  constexpr int kAhead = 2;  // tiles on their way
  ColumnScores::Box box[kAhead];
  int page[kAhead];
  const auto ask = [&](int i, int k) {
    const int col = column(i);
    page[k] = col < blk.cols ? (int)keys[col] : -1;
    box[k] = c.load(page[k]);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ask(k, k);
  Known known;
  for (int i = 0; wave + NW * i < tiles; i += kAhead)
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int col = column(i + k);  // past the last one: no page, no key
      const float score = c.scores(box[k], col, page[k]);
      const uint32_t key = lane < 16 ? column_key(s, blk, col, page[k], score) : 0u;
      ask(i + k + kAhead, k);
      if (lane < 16 && col < blk.cols) keys[col] = key;
      known.add(key);
    }
  known.done(c.error());
  const auto key = [&](int g) { return 64 * g + lane < blk.cols ? keys[64 * g + lane] : 0u; };
  const int per = (((blk.cols + 63) >> 6) + NW - 1) / NW;
  uint32_t kept[kTurns];
  choose<NW, kTurns, false>(s, c, it.sq, blk, table, per, kept, known, key, sums, Team<NW>{team, wave});
}

// Few items, whose bounds few CUs would fetch (55 GB/s each), or more columns: their keys are formed by as many
// workgroups as they fill, then chosen from by NW waves. One token, 1000 columns, 4 KV heads: 4.2 + 6.2 us, the second
// launch 1.4 us until the keys are there and 3 of the choice's barriers.
__global__ __launch_bounds__(256) void page_scores_kernel(SelectArgs s, int chunks) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63, l16 = lane & 15;
  const int wave = wave_uniform(wi_x() >> 6);
  const int jh = wg_x() / chunks;
  const int col0 = 16 * (4 * (wg_x() - jh * chunks) + wave);
  const BlockPiece it(a, jh);
  if (!it.found) return;
  const QueryBlock blk(a, it.sq, it.at);
  if (col0 >= blk.cols) return;
  const int col = col0 + l16 < blk.cols ? col0 + l16 : blk.cols - 1;
  const int page = a.table[(int64_t)it.b * a.table_s + col];
  ColumnScores c(s, it.sq, blk, it.h);
  const float score = c.scores(c.load(page), col0 + l16, page);
  const float err = c.error();
  if (lane < 16) s.keys[(int64_t)jh * s.width + col0 + lane] = column_key(s, blk, col0 + lane, page, score);
  if (lane == 0) s.error[(int64_t)jh * (s.width >> 4) + (col0 >> 4)] = err;
}

// Keys and errors are asked for before the item is known: what lies behind its columns is not used.
template <int NW, int R>
__global__ __launch_bounds__(64 * NW) void page_select_kernel(SelectArgs s) {
  const PagedArgs& a = s.p;
  __shared__ TeamLds<NW> team;
  const int lane = wi_x() & 63;
  const int wave = wave_uniform(wi_x() >> 6);
  const int jh = wg_x();
  const uint32_t* keys = s.keys + (int64_t)jh * s.width;
  const float* errors = s.error + (int64_t)jh * (s.width >> 4);
  const int per = (((s.width + 63) >> 6) + NW - 1) / NW;
  uint32_t kept[R > 0 ? R : 1];
  float err = 0.f;
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int col = 64 * (wave * per + i) + lane;
      kept[i] = i < per && col < s.width ? keys[col] : 0;
    }
    if (lane < s.width >> 4) err = errors[lane];
  }
  const BlockPiece it(a, jh);
  if (!it.found) return;
  const QueryBlock blk(a, it.sq, it.at);
  if (blk.lo >= blk.hi) return;
  const int32_t* table = a.table + (int64_t)it.b * a.table_s;
  const ColumnScores c(s, it.sq, blk, it.h);
  const int tiles = (blk.cols + 15) >> 4;
  err = lane < tiles ? err : 0.f;
  for (int t = lane + (R > 0 ? 64 : 0); t < tiles; t += 64) err = fmaxf(err, errors[t]);
  err = wave_max(err);
  const auto key = [&](int g) { return 64 * g + lane < blk.cols ? keys[64 * g + lane] : 0u; };
  Known known;
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      kept[i] = 64 * (wave * per + i) + lane < blk.cols ? kept[i] : 0;
      known.add(kept[i]);
    }
  } else {
    for (int g = wave; g < (blk.cols + 63) >> 6; g += NW) known.add(key(g));
  }
  known.done(err);
  choose<NW, R, true>(s, c, it.sq, blk, table, per, kept, known, key, s.sums + (int64_t)jh * s.width, Team<NW>{team, wave});
}

}  // namespace

hipError_t launch_page_bounds(const SelectArgs& s, int pool, hipStream_t stream) {
  const dim3 grid((unsigned)(((int64_t)s.slots * s.p.kv_heads + 3) / 4));
  if (pool == kPoolBf16)
    hipLaunchKernelGGL(page_bounds_kernel<kPoolBf16>, grid, dim3(256), 0, stream, s);
  else if (pool == kPoolInt8)
    hipLaunchKernelGGL(page_bounds_kernel<kPoolInt8>, grid, dim3(256), 0, stream, s);
  else
    hipLaunchKernelGGL(page_bounds_kernel<kPoolE4m3>, grid, dim3(256), 0, stream, s);
  return hipGetLastError();
}

hipError_t launch_select_pages(const SelectArgs& s, hipStream_t stream) {
  const unsigned items = (unsigned)(s.slots * s.p.kv_heads);
  if (!select_in_two(items, s.width)) {
    hipLaunchKernelGGL(page_pick_kernel, dim3(items), dim3(64 * kPickWaves), 0, stream, s);
    return hipGetLastError();
  }
  const int chunks = (s.width + 63) / 64;
  hipLaunchKernelGGL(page_scores_kernel, dim3(items * chunks), dim3(256), 0, stream, s, chunks);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (s.width <= 4 * 64 * 8)
    hipLaunchKernelGGL((page_select_kernel<4, 8>), dim3(items), dim3(256), 0, stream, s);
  else if (s.width <= 16 * 64 * 8)
    hipLaunchKernelGGL((page_select_kernel<16, 8>), dim3(items), dim3(1024), 0, stream, s);
  else
    hipLaunchKernelGGL((page_select_kernel<16, 0>), dim3(items), dim3(1024), 0, stream, s);
  return hipGetLastError();
}

}  // namespace bd3
