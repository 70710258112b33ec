// page_select.hip - which pages a query's attention reads: bounds of each page's keys,
// and the pages that promise most.
//
// bounds[page][KV head] = the lowest and the highest key of the page, channel by channel.
// No key k of the page has a larger q . k than
//     score = sum_d max(q_d low_d, q_d high_d) = q+ . high + q- . low
// (q+ = max(q, 0), q- = min(q, 0)), a product of length 128 on the matrix cores. The
// queries of one block of the chunk (they see the same keys) and the heads of a KV
// head choose together, by the largest score among them: columns of the page table that
// the block sees, `top` of them, the first ones and those around the block's own
// tokens always, equals by the lowest column.
//
// The order is that of the exact scores: bf16 products are exact in fp32, and their
// fp32 sum is off by at most 128 * 2^-23 sum |q_d b_d| <= 2^-16 |q|_1 max |b|, whatever
// the matrix cores' order and rounding (a bound, four times a rounding to nearest's
// for 128 terms). Where the border between taken and left pages is nearer
// than that, the scores in doubt are summed again in 64 bits, where bf16 products of any
// but extreme ratios add without a rounding.
#include "paged_seq.h"

namespace bd3 {
namespace {

// Bounds of the pages that hold tokens of the chunks: a wave a page and head.
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
#pragma unroll
  for (int m = kParts; m < 64; m <<= 1)
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
      lo[i] = fminf(lo[i], shfl_xor(lo[i], m));
      hi[i] = fmaxf(hi[i], shfl_xor(hi[i], m));
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

// Scores of 16 columns a wave: S^T (16 columns x 16 rows) = bounds . [q+ q-]^T, the largest
// of each column over the rows, and the bound of their error.
__global__ __launch_bounds__(256) void page_scores_kernel(SelectArgs s, int chunks) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63, l16 = lane & 15, hq = lane >> 4;
  const int wave = wave_uniform(wi_x() >> 6);
  const int jh = wg_x() / chunks;
  const int col0 = 16 * (4 * (wg_x() - jh * chunks) + wave);
  const int j = fast_div(jh, a.kv_heads_div);
  const int h = jh - j * a.kv_heads;
  const SeqPiece<PagedSeq> it(
      a.seqs, j, [&](int b) { return PagedSeq(a, b); }, [&](const PagedSeq& q) { return q.blocks(a); });
  if (!it.found) return;
  const QueryBlock blk(a, it.sq, it.at);
  if (col0 >= blk.cols) return;

  const int col = col0 + l16 < blk.cols ? col0 + l16 : blk.cols - 1;
  int page = a.table[(int64_t)it.b * a.table_s + col];
  page = (unsigned)page < (unsigned)a.pages ? page : 0;  // no page: left out by the selection
  const uint16_t* bp = s.bounds + ((int64_t)page * a.kv_heads + h) * (2 * kHeadDim) + 8 * hq;
  bf16x8 box[4];  // high, low: channels 32 c + 8 hq .. +7
#pragma unroll
  for (int c = 0; c < 4; ++c) box[c] = __builtin_bit_cast(bf16x8, ld16(bp + (c < 2 ? kHeadDim : 0) + 32 * (c & 1)));
  float bmax = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) bmax = fmaxf(bmax, fabsf((float)box[c][i]));

  f32x4 best = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  float q1 = 0.f;
  const int rows = (blk.hi - blk.lo) * a.group;
  for (int r0 = 0; r0 < rows; r0 += 16) {
    const int row = blk.lo * a.group + (r0 + l16 < rows ? r0 + l16 : rows - 1);
    const int tok = fast_div(row, a.group_div);
    const uint16_t* qp =
        a.q + (int64_t)(it.sq.q0 + tok) * a.sq_t + (int64_t)(h * a.group + row - tok * a.group) * a.sq_h + 8 * hq;
    const u32x4 x0 = ld16(qp), x1 = ld16(qp + 32);
    f32x4 acc = mfma16(box[0], positive(x0), f32x4{});
    acc = mfma16(box[1], positive(x1), acc);
    acc = mfma16(box[2], negative(x0), acc);
    acc = mfma16(box[3], negative(x1), acc);
    const bf16x8 b0 = __builtin_bit_cast(bf16x8, x0), b1 = __builtin_bit_cast(bf16x8, x1);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += fabsf((float)b0[i]) + fabsf((float)b1[i]);
    q1 = fmaxf(q1, sum);  // of this lane's channels: the four lanes of a row add up to at least its norm
#pragma unroll
    for (int r = 0; r < 4; ++r) best[r] = fmaxf(best[r], acc[r]);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {  // over the 16 rows: lanes of one quarter
    float v = best[r];
    v = fmaxf(v, dpp_move<0xB1>(v));
    v = fmaxf(v, dpp_move<0x4E>(v));
    v = fmaxf(v, dpp_move<0x141>(v));
    best[r] = fmaxf(v, dpp_move<0x140>(v));
  }
  q1 = fmaxf(q1, dpp_move<0xB1>(q1));
  q1 = fmaxf(q1, dpp_move<0x4E>(q1));
  q1 = fmaxf(q1, dpp_move<0x141>(q1));
  q1 = fmaxf(q1, dpp_move<0x140>(q1));
  q1 += shfl_xor(q1, 16);
  q1 = sum_xor32(q1);
  bmax = wave_max(bmax);
  const int64_t at = (int64_t)jh * s.width;
  if (l16 == 0) *reinterpret_cast<f32x4*>(s.scores + at + col0 + 4 * hq) = best;
  if (lane == 0) s.error[(int64_t)jh * (s.width >> 4) + (col0 >> 4)] = q1 * bmax * 0x1p-16f;
}

// Floats in the order of unsigned integers; 0 is below all, kForced above.
constexpr uint32_t kForced = 0xffffffffu;
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return k < 1u ? 1u : (k > kForced - 1 ? kForced - 1 : k);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ uint32_t wave_min_u32(uint32_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, m, 64);
    v = v < o ? v : o;
  }
  return v;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) { return ~wave_min_u32(~v); }

// The exact score of a page: rows to lanes, channels in turn, in 64 bits.
__device__ double exact_score(const SelectArgs& s, const PagedSeq& sq, const QueryBlock& blk, int h, int page) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63;
  const uint16_t* box = s.bounds + ((int64_t)page * a.kv_heads + h) * (2 * kHeadDim);
  double best = -__builtin_huge_val();
  const int rows = (blk.hi - blk.lo) * a.group;
  for (int r0 = 0; r0 < rows; r0 += 64) {
    const int row = blk.lo * a.group + (r0 + lane < rows ? r0 + lane : rows - 1);
    const int tok = fast_div(row, a.group_div);
    const uint16_t* qp =
        a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(h * a.group + row - tok * a.group) * a.sq_h;
    double sum = 0.0;
    for (int d = 0; d < kHeadDim; d += 8) {
      const bf16x8 x = __builtin_bit_cast(bf16x8, ld16(qp + d));
      const bf16x8 lo = __builtin_bit_cast(bf16x8, ld16(box + d)), hi = __builtin_bit_cast(bf16x8, ld16(box + kHeadDim + d));
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (double)(float)x[i] * (double)(float)((float)x[i] > 0.f ? hi[i] : lo[i]);
    }
    best = sum > best ? sum : best;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_xor(best, m, 64);
    best = o > best ? o : best;
  }
  return best;
}

// The selection of one block and KV head, a wave each. R: 64 R columns at most, their keys
// in registers; 0: any number, their keys formed again from the scores each time.
template <int R>
__global__ __launch_bounds__(64) void page_select_kernel(SelectArgs s) {
  const PagedArgs& a = s.p;
  const int lane = wi_x() & 63;
  const int jh = wg_x();
  const int j = fast_div(jh, a.kv_heads_div);
  const int h = jh - j * a.kv_heads;
  const SeqPiece<PagedSeq> it(
      a.seqs, j, [&](int b) { return PagedSeq(a, b); }, [&](const PagedSeq& q) { return q.blocks(a); });
  if (!it.found) return;
  const QueryBlock blk(a, it.sq, it.at);
  if (blk.lo >= blk.hi) return;
  const int32_t* table = a.table + (int64_t)it.b * a.table_s;
  const float* scores = s.scores + (int64_t)jh * s.width;
  double* sums = s.sums + (int64_t)jh * s.width;
  const int n = (blk.cols + 63) >> 6;
  const auto key_of = [&](int i) -> uint32_t {  // 0: not seen, or no page
    const int col = 64 * i + lane;
    if (col >= blk.cols || (unsigned)table[col] >= (unsigned)a.pages) return 0;
    if (col < s.first || col >= blk.own - s.recent) return kForced;
    return order_key(scores[col]);
  };
  uint32_t kept[R > 0 ? R : 1];
  const auto reread = [&](auto f) {
    for (int i = 0; i < n; ++i) f(i, key_of(i));
  };
  const auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (i < n) f(i, kept[i]);
    } else {
      reread(f);
    }
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) kept[i] = i < n ? key_of(i) : 0;
  }
  float err = 0.f;
  for (int t = lane; t < (blk.cols + 15) >> 4; t += 64) err = fmaxf(err, s.error[(int64_t)jh * (s.width >> 4) + t]);
  err = wave_max(err);
  int there = 0;
  each([&](int, uint32_t k) { there += __popcll(__ballot(k > 0)); });

  // The largest t that at least `top` keys reach.
  uint32_t t = 1;
  if (there > a.top) {
    t = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t up = t | 1u << bit;
      int count = 0;
      each([&](int, uint32_t k) { count += __popcll(__ballot(k >= up)); });
      if (count >= a.top) t = up;
      if (count == a.top) break;
    }
  }
  // Taken: keys from t on, if exactly `top` reach it and the next one is further below than
  // their errors; else those above the doubtful ones, and the best of these.
  uint32_t sure = t, doubt = t;  // taken from `sure` on, left below `doubt`
  int open = 0;                  // places for those in between
  if (there > a.top) {
    uint32_t least = kForced, next = 0;
    int count = 0;
    each([&](int, uint32_t k) {
      if (k >= t) least = k < least ? k : least;
      if (k < t) next = k > next ? k : next;
      count += __popcll(__ballot(k >= t));
    });
    least = wave_min_u32(least);
    next = wave_max_u32(next);
    const float v = key_value(least);
    const bool bounded = (__float_as_uint(err) & 0x7f800000u) != 0x7f800000u;
    if (count != a.top || (least != kForced && next > 0 && !(bounded && v - key_value(next) > 2.01f * err))) {
      // 2.01: these sums round as well, by 2^-24 |v| < 2^-8 err
      sure = bounded ? order_key(v + 2.01f * err) + 1 : kForced;
      doubt = bounded ? order_key(v - 2.01f * err) : 1;
      if (least == kForced) sure = doubt = kForced;  // more columns always taken than fit: the first ones
      int above = 0;
      reread([&](int i, uint32_t k) {
        above += __popcll(__ballot(k >= sure));
        uint64_t in = __ballot(k >= doubt && k < sure);
        while (in != 0) {
          const int at = 64 * i + __builtin_ctzll(in);
          in &= in - 1;
          const double e = exact_score(s, it.sq, blk, h, wave_uniform(table[at]));
          if (lane == 0) sums[at] = e;
        }
      });
      open = a.top - above;
      __threadfence_block();
    }
  }
  int base = 0;
  int32_t* out = s.out + (int64_t)(it.sq.q0 + blk.lo) * a.kv_heads * a.top + (int64_t)h * a.top;
  const int64_t step = (int64_t)a.kv_heads * a.top;
  const auto emit = [&](int i, bool take) {
    const uint64_t all = __ballot(take);
    const int at = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
    if (take && at < a.top)
      for (int tok = 0; tok < blk.hi - blk.lo; ++tok) out[tok * step + at] = 64 * i + lane;
    base += __popcll(all);
  };
  if (open <= 0) {
    each([&](int i, uint32_t k) { emit(i, k >= sure); });
  } else {
    reread([&](int i, uint32_t k) {
      const bool maybe = k >= doubt && k < sure;
      int before = 0;  // doubtful ones that are better
      if (__ballot(maybe) != 0) {
        const int col = 64 * i + lane;
        const double mine = maybe ? sums[col] : 0.0;
        reread([&](int i2, uint32_t k2) {
          uint64_t in = __ballot(k2 >= doubt && k2 < sure);
          while (in != 0) {
            const int at = 64 * i2 + __builtin_ctzll(in);
            in &= in - 1;
            const double e = sums[at];
            before += e > mine || (e == mine && at < col);
          }
        });
      }
      emit(i, k >= sure || (maybe && before < open));
    });
  }
  for (int at = base + lane; at < a.top; at += 64)
    for (int tok = 0; tok < blk.hi - blk.lo; ++tok) out[tok * step + at] = -1;
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
  const int chunks = (s.width + 63) / 64;
  const unsigned items = (unsigned)(s.slots * s.p.kv_heads);
  hipLaunchKernelGGL(page_scores_kernel, dim3(items * chunks), dim3(256), 0, stream, s, chunks);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (s.width <= 64 * 8)
    hipLaunchKernelGGL(page_select_kernel<8>, dim3(items), dim3(64), 0, stream, s);
  else if (s.width <= 64 * 24)
    hipLaunchKernelGGL(page_select_kernel<24>, dim3(items), dim3(64), 0, stream, s);
  else
    hipLaunchKernelGGL(page_select_kernel<0>, dim3(items), dim3(64), 0, stream, s);
  return hipGetLastError();
}

}  // namespace bd3
