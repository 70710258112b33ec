// paged_quant.hip - keys and values of a ragged batch into pages of 8-bit codes, and
// back.
//
// Each 16 slots (a block: slots 16 i .. 16 i + 15 of a page) of a head share an fp32
// scale, value = scale * code. A block whose first token is of this call takes the scale
// that its new values need: max|x| / 127 (int8: as fine as they allow), or the
// least power of two with 448 scale >= max|x| (e4m3: its codes are as precise
// at any scale, and a power of two changes none of their bits), never below 2^-100. A
// block that holds earlier tokens of the sequence keeps its scale while the new values fit,
// else the scale grows by the least power of two 2^k that makes them fit, and
// the block's other codes become round(code / 2^k): an earlier value is off by less
// than one step of the final scale however often that happened (half a step, plus
// halves of the smaller steps before), where scales chosen afresh would add half a
// step each time. Codes are the fp32 quotients x / scale rounded to nearest, ties to even: a value that is half of
// its block's largest is a tie in int8 (63.5), so the quotient has to be the division's. It is the product with the
// reciprocal, corrected once by its remainder, which is exact where the reciprocal is correctly rounded (Markstein 1990):
// 0.15 us more than the product alone at 1024 and 13000 tokens; divisions took 1.0-1.5.
#include "paged_seq.h"

namespace bd3 {
namespace {

constexpr uint32_t kSmallestScale = (127u - 100u) << 23;  // 2^-100
constexpr uint32_t kInf = 0x7f800000u;

// One sequence's share of the tokens and where they go; positions past every table stay
// past it (a table covers 2^30 keys at most, a chunk has fewer than 2^28 tokens).
struct RopeSeq {
  int q0, n, kv;
  __device__ __forceinline__ RopeSeq of_lane(int lane) const {
    return {__builtin_amdgcn_readlane(q0, lane), __builtin_amdgcn_readlane(n, lane), __builtin_amdgcn_readlane(kv, lane)};
  }
};

// The scale that values of up to m need.
template <int POOL>
__device__ __forceinline__ uint32_t needed_scale(float m) {
  uint32_t s;
  if constexpr (POOL == kPoolInt8) {
    s = __float_as_uint(m / 127.0f);
  } else {  // 448 = 1.75 * 2^8
    const uint32_t u = __float_as_uint(m);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
    s = e > 0 ? (uint32_t)e << 23 : 0;
  }
  return s > kSmallestScale ? s : kSmallestScale;  // positive floats are ordered as their bits
}

// Four codes, of numbers that a rounding leaves at 127 or 448 at most.
template <int POOL>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  if constexpr (POOL == kPoolInt8) {
    const auto one = [](float x) { return (uint32_t)(int)__builtin_rintf(x) & 0xffu; };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
}

// A wave: a block of 16 positions of one sequence and one head of q | k | v. Lane (row
// lane / 4, part j = lane % 4) holds the coordinate pairs (8 j + i, 32 + 8 j + i) of its
// row, so the rotation is lane-local and the block's maximum one wave reduction. The
// rotation is paged_rope_kernel's; keys are encoded from its fp32 results. Bound by memory for chunks (13000 tokens, 16 heads
// on 4: 18.2 us, 75 MB, 4.1 TB/s; 19.4 before the page and the scale were asked for first), by three
// round trips else (lengths; page; old scale, with the rotation between: 4 tokens 4.4 us, 1024 4.6). Four
// heads a wave gained nothing.
template <int POOL>
__global__ __launch_bounds__(256) void paged_rope8_kernel(PagedRopeArgs a) {
  const int lane = wi_x() & 63;
  const int w = wave_uniform(wg_x() * 4 + (wi_x() >> 6));
  const int parts = a.heads + 2 * a.kv_heads;
  const int jb = fast_div(w, a.parts_div);
  const int hh = w - jb * parts;
  const SeqPiece<RopeSeq> it(
      a.seqs, jb,
      [&](int s) {
        RopeSeq r;
        r.q0 = clampi(a.q_starts[s], 0, a.tokens);
        r.n = clampi(a.q_starts[s + 1], r.q0, a.tokens) - r.q0;
        r.kv = clampi(a.kv_lens[s], 0, (1 << 30) + (1 << 28));
        return r;
      },
      [](const RopeSeq& r) { return r.n > 0 ? ((r.kv - 1) >> 4) - ((r.kv - r.n) >> 4) + 1 : 0; });
  if (!it.found) return;
  const int c = it.sq.kv - it.sq.n;
  const int begin = ((c >> 4) + it.at) * 16;  // the block's first position
  const int r = lane >> 2, j = lane & 3;
  const int pos = begin + r;
  const bool mine = pos >= c && pos < it.sq.kv;
  const int tok = it.sq.q0 + pos - c;

  // The page and the block's scale are asked for first, so that their round trips are the rotation's. Nothing
  // is written where the table has no page for the block.
  const bool is_q = hh < a.heads, is_k = !is_q && hh < a.heads + a.kv_heads;
  const int kh = hh - a.heads - (is_k ? 0 : a.kv_heads);
  const int64_t slot = begin & (a.page - 1);
  int page = -1;
  if (!is_q && begin >= 0 && (begin >> a.page_shift) < a.width)
    page = a.table[(int64_t)it.b * a.table_s + (begin >> a.page_shift)];
  u32x4 x1 = {}, x2 = {};
  if (mine) {
    const uint16_t* src = a.qkv + (int64_t)tok * a.sx_t + hh * kHeadDim + 8 * j;
    x1 = ld16(src);
    x2 = ld16(src + kHeadDim / 2);
  }
  page = wave_uniform(page);
  const bool there = (unsigned)page < (unsigned)a.pages;
  float* scale_p =
      (is_k ? a.k_scales : a.v_scales) + ((int64_t)(there ? page : 0) * a.kv_heads + (is_q ? 0 : kh)) * (a.page >> 4) + (slot >> 4);
  const bool kept = begin < c;  // the block holds earlier tokens
  float old_scale = 0.f;
  if (there && kept) old_scale = *scale_p;

  f32x4 y[4] = {};  // [half][4 of the 8]
  if (mine) {
    const bf16x8 b1 = __builtin_bit_cast(bf16x8, x1), b2 = __builtin_bit_cast(bf16x8, x2);
    if (is_q || is_k) {
      const int64_t tp = pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos);
      const float* cp = a.cos_t + tp * (kHeadDim / 2) + 8 * j;
      const float* sp = a.sin_t + tp * (kHeadDim / 2) + 8 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f1 = (float)b1[i], f2 = (float)b2[i];
        y[i >> 2][i & 3] = f1 * cp[i] - f2 * sp[i];
        y[2 + (i >> 2)][i & 3] = f1 * sp[i] + f2 * cp[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i >> 2][i & 3] = (float)b1[i];
        y[2 + (i >> 2)][i & 3] = (float)b2[i];
      }
    }
  }
  if (is_q) {
    if (!mine) return;
    uint16_t* dst = a.q + (int64_t)tok * a.sq_t + (int64_t)hh * a.sq_h + 8 * j;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
      *reinterpret_cast<bf16x8*>(dst + 32 * h2) =
          to_bf16x8(y[2 * h2][0], y[2 * h2][1], y[2 * h2][2], y[2 * h2][3], y[2 * h2 + 1][0], y[2 * h2 + 1][1],
                    y[2 * h2 + 1][2], y[2 * h2 + 1][3]);
    return;
  }
  if (!there) return;
  const int64_t row_s = is_k ? a.sk_s : a.sv_s;
  uint8_t* dst = static_cast<uint8_t*>(is_k ? a.k : a.v) + (int64_t)page * (is_k ? a.sk_p : a.sv_p) +
                 (int64_t)kh * (is_k ? a.sk_h : a.sv_h) + (slot + r) * row_s + 8 * j;

  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(y[i >> 2][i & 3]));
  m = fminf(wave_max(m), 3.4028235e38f);
  const uint32_t need = wave_uniform_u32(needed_scale<POOL>(m));
  const uint32_t old = wave_uniform_u32(__float_as_uint(old_scale));
  uint32_t scale = need;
  int grow = 0;
  if (kept && old >= kSmallestScale && old < kInf) {  // at a scale that is one
    grow = (int)(need >> 23) - (int)(old >> 23) + ((need & 0x7fffffu) > (old & 0x7fffffu));
    grow = grow > 0 ? grow : 0;
    scale = old + ((uint32_t)grow << 23);
  }
  u32x2 codes[2];
  if (mine) {
    const float s = __uint_as_float(scale), inv = 1.0f / s;
    const auto over = [&](float x) {
      x = fminf(fmaxf(x, -3.4028235e38f), 3.4028235e38f);
      const float q = x * inv;
      return fmaf(fmaf(-q, s, x), inv, q);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
      codes[i >> 1][i & 1] = encode4<POOL>(over(y[i][0]), over(y[i][1]), over(y[i][2]), over(y[i][3]));
  } else {
    if (grow == 0) return;
    const float f = __uint_as_float((uint32_t)(127 - (grow < 126 ? grow : 126)) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 x = codes_f32<POOL>(reinterpret_cast<const uint32_t*>(dst + 32 * (i >> 1))[i & 1]);
      codes[i >> 1][i & 1] = encode4<POOL>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
    }
  }
  *reinterpret_cast<u32x2*>(dst) = codes[0];
  *reinterpret_cast<u32x2*>(dst + 32) = codes[1];
  if (r == (kept ? c - begin : 0) && j == 0) *scale_p = __uint_as_float(scale);  // the first new row's lane
}

// Values of whole pools: a wave takes a block of 16 rows of a head, 16 codes a lane. Bound by memory: 29 MB of codes to 58
// of values 16.6 us, 5.2 TB/s.
template <int POOL>
__global__ __launch_bounds__(256) void page_values_kernel(PageValuesArgs a) {
  const int lane = wi_x() & 63;
  int64_t t = (int64_t)wg_x() * 4 + wave_uniform(wi_x() >> 6);
  if (t >= 2 * a.total) return;
  const int which = t >= a.total;
  if (which) t -= a.total;
  const int64_t ph = t / a.blocks;
  const int sub = (int)(t - ph * a.blocks);
  const int64_t page = ph / a.kv_heads;
  const int h = (int)(ph - page * a.kv_heads);
  const uint8_t* src = static_cast<const uint8_t*>(a.codes[which]) + page * a.s_p[which] + h * a.s_h[which] +
                       (int64_t)(16 * sub + (lane >> 2)) * a.s_s[which] + 16 * (lane & 3);
  const float scale = a.scales[which][t];
  const u32x4 w = ld16(src);
  uint16_t* dst = a.out[which] + (t * 16 + (lane >> 2)) * kHeadDim + 16 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4 x = codes_f32<POOL>(w[2 * i]) * scale, y = codes_f32<POOL>(w[2 * i + 1]) * scale;
    *reinterpret_cast<bf16x8*>(dst + 8 * i) = to_bf16x8(x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]);
  }
}

}  // namespace

hipError_t launch_paged_rope8(const PagedRopeArgs& a, int pool, hipStream_t stream) {
  const dim3 grid((unsigned)(((int64_t)a.blocks * (a.heads + 2 * a.kv_heads) + 3) / 4));
  if (pool == kPoolInt8)
    hipLaunchKernelGGL(paged_rope8_kernel<kPoolInt8>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(paged_rope8_kernel<kPoolE4m3>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_page_values(const PageValuesArgs& a, int pool, hipStream_t stream) {
  const dim3 grid((unsigned)((2 * a.total + 3) / 4));
  if (pool == kPoolInt8)
    hipLaunchKernelGGL(page_values_kernel<kPoolInt8>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(page_values_kernel<kPoolE4m3>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bd3
