// paged.hip - attention of ragged batches over a paged KV cache in bf16, and the
// attention inputs written into its pages. The tiles are in paged_tiles.h.
//
// Pages cost 11% against a contiguous cache in full launches: 32 sequences x 12 heads,
// 16 rows over 4112 keys, 70 us at 16- to 256-key pages (5.8 TB/s) against 63; short
// ones pay two dependent reads (lengths, table entries) before the first key.
#include "paged_tiles.h"

namespace bd3 {
namespace {

// Rotary embedding of q and k at each token's position, q to packed tokens, k and
// v into the pages. y1 = x1 c - x2 s, y2 = x1 s + x2 c on the halves of a head
// row, in fp32 with the fp32 tables and rounded once (qkv_rope.hip instead repeats
// an eager bf16 path's five roundings, which no caller of pages has to match).
// Bound by HBM: 24 chunks of 100-2000 tokens, 16 + 2 x 4 heads, 20.0 us, 4.9 TB/s read
// and written (a large copy: 5.1); a denoising step's 1024 tokens take 4.4 us.
// Work item: (token, head of q | k | v, j): coordinate pairs (8j + i, 32 + 8j + i).
__global__ __launch_bounds__(256) void paged_rope_kernel(PagedRopeArgs a) {
  const uint32_t e0 = (uint32_t)wg_x() * 256u, e = e0 + wi_x();
  const uint32_t per_tok = 4u * (uint32_t)(a.heads + 2 * a.kv_heads);
  // The sequence of the workgroup's first token: those that end before it.
  const int tok0 = (int)(e0 / per_tok);
  int b = 0;
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    const int s = s0 + (wi_x() & 63);
    b += __popcll(__ballot(s < a.seqs && a.q_starts[s + 1] <= tok0));
  }
  if (e >= (uint32_t)a.total) return;
  const int tok = (int)(e / per_tok);
  const int r = (int)(e - (uint32_t)tok * per_tok);
  const int hh = r >> 2, j = r & 3;
  while (b < a.seqs && a.q_starts[b + 1] <= tok) ++b;
  if (b >= a.seqs || a.q_starts[b] > tok) return;  // behind the last sequence
  const int end = a.q_starts[b + 1] < a.tokens ? a.q_starts[b + 1] : a.tokens;
  const int64_t pos = (int64_t)a.kv_lens[b] - (end - tok);

  const uint16_t* src = a.qkv + (int64_t)tok * a.sx_t + hh * kHeadDim + 8 * j;
  u32x4 x1 = ld16(src), x2 = ld16(src + kHeadDim / 2);
  uint16_t* dst;
  if (hh < a.heads) {
    dst = a.q + (int64_t)tok * a.sq_t + (int64_t)hh * a.sq_h;
  } else {
    // Nothing is written where the table has no page for the position.
    if (pos < 0 || (pos >> a.page_shift) >= a.width) return;
    const int page = a.table[(int64_t)b * a.table_s + (pos >> a.page_shift)];
    if ((unsigned)page >= (unsigned)a.pages) return;
    const int64_t slot = pos & (a.page - 1);
    const int kh = hh - a.heads;
    dst = kh < a.kv_heads ? static_cast<uint16_t*>(a.k) + (int64_t)page * a.sk_p + (int64_t)kh * a.sk_h + slot * a.sk_s
                          : static_cast<uint16_t*>(a.v) + (int64_t)page * a.sv_p + (int64_t)(kh - a.kv_heads) * a.sv_h + slot * a.sv_s;
  }
  if (hh < a.heads + a.kv_heads) {
    const int64_t tp = pos < 0 ? 0 : (pos >= a.max_pos ? a.max_pos - 1 : pos);
    const float* cp = a.cos_t + tp * (kHeadDim / 2) + 8 * j;
    const float* sp = a.sin_t + tp * (kHeadDim / 2) + 8 * j;
    bf16x8 b1 = __builtin_bit_cast(bf16x8, x1), b2 = __builtin_bit_cast(bf16x8, x2), y1, y2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f1 = (float)b1[i], f2 = (float)b2[i], c = cp[i], s = sp[i];
      y1[i] = (__bf16)(f1 * c - f2 * s);
      y2[i] = (__bf16)(f1 * s + f2 * c);
    }
    x1 = __builtin_bit_cast(u32x4, y1);
    x2 = __builtin_bit_cast(u32x4, y2);
  }
  st16(dst + 8 * j, x1);
  st16(dst + 8 * j + kHeadDim / 2, x2);
}

}  // namespace

hipError_t launch_paged_attn(const PagedArgs& a, hipStream_t stream) { return launch_paged_tiles<kPoolBf16, false>(a, stream); }

hipError_t launch_paged_rope(const PagedRopeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(paged_rope_kernel, dim3((unsigned)((a.total + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bd3
