// bd3_launch.h - argument blocks and launchers shared between the kernel
// translation units and the C-ABI layer (capi.hip). Internal to the library.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "bd3attn.h"

namespace bd3 {

constexpr int kHeadDim = 64;
constexpr int kBwdOrderMax = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Strides3 {
  int64_t b, h, s;  // element strides; the head_dim stride is 1
};

struct FwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* lse;  // contiguous (B, H, 2n), natural log
  Strides3 sq, sk, sv, so;
  int heads;
  int bh;  // batch * heads
  int n;
  int bs;
  int subs;  // sets of 4 waves per workgroup, 1 or 2
  float scale_log2;  // softmax scale * log2(e)
};

struct BwdArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* dout;
  const float* lse;  // natural log, contiguous (B, H, 2n)
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float* delta;  // 2 x (B, H, 2n) fp32: Delta, then -L / scale (the Delta pass writes both)
  // Work items of one batch*head, in launch order (host built, longest
  // first): code c < 2n/128 is dQ query tile c, otherwise dK/dV key tile
  // c - 2n/128 (see attn_bwd.hip). With more than kBwdOrderMax items the
  // codes run first_code, first_code + 1, ... instead.
  uint16_t order[256];
  int n_items;
  int first_code;
  // 1: the noisy key tiles' dK/dV (block sizes dividing 32, so only their
  // diagonal blocks are live) are formed at the end of the dQ items of the
  // same rows, and the launch holds no dK/dV item for them.
  int fold_diag;
  int subs;  // sets of 4 waves per workgroup, 1 or 2 (both kinds of items in the launch)
  Strides3 sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int heads;
  int bh;
  int n;
  int bs;
  float scale;       // softmax scale
  float scale_log2;  // scale * log2(e)
};

struct DecodeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  float* part_o;    // (BH, q_tiles, n_splits, QT, 64) fp32, or null
  float* part_lse;  // (BH, q_tiles, n_splits, QT) log2 LSE, or null
  Strides3 sq, sk, sv, so;
  int heads;
  int bh;
  int q_len;
  int kv_len;
  int bs;
  int n_splits;   // key ranges (workgroups per query tile and batch*head)
  int split_len;  // keys per split (multiple of 32)
  int subs;       // prefill: sets of 4 waves per workgroup, 1, 2 or 4
  int q_tiles;
  float scale_log2;
};

struct QkvRopeArgs {
  const uint16_t* qkv;  // (batch, seq, 3 * heads * 64), last stride 1
  int64_t sx_b, sx_s;
  const int64_t* positions;  // (seq) absolute positions, or null: pos0 + s
  int pos0;
  const float* sin_t;  // (max_pos, 32) fp32
  const float* cos_t;
  int max_pos;
  uint16_t* q;
  uint16_t* k;
  uint16_t* v;
  Strides3 sq, sk, sv;
  int heads;
  int seq;
  int64_t total;  // batch * seq * 4 * heads work items (< 2^31)
};

struct KvWriteArgs {
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* k_dst;
  uint16_t* v_dst;
  Strides3 sk, sv, skd, svd;
  int batch, heads, seq;
  int64_t total;  // 2 * batch * heads * seq * 8 16-byte parts
};

struct SubsArgs {
  const void* logits;  // (rows, ld) bf16 or fp32
  int64_t ld;          // row stride in elements
  int fp32;            // 1: fp32 logits, 0: bf16
  const int64_t* xt;   // (rows) current tokens
  int64_t* out;        // (rows) next tokens
  int rows, vocab;
  int mask_index;
  double keep;         // s / t
  const double* u;     // (rows, vocab) uniforms, or null: Philox4x32-10(seed, offset)
  uint64_t seed, offset;
  // Few rows: `spread` workgroups dealt out over the masked rows, at most
  // `slices` to a row, their results in ws (rows, slices) of kSubsSliceBytes;
  // 0: one workgroup per row, which needs no workspace.
  int spread, slices;
  void* ws;
};
constexpr size_t kSubsSliceBytes = 512;
constexpr int kSubsSpreadRows = 1024;  // most rows of a spread call

struct GlueArgs {
  const void* x;       // (batch, seq, d) rows, fp32 or bf16
  const void* weight;  // (d) LayerNorm gain
  const void* shift;   // (batch, d): shift (ln_modulate) or gate (gate_residual)
  const void* scale;   // (batch, d)
  const void* y;       // (batch, seq, d) sublayer output (gate_residual)
  void* out;
  const void* gate;    // (batch, d) gate of the fused residual + LayerNorm (stride sm_b)
  void* out_x;         // (batch, seq, d) updated residual of the fused form
  int x_fp32, w_fp32, m_fp32, y_fp32, out_fp32;
  int rows, seq, d;
  int64_t sx_b, sx_s, sm_b, sy_b, sy_s, so_b, so_s, sxo_b, sxo_s;  // element strides
  float eps;
  int wave_rows, wg_threads;  // set at the launch: rows per wave, threads per workgroup
  int row0;                   // first row of the launch (rows: the one past its last)
};

// Division of 0 <= n < 2^31 by a number d known at the launch: the upper word of n
// times m = floor(2^(31 + s) / d) + 1, 2^(s - 1) < d <= 2^s, exceeds n / d by n e / (d
// 2^(31 + s)) with 0 < e <= d <= 2^s, less than 1 / d, so its floor is exact.
struct FastDiv {
  uint32_t m;
  int s;  // -1: d is 1
  static FastDiv of(int d) {
    int s = 0;
    while (((int64_t)1 << s) < d) ++s;
    return s == 0 ? FastDiv{0, -1} : FastDiv{(uint32_t)(((uint64_t)1 << (31 + s)) / (uint32_t)d + 1), s - 1};
  }
};

constexpr int kMergeRows = 16;
constexpr int kPagedMaxKeys = 1 << 30;  // of a sequence: key positions stay below 2^31 when rounded up to a block
enum PoolType { kPoolBf16 = BD3_POOL_BF16, kPoolInt8 = BD3_POOL_INT8, kPoolE4m3 = BD3_POOL_E4M3 };
struct PagedArgs {
  const uint16_t* q;        // (tokens, heads, 64)
  const void* k;            // (pages, kv_heads, page, 64) bf16 or codes
  const void* v;
  const float* k_scales;    // 8-bit pools: (pages, kv_heads, page / 16)
  const float* v_scales;
  const int32_t* columns;   // (tokens, kv_heads, top) columns of the table, or null: all keys
  uint16_t* o;              // (tokens, heads, 64)
  const int32_t* table;     // (seqs, width) page numbers
  const int32_t* q_starts;  // (seqs + 1)
  const int32_t* kv_lens;   // (seqs)
  float* part_o;            // (kv_heads, part_rows, n_splits, 64) fp32, or null
  float* part_lse;          // (kv_heads, part_rows, n_splits) log2 LSE, or null
  int64_t sq_t, sq_h, sk_p, sk_h, sk_s, sv_p, sv_h, sv_s, so_t, so_h, table_s, sc_t, sc_h;  // element strides
  int seqs, tokens, kv_heads, group, pages, page, page_shift;
  int top;          // entries of a list
  int block_tiles;  // lists: tiles of a block of bs tokens
  int max_q;      // most tokens of a chunk: the caller's bound
  int max_kv;     // most keys of a sequence: the caller's bound, at most the table's
  int bs;
  FastDiv bs_div, group_div, kv_heads_div, tile_div;
  int tile;       // query rows per workgroup
  int subs;       // sets of 4 waves per workgroup: 1, 2 or (128-row tiles) 4
  int q_tiles;    // tiles of the longest chunk
  int part_slots;  // workgroups of the merge for a KV head: kMergeRows of its part_rows each
  int part_rows;   // tokens * group: the packed rows of a KV head, row q0 * group + r that of row r of a chunk at q0
  int n_splits;    // most key ranges of a tile
  int split_shift;  // log2 of about a range's keys
  int workgroups;
  // 128-row tiles, not cut: taken in the order of TileItem. level_step: 64^k levels
  // to a lane, so that 64 lanes cover them all.
  int sorted, level_step;
  FastDiv level_div;
  float scale_log2;
};

struct PagedRopeArgs {
  const uint16_t* qkv;  // (tokens, (heads + 2 kv_heads) * 64), last stride 1
  const float* sin_t;   // (max_pos, 32) fp32
  const float* cos_t;
  uint16_t* q;          // (tokens, heads, 64)
  void* k;              // (pages, kv_heads, page, 64) bf16 or codes
  void* v;
  float* k_scales;      // 8-bit pools: (pages, kv_heads, page / 16)
  float* v_scales;
  const int32_t* table;
  const int32_t* q_starts;
  const int32_t* kv_lens;
  int64_t sx_t, sq_t, sq_h, sk_p, sk_h, sk_s, sv_p, sv_h, sv_s, table_s;
  int seqs, tokens, heads, kv_heads, pages, page, page_shift, width, max_pos;
  int64_t total;  // tokens * (heads + 2 kv_heads) * 4 work items (< 2^31)
  int blocks;     // 8-bit pools: most blocks of 16 slots that the chunks touch
  FastDiv parts_div;
};

struct PageValuesArgs {
  const void* codes[2];      // k, v: (pages, kv_heads, page, 64)
  const float* scales[2];    // (pages, kv_heads, page / 16)
  uint16_t* out[2];          // (pages, kv_heads, page, 64) bf16, contiguous
  int64_t s_p[2], s_h[2], s_s[2];
  int kv_heads, blocks;      // blocks of a page
  int64_t total;             // blocks of 16 rows of one of the two
};

constexpr int kPickColumns = 2048;  // most that one workgroup scores and chooses from
// Whether a selection goes through a workspace: scored by as many workgroups as there are groups of 64 columns, then
// chosen from. With one launch and with two, us: 4 items of 187, 500, 1000 columns 11.1, 12.6; 12.2, 11.8; 15.7, 11.8; 24 of
// 500, 1000 15.1, 14.8; 18.8, 15.1; 96 14.7, 15.1; 20.5, 18.7; 192 17.2, 19.0; 21.5, 23.8.
inline bool select_in_two(int64_t items, int64_t width) { return width > kPickColumns || (items < 128 && width > 256); }
struct SelectArgs {
  PagedArgs p;               // batch, pool (bounds) and queries (selection)
  uint16_t* bounds;          // (pages, kv_heads, 2, 64): lowest and highest key
  int32_t* out;              // (tokens, kv_heads, top)
  int slots;                 // most pages that the chunks touch (bounds), most blocks of the chunks (selection)
  int width;                 // columns within max_kv
  int first, recent;         // columns always taken
  // Where select_in_two:
  uint32_t* keys;            // (slots, kv_heads, width): the scores as ordered numbers
  float* error;              // (slots, kv_heads, ceil(width / 16)): bound of the scores' distance from the exact sums
  double* sums;              // (slots, kv_heads, width)
};

constexpr int kLogitSlice = 2048;  // tokens of the vocabulary per workgroup of adjust_logits
struct LogitArgs {
  const void* logits;       // (batch, rows, vocab), fp32 or bf16
  void* out;
  const int64_t* tokens;    // (batch, history) or null
  const int32_t* lengths;   // (batch) or null: all of the history
  const float* repetition_p;  // (batch) each, or null: the scalar
  const float* frequency_p;
  const float* presence_p;
  const float* bias;        // (vocab) or (batch, vocab), or null
  const int32_t* allowed;   // bits, (words), (batch, words) or (batch, rows, words), or null
  int64_t in_b, in_r, out_b, out_r, tokens_s, bias_s, allowed_b, allowed_r;  // element strides
  int fp32;
  int batch, rows, vocab, history;
  float repetition, frequency, presence, fill;
  int slices, row_parts, part_rows;  // workgroups: vocabulary slices x parts of a sequence's rows x batch
};

// Launch shape of the kernels that walk rows (ln_modulate, the fused one), for
// each launch of `rows` rows (the last may have fewer).
struct GlueGrid {
  int wave_rows, threads, rows;
  unsigned workgroups;
};
GlueGrid glue_grid(int rows, int d);

hipError_t launch_attn_fwd(const FwdArgs& a, hipStream_t stream);
// The backward's Delta pass (Delta and -L / scale), then one launch of the
// items in a.order (dQ and / or dK/dV).
hipError_t launch_attn_bwd_delta(const BwdArgs& a, hipStream_t stream);
hipError_t launch_attn_bwd_items(const BwdArgs& a, hipStream_t stream);
hipError_t launch_decode(const DecodeArgs& a, int qt, hipStream_t stream);
hipError_t launch_prefill(const DecodeArgs& a, hipStream_t stream);
hipError_t launch_qkv_rope(const QkvRopeArgs& a, hipStream_t stream);
hipError_t launch_kv_write(const KvWriteArgs& a, hipStream_t stream);
hipError_t launch_subs_sample(const SubsArgs& a, hipStream_t stream);
hipError_t launch_paged_attn(const PagedArgs& a, hipStream_t stream);
hipError_t launch_paged_pool(const PagedArgs& a, int pool, hipStream_t stream);  // 8-bit pools, lists
hipError_t launch_paged_rope(const PagedRopeArgs& a, hipStream_t stream);
hipError_t launch_paged_rope8(const PagedRopeArgs& a, int pool, hipStream_t stream);
hipError_t launch_page_values(const PageValuesArgs& a, int pool, hipStream_t stream);
hipError_t launch_page_bounds(const SelectArgs& a, int pool, hipStream_t stream);
hipError_t launch_select_pages(const SelectArgs& a, hipStream_t stream);
hipError_t launch_adjust_logits(const LogitArgs& a, hipStream_t stream);
hipError_t launch_ln_modulate(const GlueArgs& a, hipStream_t stream);
hipError_t launch_gate_residual_ln_modulate(const GlueArgs& a, hipStream_t stream);
hipError_t launch_gate_residual(const GlueArgs& a, hipStream_t stream);
hipError_t launch_mask_dump(uint8_t* out, int mode, int rows, int kv_len,
                            int bs, hipStream_t stream);
hipError_t launch_clock_probe(uint64_t* out, int workgroups, int iters, hipStream_t stream);

}  // namespace bd3
