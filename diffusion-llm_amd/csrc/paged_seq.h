// paged_seq.h - what a workgroup learns of a ragged batch from the device arrays
// that describe it: a sequence's share, bounded, its blocks, and which sequence the
// j-th piece of work belongs to.
#pragma once

#include "bd3_device.h"
#include "bd3_launch.h"

namespace bd3 {
namespace {

typedef const __attribute__((address_space(1))) u32x4 global_u32x4;

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

__device__ __forceinline__ int fast_div(int n, FastDiv d) {
  return d.s < 0 ? n : (int)(__umulhi((uint32_t)n, d.m) >> d.s);
}

// One sequence's share of the batch, bounded (see above).
struct PagedSeq {
  int q0, n, kv, rows;
  PagedSeq() = default;
  __device__ __forceinline__ PagedSeq(const PagedArgs& a, int b) {
    q0 = clampi(a.q_starts[b], 0, a.tokens);
    n = clampi(a.q_starts[b + 1], q0, a.tokens) - q0;
    kv = clampi(a.kv_lens[b], 0, a.max_kv);
    rows = (n < a.max_q ? n : a.max_q) * a.group;  // what the launch and its partials have room for
  }
  __device__ __forceinline__ PagedSeq of_lane(int lane) const {
    PagedSeq r;
    r.q0 = __builtin_amdgcn_readlane(q0, lane);
    r.n = __builtin_amdgcn_readlane(n, lane);
    r.kv = __builtin_amdgcn_readlane(kv, lane);
    r.rows = __builtin_amdgcn_readlane(rows, lane);
    return r;
  }
  // Place of a row's partial of one range: the packed rows of a KV head after those of
  // the head before it, a row's ranges side by side. So partials take what the
  // tokens there are need, however long the longest chunk is. (With the ranges outermost
  // 32 sequences of 16 rows took 0.6 us more: writes 128 KB apart.) At most 2^20
  // places: kPagedPartRows.
  __device__ __forceinline__ int part_row(const PagedArgs& a, int h, int split, int r0) const {
    return (h * a.part_rows + q0 * a.group + r0) * a.n_splits + split;
  }
  // First position and block of the chunk's tokens (before 0 if it has more tokens than keys).
  __device__ __forceinline__ int first_pos() const { return kv - n; }
  __device__ __forceinline__ static int block_of(const PagedArgs& a, int p) {  // rounded down
    return p < 0 ? -1 - fast_div(-1 - p, a.bs_div) : fast_div(p, a.bs_div);
  }
  // Blocks of the chunk's tokens, those within the caller's bound.
  __device__ __forceinline__ int blocks(const PagedArgs& a) const {
    const int m = n < a.max_q ? n : a.max_q;
    return m > 0 ? block_of(a, kv - n + m - 1) - block_of(a, kv - n) + 1 : 0;
  }
  // The chunk's tokens of its g-th block: [lo, hi), bounded like rows.
  __device__ __forceinline__ void block_tokens(const PagedArgs& a, int g, int& lo, int& hi) const {
    const int m = n < a.max_q ? n : a.max_q;
    const int64_t at = ((int64_t)block_of(a, kv - n) + g) * a.bs - ((int64_t)kv - n);
    lo = at < 0 ? 0 : (at < m ? (int)at : m);
    hi = at + a.bs < m ? (int)(at + a.bs) : m;
  }
  // Keys of the longest list of the sequence's blocks.
  __device__ __forceinline__ int listed_keys(const PagedArgs& a) const {
    const int cols = (int)(((int64_t)kv + a.page - 1) >> a.page_shift);
    return (cols < a.top ? cols : a.top) << a.page_shift;
  }
  // Keys that token i sees: [0, key_end).
  __device__ __forceinline__ int key_end(const PagedArgs& a, int i) const {
    const int p = kv - n + i;
    const int e = (fast_div(p < 0 ? 0 : p, a.bs_div) + 1) * a.bs;
    return p < 0 ? 0 : (e < kv ? e : kv);
  }
  // One past the last key of the tile of `tile` rows at row r0 (r0 < rows).
  __device__ __forceinline__ int tile_end(const PagedArgs& a, int r0) const {
    const int last = (r0 + a.tile < rows ? r0 + a.tile : rows) - 1;
    return wave_uniform(key_end(a, fast_div(last, a.group_div)));
  }
};

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
  return v;
}

// Piece j of those that count(sequence) numbers, in the order of the sequences: the
// sequence it belongs to and its place among that one's. `seq(b)` reads a sequence, a
// lane each.
template <class Seq>
struct SeqPiece {
  int b, at;
  Seq sq;
  bool found;
  template <class Read, class Count>
  __device__ __forceinline__ SeqPiece(int seqs, int j, Read read, Count count) : b(0), at(0), sq(), found(false) {
    const int lane = wi_x() & 63;
    int before = 0;
    for (int s0 = 0; s0 < seqs; s0 += 64) {
      Seq mine = {};
      int n = 0;
      if (s0 + lane < seqs) {
        mine = read(s0 + lane);
        n = count(mine);
      }
      const int upto = wave_scan(n);
      const int k = __popcll(__ballot(before + upto <= j));
      if (k < 64) {
        b = s0 + k;
        at = j - before - (__builtin_amdgcn_readlane(upto, k) - __builtin_amdgcn_readlane(n, k));
        sq = mine.of_lane(k);
        found = true;
        return;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
};

// A signed byte of a word to fp32, in one instruction (from C++ the compiler makes one and a half).
template <int BYTE>
__device__ __forceinline__ float byte_f32(uint32_t w) {
  float x;
  if constexpr (BYTE == 0)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(x) : "v"(w));
  else if constexpr (BYTE == 1)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(x) : "v"(w));
  else if constexpr (BYTE == 2)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(x) : "v"(w));
  else
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(x) : "v"(w));
  return x;
}

// Codes to fp32 and bf16 (exactly), four to a word.
template <int POOL>
__device__ __forceinline__ f32x4 codes_f32(uint32_t w) {
  if constexpr (POOL == kPoolInt8) {
    return f32x4{byte_f32<0>(w), byte_f32<1>(w), byte_f32<2>(w), byte_f32<3>(w)};
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return f32x4{lo[0], lo[1], hi[0], hi[1]};
  }
}
template <int POOL>
__device__ __forceinline__ bf16x4 codes4(uint32_t w) {
  if constexpr (POOL == kPoolInt8) {
    const f32x4 x = codes_f32<POOL>(w);
    return to_bf16x4(x[0], x[1], x[2], x[3]);
  } else {
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3);
  }
}

}  // namespace
}  // namespace bd3
