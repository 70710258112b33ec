// paged_tiles.h - attention of ragged batches over a paged KV cache: the tiles, as
// templates over what the pool holds (bf16, or 8-bit codes with scales) and over
// whether every key is read or only the pages of a list.
//
// Sequence b owns the packed tokens q_starts[b] .. q_starts[b + 1] - 1 (n of
// them) and kv = kv_lens[b] keys, the chunk's own included; key j lies in slot
// j % page of page page_table[b][j / page]. Token i is at position p = kv - n + i
// and sees keys j < min((p / bs + 1) * bs, kv), none if p < 0. `group` query heads
// share a KV head: their rows are one matrix of n * group rows, row r token
// r / group of head h * group + r % group, so a page is read once for all of them.
//
// O = softmax(q K^T * scale) V over the keys seen, in one pass over the pages with a
// running maximum and sum (fp32, base 2) per row; probabilities are rounded to bf16
// for the second product (relative 2^-8 each, as in every attention kernel here),
// the result once. Long sequences are cut into key ranges whose fp32 partials a
// second launch merges.
//
// The lengths and the table are device data, so workgroups find their items from
// them (PagedItem, TileItem). Everything read through device data is bounded: token
// ranges by the tokens there are, lengths by the table and the caller's bound, page
// numbers by the pages there are. Keys of an entry outside [0, pages) are not seen
// (their rows come from a zero row, their scores are masked); keys past the length
// re-read the last one, so nothing that a page holds behind it comes in.
//
// 8-bit pools hold a code (int8 or e4m3) per element and an fp32 scale per 16 slots and
// head, value = scale * code. A code is exact in bf16, so the products run on codes:
// the scale of 16 keys is a factor of their scores, which the softmax applies with
// its own (one fma either way), and that of 16 values one of their
// probabilities, in fp32 before they are rounded. No value is rounded on the way in.
//
// Lists (COLS): the queries of one block of bs positions read the pages in the table's
// columns columns[first token of the block in the chunk][KV head], at most `top` of
// them, in that order; what is masked is the same. Tiles then hold rows of one
// block, and "keys" of a range count along the list, column after column.
#pragma once

#include "bd3_swz.h"
#include "paged_seq.h"

namespace bd3 {
namespace {

constexpr int kQT = 32;       // rows of the 32-row tile
constexpr int kSub = 32;      // keys per wave step
constexpr int kStride = 72;   // padded LDS row (bf16)
constexpr int kMergeRow = kHeadDim + 4;
constexpr float kRescale = 8.0f;  // log2: growth of a running maximum that is let pass

__device__ __attribute__((aligned(128))) uint16_t zero_row[kHeadDim];

// How a sequence of kv keys is cut into ranges of `len` keys; a tile that sees only
// some of the keys has fewer of them.
// Plain (16- and 32-row tiles): 2^split_shift keys, up to half a range more in the last one.
// EVEN (128-row tiles): about 2^split_shift keys, whole 64-key tiles, as many in every
// range but the last: the plain form let the longest items end 4 us after the others
// (96 rows over 500-4000 keys of 24 sequences, 512-key ranges: 30 us, 24 so). The
// shorter launches lose 0.5 us to its arithmetic and gain nothing. Its quotients are
// products with a reciprocal, made exact where it matters.
template <bool EVEN>
struct KeySplit {
  int len, shift;
  __device__ __forceinline__ KeySplit(const PagedArgs& a, int kv) : len(1 << a.split_shift), shift(a.split_shift) {
    if constexpr (EVEN) {
      const int n = (kv + (1 << shift >> 1)) >> shift;
      len = kv;
      // at least kv / n: 2^-20 more than covers the reciprocal's and the product's errors
      if (n > 1) len = (int)((float)kv * __builtin_amdgcn_rcpf((float)n) * 1.000001f) + 1;
      len = (len + kSwRows - 1) & -kSwRows;
    }
  }
  __device__ __forceinline__ int ranges(int keys) const {  // at least 1
    if constexpr (EVEN) {  // ceil(keys / len): the estimate's floor is at most two below it
      int q = (int)((float)keys * __builtin_amdgcn_rcpf((float)(len > 1 ? len : 1)));
      q += q * len < keys;
      q += q * len < keys;
      return q > 1 ? q : 1;
    }
    const int q = (keys + (1 << shift >> 1)) >> shift;
    return q > 1 ? q : 1;
  }
};

// What a chunk's two halves of 16 keys are: whether their page is there, the position of
// their first key.
struct ChunkInfo {
  uint32_t there;
  int base[2];
};

// The 32-key chunks of one key range that one of NW waves takes in turn (chunks
// wave, wave + NW, ...): from the pages to registers, the next chunk's loads in
// flight while the last one, staged in the wave's LDS tiles, is computed.
template <int NW, bool COLS>
struct ChunkStream {
  const PagedArgs& a;
  const int32_t* table;
  const int32_t* list;  // COLS: the block's columns
  const uint16_t *kh, *vh;  // the head's rows of page 0
  int lo, hi, end, wave, lane, mine;
  int ids;        // lane 2 i + half: page of the half's 16 keys (a page holds at least 16) of chunk base + i
  int at_key;     // COLS: position of the first of them
  uint64_t ok;    // which of them exist
  u32x4 kr[4], vr[4];  // lane + 64 j -> key row 8 j + lane / 8 of the chunk, 16-byte part lane % 8
  ChunkInfo info;      // of the loaded chunk

  // Keys lo .. hi - 1 of the range (of the list, COLS); none from `end` on is a key of the rows.
  __device__ __forceinline__ ChunkStream(const PagedArgs& a_, int b, int h_, const int32_t* list_, int lo_, int hi_,
                                         int end_, int wave_, int lane_)
      : a(a_), list(list_), lo(lo_), hi(hi_), end(end_), wave(wave_), lane(lane_), info() {
    table = a.table + (int64_t)b * a.table_s;
    kh = static_cast<const uint16_t*>(a.k) + h_ * a.sk_h;
    vh = static_cast<const uint16_t*>(a.v) + h_ * a.sv_h;
    const int n = hi > lo ? (hi - lo + kSub - 1) / kSub : 0;
    mine = n > wave ? (n - wave + NW - 1) / NW : 0;
  }
  __device__ __forceinline__ int first_key(int i) const { return lo + (wave + NW * i) * kSub; }
  __device__ __forceinline__ void find(int i) {  // pages of 32 chunks
    int key = first_key(i + (lane >> 1)) + 16 * (lane & 1);
    ids = -1;
    if (key < hi) {
      if constexpr (COLS) {
        const int col = list[key >> a.page_shift];
        const int cols = (int)(((int64_t)end + a.page - 1) >> a.page_shift);
        const bool is = (unsigned)col < (unsigned)cols;
        key = ((is ? col : 0) << a.page_shift) + (key & (a.page - 1));
        if (is && key < end) ids = table[col];
      } else {
        ids = table[key >> a.page_shift];
      }
    }
    if constexpr (COLS) at_key = key;
    ok = __ballot((unsigned)ids < (unsigned)a.pages);
  }
  __device__ __forceinline__ void load(int i) {
    if ((i & 31) == 0) find(i);
    info.there = (uint32_t)(ok >> (2 * (i & 31))) & 3u;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int at = 2 * (i & 31) + hh;
      const int key = COLS ? __builtin_amdgcn_readlane(at_key, at) : first_key(i) + 16 * hh;
      info.base[hh] = key;
      const bool is = (info.there >> hh) & 1;
      const int64_t page = __builtin_amdgcn_readlane(ids, at);
      const int64_t slot = key & (a.page - 1);
      const uint64_t kb = (uint64_t)(uintptr_t)(is ? kh + page * a.sk_p + slot * a.sk_s : zero_row);
      const uint64_t vb = (uint64_t)(uintptr_t)(is ? vh + page * a.sv_p + slot * a.sv_s : zero_row);
      const int last = is ? (COLS ? end : hi) - 1 - key : 0;  // rows past the last key re-read it
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int mine = (lane >> 3) + 8 * j, part = 16 * (lane & 7);
        const int r = mine < last ? mine : last;
        kr[2 * hh + j] = __builtin_nontemporal_load((global_u32x4*)(kb + (uint32_t)(2 * r * (int)a.sk_s + part)));
        vr[2 * hh + j] = __builtin_nontemporal_load((global_u32x4*)(vb + (uint32_t)(2 * r * (int)a.sv_s + part)));
      }
    }
  }
  // Whether some row does not see some key of the chunk.
  __device__ __forceinline__ bool masked(const ChunkInfo& c, int kfull) const {
    if constexpr (COLS) return c.base[0] + 16 > kfull || c.base[1] + 16 > kfull || c.there != 3;
    return c.base[0] + kSub > kfull || c.base[0] + kSub > hi || c.there != 3;
  }
  __device__ __forceinline__ void stage(__bf16* ks, __bf16* vs) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int off = (8 * j + (lane >> 3)) * kStride + 8 * (lane & 7);
      *reinterpret_cast<u32x4*>(&ks[off]) = kr[j];
      *reinterpret_cast<u32x4*>(&vs[off]) = vr[j];
    }
  }
};

// Item `id` of the list: KV head (fastest), row tile, range, in the order of the
// sequences. Every sequence has items of its own number, so the list
// is made here from the lengths, a lane a sequence: a launch of the most items that
// the bounds allow spent about 1 ns on each empty workgroup (32 sequences of
// 100-8192 keys, 12 heads: 67 us at the best range length, 55 with the list).
template <bool EVEN, bool COLS>
struct PagedItem {
  int b, h, split;
  int r0, r1;            // the tile's rows of the chunk
  const int32_t* list;   // COLS: the block's columns
  PagedSeq sq;
  int total;  // items of all, or (more than 64 sequences) INT_MAX while not known
  bool found;
  __device__ __forceinline__ PagedItem(const PagedArgs& a, int id) {
    const int lane = wi_x() & 63;
    const int j = wave_uniform(fast_div(id, a.kv_heads_div));
    h = id - j * a.kv_heads;
    found = false;
    int before = 0;  // items of the sequences up to s0, of one head
    for (int s0 = 0; s0 < a.seqs; s0 += 64) {
      PagedSeq mine = {};
      int items = 0, tiles = 0;
      if (s0 + lane < a.seqs) {
        mine = PagedSeq(a, s0 + lane);
        tiles = COLS ? mine.blocks(a) * a.block_tiles : (mine.rows + a.tile - 1) / a.tile;
        const int keys = COLS ? mine.listed_keys(a) : mine.kv;
        items = tiles * KeySplit<EVEN>(a, keys).ranges(keys);
      }
      const int upto = wave_scan(items);
      const int at = __popcll(__ballot(before + upto <= j));
      total = s0 + 64 < a.seqs ? INT32_MAX : (before + __builtin_amdgcn_readlane(upto, 63)) * a.kv_heads;
      if (at < 64) {
        int rem = j - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(items, at));
        const int t = __builtin_amdgcn_readlane(tiles, at);
        b = s0 + at;
        sq = mine.of_lane(at);
        for (split = 0; rem >= t; rem -= t) ++split;
        found = true;
        if constexpr (COLS) {
          const int g = rem / a.block_tiles;
          int lo, hi;
          sq.block_tokens(a, g, lo, hi);
          r0 = lo * a.group + (rem - g * a.block_tiles) * a.tile;
          r1 = hi * a.group;
          list = a.columns + (int64_t)(sq.q0 + lo) * a.sc_t + h * a.sc_h;
        } else {
          r0 = rem * a.tile;
          r1 = sq.rows;
          list = nullptr;
        }
        r1 = r1 < r0 + a.tile ? r1 : r0 + a.tile;  // no rows: a block shorter than others
        return;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
  }
};

// Tile `j` of all sequences' 128-row tiles of one head, those that see most keys
// first (up to 64 sequences). A sequence's tiles, last one first, see kv, kv - u, kv
// - 2 u, ... keys (u tokens a tile), so its r-th one belongs to level (max_kv - kv) /
// u + r, and the tiles below level l number the sum of clamp(l - first level, 0,
// tiles). Each lane forms that sum for a level of its own, 64 levels at a time.
struct TileItem {
  int b, rank;
  PagedSeq sq;
  bool found;
  __device__ __forceinline__ TileItem(const PagedArgs& a, int j) {
    const int lane = wi_x() & 63;
    found = false;
    PagedSeq mine = {};
    if (lane < a.seqs) mine = PagedSeq(a, lane);
    const int tiles = (mine.rows + 127) / 128;
    const int first = fast_div(a.max_kv - mine.kv, a.level_div);
    auto below = [&](int level) {  // every lane for its own level
      int sum = 0;
      for (int s = 0; s < a.seqs; ++s) {
        const int c = level - __builtin_amdgcn_readlane(first, s), t = __builtin_amdgcn_readlane(tiles, s);
        sum += c < 0 ? 0 : (c < t ? c : t);
      }
      return sum;
    };
    // The last level with at most j tiles below it: `step` levels to a lane, then 1.
    int at = 0, before = 0;
    for (int step = a.level_step; step > 0; step >>= 6) {
      const int sum = below(at + step * lane);
      const int n = __popcll(__ballot(sum <= j)) - 1;  // lane 0's sum is at most j
      at += step * n;
      before = __builtin_amdgcn_readlane(sum, n);
    }
    const int nth = j - before;  // of the level's tiles
    const bool live = at >= first && at < first + tiles;
    const uint64_t all = __ballot(live);
    const int mine_th = __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
    const uint64_t it = __ballot(live && mine_th == nth);
    if (it == 0) return;  // j is past the last tile
    b = __builtin_ctzll(it);
    sq = mine.of_lane(b);
    rank = at - __builtin_amdgcn_readlane(first, b);
    found = true;
  }
};

// The waves' states, unnormalised, merged by threads of 4 d each (16 a row): to the
// result where the tile has one range, else to its partial.
template <int NW, int ROWS>
struct MergeLds {
  float o[NW][ROWS][kMergeRow];
  float m[NW][ROWS];
  float l[NW][ROWS];
  template <class Item>
  __device__ __forceinline__ void write_row(const PagedArgs& a, int ranges, const Item& it, int rt, int d,
                                            int first = 0) const {  // first: row of the tile that the states begin with
    float mw[NW], mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      mw[w] = m[w][rt];
      mm = fmaxf(mm, mw[w]);
    }
    const float mu = (mm == -INFINITY) ? 0.f : mm;
    float lt = 0.f;
    f32x4 ot = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float wgt = fast_exp2(mw[w] - mu);
      lt += wgt * l[w][rt];
      ot += wgt * *reinterpret_cast<const f32x4*>(&o[w][rt][d]);
    }
    const float inv = lt > 0.f ? 1.f / lt : 0.f;  // a row that sees no key: 0
    const int row = it.r0 + first + rt;
    if (ranges == 1) {
      if (row < it.r1) {
        const int t = fast_div(row, a.group_div);
        *reinterpret_cast<bf16x4*>(a.o + (int64_t)(it.sq.q0 + t) * a.so_t +
                                   (int64_t)(it.h * a.group + row - t * a.group) * a.so_h + d) =
            to_bf16x4(ot[0] * inv, ot[1] * inv, ot[2] * inv, ot[3] * inv);
      }
    } else {
      if (row >= it.r1) return;
      const int at = it.sq.part_row(a, it.h, it.split, row);
      *reinterpret_cast<f32x4*>(&a.part_o[at * kHeadDim + d]) = ot * inv;
      if (d == 0) a.part_lse[at] = lt > 0.f ? mm + fast_log2(lt) : -INFINITY;
    }
  }
};
// 8-bit pools: chunks of KC keys (groups of 16, each in one page under one scale) that one of NW waves takes
// in turn: from the pages to registers, full rows (4 lanes a row of 64 codes), the next chunk's
// loads in flight while the last one is computed from the wave's LDS tile. Codes stay bytes there:
// the 16-byte part p of row r lies at part p ^ (r / 4 % 4), so that the row reads (16 rows, one part)
// and the transposed ones (8 rows, one part, twice) meet every bank once.
template <int NW, int KC, int POOL, bool COLS>
struct CodeStream {
  static constexpr int kGroups = KC / 16;
  static constexpr int kFound = 64 / kGroups;  // chunks whose pages are looked up at once
  static constexpr int kTile = KC * kHeadDim;  // bytes
  const PagedArgs& a;
  const int32_t* table;
  const int32_t* list;  // COLS: the block's columns
  const uint8_t *kh, *vh;  // the head's rows of page 0
  int h, lo, hi, end, wave, lane, mine;
  int ids;        // lane kGroups i + g: page of group g of chunk base + i
  int at_key;     // COLS: position of its first key
  float k_scale, v_log, v_inv;
  uint64_t ok;    // which of them exist
  u32x4 kr[kGroups], vr[kGroups];  // row lane / 4 of the group, part lane % 4
  struct Info {
    uint32_t there;
    int base[kGroups];
    float ks[kGroups], v_log[kGroups], v_inv[kGroups];  // K's scales, log2 and inverse of V's
  } info;  // of the loaded chunk

  __device__ __forceinline__ CodeStream(const PagedArgs& a_, int b, int h_, const int32_t* list_, int lo_, int hi_, int end_,
                                        int wave_, int lane_)
      : a(a_), list(list_), h(h_), lo(lo_), hi(hi_), end(end_), wave(wave_), lane(lane_), info() {
    table = a.table + (int64_t)b * a.table_s;
    kh = static_cast<const uint8_t*>(a.k) + h * a.sk_h;
    vh = static_cast<const uint8_t*>(a.v) + h * a.sv_h;
    const int n = hi > lo ? (hi - lo + KC - 1) / KC : 0;
    mine = n > wave ? (n - wave + NW - 1) / NW : 0;
  }
  __device__ __forceinline__ int first_key(int i) const { return lo + (wave + NW * i) * KC; }
  __device__ __forceinline__ void find(int i) {
    int key = first_key(i + lane / kGroups) + 16 * (lane % kGroups);
    ids = -1;
    if (key < hi) {
      if constexpr (COLS) {
        const int col = list[key >> a.page_shift];
        const int cols = (int)(((int64_t)end + a.page - 1) >> a.page_shift);
        const bool is = (unsigned)col < (unsigned)cols;
        key = ((is ? col : 0) << a.page_shift) + (key & (a.page - 1));
        if (is && key < end) ids = table[col];
      } else {
        ids = table[key >> a.page_shift];
      }
    }
    if constexpr (COLS) at_key = key;
    const bool is = (unsigned)ids < (unsigned)a.pages;
    ok = __ballot(is);
    k_scale = 1.f;
    float v_scale = 1.f;
    if (is) {
      const int64_t at = ((int64_t)ids * a.kv_heads + h) * (a.page >> 4) + ((key & (a.page - 1)) >> 4);
      k_scale = a.k_scales[at];
      v_scale = a.v_scales[at];
    }
    v_log = fast_log2(v_scale);
    v_inv = __builtin_amdgcn_rcpf(v_scale);
  }
  __device__ __forceinline__ void load(int i) {
    const int turn = i % kFound;
    if (turn == 0) find(i);
    info.there = (uint32_t)(ok >> (kGroups * turn)) & ((1u << kGroups) - 1);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int at = kGroups * turn + g;
      const int key = COLS ? __builtin_amdgcn_readlane(at_key, at) : first_key(i) + 16 * g;
      info.base[g] = key;
      const bool is = (info.there >> g) & 1;
      const int64_t page = __builtin_amdgcn_readlane(ids, at);
      const int64_t slot = key & (a.page - 1);
      const uint64_t kb = (uint64_t)(uintptr_t)(is ? kh + page * a.sk_p + slot * a.sk_s : (const uint8_t*)zero_row);
      const uint64_t vb = (uint64_t)(uintptr_t)(is ? vh + page * a.sv_p + slot * a.sv_s : (const uint8_t*)zero_row);
      const int last = is ? (COLS ? end : hi) - 1 - key : 0;  // rows past the last key re-read it
      const int r = (lane >> 2) < last ? lane >> 2 : last;
      kr[g] = __builtin_nontemporal_load((global_u32x4*)(kb + (uint32_t)(r * (int)a.sk_s + 16 * (lane & 3))));
      vr[g] = __builtin_nontemporal_load((global_u32x4*)(vb + (uint32_t)(r * (int)a.sv_s + 16 * (lane & 3))));
    }
    // The scales last: the first chunk's are on their way with its codes.
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      info.ks[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k_scale), kGroups * turn + g));
      info.v_log[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_log), kGroups * turn + g));
      info.v_inv[g] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_inv), kGroups * turn + g));
    }
  }
  __device__ __forceinline__ void stage(uint8_t* ks, uint8_t* vs) const {
    const int at = (lane >> 2) * 64 + 16 * ((lane & 3) ^ (lane >> 4));
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      *reinterpret_cast<u32x4*>(&ks[1024 * g + at]) = kr[g];
      *reinterpret_cast<u32x4*>(&vs[1024 * g + at]) = vr[g];
    }
  }
  // Codes 16 hq .. + 15 of key lane % 16 of group g (hq = lane / 16).
  __device__ __forceinline__ u32x4 key_codes(const uint8_t* ks, int g) const {
    const int r = lane & 15;
    return *reinterpret_cast<const u32x4*>(&ks[1024 * g + 64 * r + 16 * ((lane >> 4) ^ (r >> 2))]);
  }
  // Codes of column 16 db + lane % 16 of the keys 4 hq .. + 3 of groups 2 h2 and 2 h2 + 1: the order of the scores in
  // the registers.
  __device__ __forceinline__ bf16x8 value_codes(const uint8_t* vs, int h2, int db) const {
    const int s = lane & 15, hq = lane >> 4;
    const int r = 4 * hq + ((s >> 1) & 3);  // row of the group, s / 8 the group
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    const i32x2 w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
        (lds_i32x2*)(&vs[1024 * (2 * h2 + (s >> 3)) + 64 * r + 16 * (db ^ hq) + 8 * (s & 1)]));
    return cat8(codes4<POOL>((uint32_t)w[0]), codes4<POOL>((uint32_t)w[1]));
  }
  // Whether some row does not see some key of the chunk.
  __device__ __forceinline__ bool masked(const Info& c, int kfull) const {
    bool m = c.there != (1u << kGroups) - 1;
    if constexpr (COLS) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) m = m || c.base[g] + 16 > kfull;
      return m;
    }
    return m || c.base[0] + KC > kfull || c.base[0] + KC > hi;
  }
};

template <int NW, int ROWS>
constexpr size_t chunk_smem() {
  constexpr size_t v = sizeof(__bf16) * NW * 2 * kSub * kStride;
  return v > sizeof(MergeLds<NW, ROWS>) ? v : sizeof(MergeLds<NW, ROWS>);
}

// The keys of an item: its range of those that its rows see, of `ranges` in all.
template <bool COLS>
struct ItemKeys {
  int ranges, lo, hi, end;
  bool any;  // an item past a tile's last range has none and writes nothing
  __device__ __forceinline__ ItemKeys(const PagedArgs& a, const PagedItem<false, COLS>& it) {
    end = wave_uniform(it.sq.key_end(a, fast_div(it.r1 - 1, a.group_div)));
    const int keys = COLS ? it.sq.listed_keys(a) : end;
    const KeySplit<false> cut(a, keys);
    ranges = cut.ranges(keys);
    any = it.split < ranges;
    lo = it.split << cut.shift;
    hi = it.split + 1 < ranges ? lo + cut.len : keys;
    if constexpr (COLS) {
      // A list ends with its last column; the places behind it hold none.
      const int lane = wi_x() & 63;
      int cols = 0;
      for (int s0 = lo >> a.page_shift; s0 << a.page_shift < hi; s0 += 64) {
        const bool is = s0 + lane < a.top && (s0 + lane) << a.page_shift < hi && it.list[s0 + lane] >= 0;
        const uint64_t all = __ballot(is);
        if (all != 0) cols = s0 + 64 - __builtin_clzll(all);
      }
      hi = hi < cols << a.page_shift ? hi : cols << a.page_shift;
    }
  }
};

// 32-row tiles: NW waves share the key chunks of a range. S^T (32 keys x 32 rows) =
// K Q^T on v_mfma_f32_32x32x16_bf16 with the K tile's rows as A operands; O^T += V^T
// P^T with V read transposed. Eight waves for few items (one workgroup a CU at 160
// registers), four for many (three a CU), each at its best ranges: 32 rows over 500-2000
// keys of 8 sequences 13.9 us against 15.1; over 4032 keys of 48 sequences 111, 104.
// At four waves per SIMD it spills (43 -> 50 us). Full launches are bound by HBM (32
// sequences x 4128 keys 73 us, 5.6 TB/s; contiguous 65).
template <int NW, bool COLS>
__device__ __forceinline__ void paged32_item(const PagedArgs& a, const PagedItem<false, COLS>& it, char* smem) {
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform(tid >> 6);
  const int l32 = lane & 31;
  const int g = lane >> 5;
  __bf16* ks = reinterpret_cast<__bf16*>(smem) + wave * 2 * kSub * kStride;
  __bf16* vs = ks + kSub * kStride;

  const PagedSeq& sq = it.sq;
  const ItemKeys<COLS> keys(a, it);
  if (!keys.any) return;
  // Q^T B operand: lane holds row r0 + l32 (clamped), d = 16c + 8g .. +7.
  const int row = it.r0 + l32 < it.r1 ? it.r0 + l32 : it.r1 - 1;
  const int tok = fast_div(row, a.group_div);
  const uint16_t* qp = a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(it.h * a.group + row - tok * a.group) * a.sq_h;
  bf16x8 qreg[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) qreg[c] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * c + 8 * g));
  const int ends = sq.key_end(a, tok);
  const int khi = COLS || ends < keys.hi ? ends : keys.hi;
  const int kfull = wave_uniform(sq.key_end(a, fast_div(it.r0, a.group_div)));  // every row of the tile sees these
  ChunkStream<NW, COLS> kv(a, it.b, it.h, it.list, keys.lo, keys.hi, keys.end, wave, lane);
  if (kv.mine > 0) kv.load(0);
  // Q is waited for here: in the loop the wait would be for the next chunk as well.
#pragma unroll
  for (int c = 0; c < 4; ++c) asm volatile("" ::"v"(qreg[c]));

  f32x16 oacc[2] = {};
  float m = -INFINITY, lsum = 0.f;
  const int tr_row = (lane & 15) >> 2;
  const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  for (int i = 0; i < kv.mine; ++i) {
    const ChunkInfo info = kv.info;
    kv.stage(ks, vs);
    if (i + 1 < kv.mine) kv.load(i + 1);
    // A = K rows from the tile (lane: key l32, d 16c + 8g .. +7).
    f32x16 s = {};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      s = mfma32(*reinterpret_cast<const bf16x8*>(&ks[l32 * kStride + 16 * c + 8 * g]), qreg[c], s);
    if (kv.masked(info, kfull)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = info.base[r >> 3] + 8 * ((r >> 2) & 1) + 4 * g + (r & 3);
        s[r] = key < khi && ((info.there >> (r >> 3)) & 1) ? s[r] : -INFINITY;
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[r]);
    mt = max_xor32(mt) * a.scale_log2;
    if (__ballot(mt > m) != 0) {
      const float mn = fmaxf(m, mt);
      const float alpha = (mn == -INFINITY) ? 1.f : fast_exp2(m - mn);
      m = mn;
      lsum *= alpha;
      oacc[0] *= alpha;
      oacc[1] *= alpha;
    }
    const float mu = (m == -INFINITY) ? 0.f : m;
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = fast_exp2(fmaf(s[r], a.scale_log2, -mu));
      lsum += p[r];
    }
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      const bf16x8 pop = to_bf16x8(p[8 * kc], p[8 * kc + 1], p[8 * kc + 2], p[8 * kc + 3],
                                   p[8 * kc + 4], p[8 * kc + 5], p[8 * kc + 6], p[8 * kc + 7]);
      const int vrow = 16 * kc + 4 * g + tr_row;
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const bf16x8 va = cat8(lds_read_tr(&vs[vrow * kStride + 32 * db + tr_col]),
                               lds_read_tr(&vs[(vrow + 8) * kStride + 32 * db + tr_col]));
        oacc[db] = mfma32(va, pop, oacc[db]);
      }
    }
  }

  lsum = sum_xor32(lsum);
  __syncthreads();  // the tiles are reused below
  auto* ml = reinterpret_cast<MergeLds<NW, kQT>*>(smem);
#pragma unroll
  for (int db = 0; db < 2; ++db)
#pragma unroll
    for (int rg = 0; rg < 4; ++rg)
      *reinterpret_cast<f32x4*>(&ml->o[wave][l32][32 * db + 8 * rg + 4 * g]) =
          f32x4{oacc[db][4 * rg], oacc[db][4 * rg + 1], oacc[db][4 * rg + 2], oacc[db][4 * rg + 3]};
  if (g == 0) {
    ml->m[wave][l32] = m;
    ml->l[wave][l32] = lsum;
  }
  __syncthreads();
#pragma unroll
  for (int t0 = 0; t0 < kQT; t0 += NW * 4) ml->write_row(a, keys.ranges, it, t0 + (tid >> 4), 4 * (tid & 15));
}

// Up to 16 rows (a block of 16, a few tokens of shared heads, one token): the same
// on v_mfma_f32_16x16x32_bf16, so no MFMA row or softmax lane is spent on absent
// rows. S^T of 16 keys x 16 rows: A = K read from the tile (lane: key 16 kb + lane %
// 16, d 32 c + 8 hq .. +7, hq = lane / 16), B = Q^T; result lane (row lane % 16, hq)
// holds keys 16 kb + 4 hq + r. O^T (16 d x 16 rows) += V^T P^T over the 32 keys.
// Eight waves always: four took 8.4 us for 6.8 over 600 keys and 52.2 for 51.3 of a full
// launch (100-8192 keys). Few workgroups are bound by latency: over 3600 keys of one sequence
// lengths are there after 0.5 us, the first chunk is staged after 2.8, done after 3.4,
// merged and written after 4.6 of the kernel's 7.8 us. Many are bound by HBM: 32
// sequences of 100-8192 keys 48 us, 5.5 TB/s.
template <int NW, bool COLS>
__device__ __forceinline__ void paged16_item(const PagedArgs& a, const PagedItem<false, COLS>& it, char* smem) {
  constexpr int kRows = 16;
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform(tid >> 6);
  const int l16 = lane & 15;
  const int hq = lane >> 4;
  __bf16* ks = reinterpret_cast<__bf16*>(smem) + wave * 2 * kSub * kStride;
  __bf16* vs = ks + kSub * kStride;

  const PagedSeq& sq = it.sq;
  const ItemKeys<COLS> keys(a, it);
  if (!keys.any) return;
  const int row = it.r0 + l16 < it.r1 ? it.r0 + l16 : it.r1 - 1;
  const int tok = fast_div(row, a.group_div);
  const uint16_t* qp = a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(it.h * a.group + row - tok * a.group) * a.sq_h;
  bf16x8 qreg[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) qreg[c] = __builtin_bit_cast(bf16x8, ld16(qp + 32 * c + 8 * hq));
  const int ends = sq.key_end(a, tok);
  const int khi = COLS || ends < keys.hi ? ends : keys.hi;
  const int kfull = wave_uniform(sq.key_end(a, fast_div(it.r0, a.group_div)));  // every row sees these
  ChunkStream<NW, COLS> kv(a, it.b, it.h, it.list, keys.lo, keys.hi, keys.end, wave, lane);
  if (kv.mine > 0) kv.load(0);
  // Q is waited for here: in the loop the wait would be for the next chunk as well.
#pragma unroll
  for (int c = 0; c < 2; ++c) asm volatile("" ::"v"(qreg[c]));

  f32x4 o[4] = {};  // O^T [16-d block]: lane (row l16, hq) holds d 16 db + 4 hq + r
  float m = -INFINITY, lsum = 0.f;
  const int tr_row = l16 >> 2;
  const int tr_col = 4 * (lane & 3);
  for (int i = 0; i < kv.mine; ++i) {
    const ChunkInfo info = kv.info;
    kv.stage(ks, vs);
    if (i + 1 < kv.mine) kv.load(i + 1);
    f32x4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const __bf16* kt = &ks[(16 * kb + l16) * kStride + 8 * hq];
      s[kb] = mfma16(*reinterpret_cast<const bf16x8*>(kt), qreg[0], f32x4{});
      s[kb] = mfma16(*reinterpret_cast<const bf16x8*>(kt + 32), qreg[1], s[kb]);
    }
    if (kv.masked(info, kfull)) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[kb][r] = info.base[kb] + 4 * hq + r < khi && ((info.there >> kb) & 1) ? s[kb][r] : -INFINITY;
    }
    const float mx0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
    const float mx1 = fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]));
    float mt = fmaxf(mx0, mx1);
    mt = fmaxf(mt, shfl_xor(mt, 16));
    mt = max_xor32(mt) * a.scale_log2;
    if (__ballot(mt > m) != 0) {
      const float mn = fmaxf(m, mt);
      const float alpha = (mn == -INFINITY) ? 1.f : fast_exp2(m - mn);
      m = mn;
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) o[db] *= alpha;
    }
    const float mu = (m == -INFINITY) ? 0.f : m;
    float p[2][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[kb][r] = fast_exp2(fmaf(s[kb][r], a.scale_log2, -mu));
        lsum += p[kb][r];
      }
    const bf16x8 pop = to_bf16x8(p[0][0], p[0][1], p[0][2], p[0][3], p[1][0], p[1][1], p[1][2], p[1][3]);
    const int vrow = 4 * hq + tr_row;
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      const bf16x8 va = cat8(lds_read_tr(&vs[vrow * kStride + 16 * db + tr_col]),
                             lds_read_tr(&vs[(vrow + 16) * kStride + 16 * db + tr_col]));
      o[db] = mfma16(va, pop, o[db]);
    }
  }

  lsum += shfl_xor(lsum, 16);
  lsum = sum_xor32(lsum);
  __syncthreads();  // the tiles are reused below
  auto* ml = reinterpret_cast<MergeLds<NW, kRows>*>(smem);
#pragma unroll
  for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(&ml->o[wave][l16][16 * db + 4 * hq]) = o[db];
  if (hq == 0) {
    ml->m[wave][l16] = m;
    ml->l[wave][l16] = lsum;
  }
  __syncthreads();
  if (tid < 16 * kRows) ml->write_row(a, keys.ranges, it, tid >> 4, 4 * (tid & 15));
}

// Row tiles whose states are merged in one stage: both of 32 rows (1 sequence 7.9 -> 7.6 us, 4 of them 11.6 -> 11.2), one of 48
// rows (lists 28.1 us, all three at once 28.7).
template <int RT>
constexpr int codes_stage = RT == 2 ? 2 : 1;

// Rows of 8-bit pools: 16 RT rows, NW waves that share the chunks of a range. S^T of 16 keys x 16 rows on
// v_mfma_f32_16x16x32_bf16 from 16 codes of a key to a lane: the sums run over d in the order that
// gives (16 hq + 8 c + e), which Q's operand takes as well. A chunk's codes are converted once for all RT
// row tiles. Its scales enter with the softmax: K's with the factor, V's in the exponent, so that what is
// rounded to bf16 is P times it; the row sum takes its inverse again, once for 4 of the elements. (log2 scale - maximum
// is off by 2^-24 of the maximum, no more than the scores' own fp32 sums.) The running maximum is updated when it grew by more
// than kRescale: among 16 rows some maximum grows in most chunks (lists 28.1 -> 27.3 us, 12 sequences of 32 rows 15.4 -> 14.9).
// 16 rows: 4 waves where many items are bound by HBM (32 sequences of 100-8192 keys, 12 heads: 26 us, 4.4 TB/s of
// codes, of which 5.5 us until the first are there; 48 of 8192 keys 110, 5.6 TB/s), 8 for few, long ones. 32
// and 48 rows: a conversion serves 2 or 3 row tiles, at most two waves a SIMD at 64-key chunks (209 and 253 registers);
// lists of 40 pages of 32, 340 items: 27.3 us with 48 rows, 33 with 32. An item is 5 us until its first chunk is there (2.9 to
// find it and the end of its list), a chunk 2.9 us (48 products, ~650 VALU instructions, 805 where it is masked), the merge 2; on
// the 84 CUs that have two a chunk is 3.8, and these end last. Eight waves of 32-key chunks took 38 us, four 29. Codes stay bytes
// in LDS because a bf16 tile would be twice the writes and the room of half the waves (the first form, 32-key chunks staged in bf16: batch 50.6 -> 37 us).
template <int NW, int RT, int KC, int POOL, bool COLS>
__device__ __forceinline__ void paged_codes_item(const PagedArgs& a, const PagedItem<false, COLS>& it, char* smem) {
  using Stream = CodeStream<NW, KC, POOL, COLS>;
  constexpr int kG = KC / 16;
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform(tid >> 6);
  const int l16 = lane & 15;
  const int hq = lane >> 4;
  uint8_t* ks = reinterpret_cast<uint8_t*>(smem) + wave * 2 * Stream::kTile;
  uint8_t* vs = ks + Stream::kTile;

  const PagedSeq& sq = it.sq;
  const ItemKeys<COLS> keys(a, it);
  if (!keys.any) return;

  bf16x8 qreg[RT][2];
  int khi[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = it.r0 + 16 * t + l16 < it.r1 ? it.r0 + 16 * t + l16 : it.r1 - 1;
    const int tok = fast_div(row, a.group_div);
    const uint16_t* qp =
        a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(it.h * a.group + row - tok * a.group) * a.sq_h + 16 * hq;
#pragma unroll
    for (int c = 0; c < 2; ++c) qreg[t][c] = __builtin_bit_cast(bf16x8, ld16(qp + 8 * c));
    const int ends = sq.key_end(a, tok);
    khi[t] = COLS || ends < keys.hi ? ends : keys.hi;
  }
  Stream kv(a, it.b, it.h, it.list, keys.lo, keys.hi, keys.end, wave, lane);
  if (kv.mine > 0) kv.load(0);
  // Q is waited for here: in the loop the wait would be for the next chunk's codes as well.
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c) asm volatile("" ::"v"(qreg[t][c]));
  const int kfull = wave_uniform(sq.key_end(a, fast_div(it.r0, a.group_div)));  // every row sees these

  f32x4 o[RT][4] = {};  // O^T [16-d block]: lane (row l16, hq) holds d 16 db + 4 hq + r
  float m[RT], lsum[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = -INFINITY;
    lsum[t] = 0.f;
  }
  for (int i = 0; i < kv.mine; ++i) {
    const typename Stream::Info info = kv.info;
    kv.stage(ks, vs);
    if (i + 1 < kv.mine) kv.load(i + 1);
    bf16x8 kop[kG][2];
#pragma unroll
    for (int g = 0; g < kG; ++g) {
      const u32x4 w = kv.key_codes(ks, g);
      kop[g][0] = cat8(codes4<POOL>(w[0]), codes4<POOL>(w[1]));
      kop[g][1] = cat8(codes4<POOL>(w[2]), codes4<POOL>(w[3]));
    }
    const bool masked = kv.masked(info, kfull);
    float c2[kG];
#pragma unroll
    for (int g = 0; g < kG; ++g) c2[g] = a.scale_log2 * info.ks[g];
    bf16x8 pop[RT][kG / 2];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      f32x4 s[kG];
      float mt = -INFINITY;
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        s[g] = mfma16(kop[g][0], qreg[t][0], f32x4{});
        s[g] = mfma16(kop[g][1], qreg[t][1], s[g]);
      }
      if (masked) {
        asm volatile("");  // a branch: few chunks have any of it
#pragma unroll
        for (int g = 0; g < kG; ++g)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[g][r] = info.base[g] + 4 * hq + r < khi[t] && ((info.there >> g) & 1) ? s[g][r] : -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < kG; ++g) mt = fmaxf(mt, fmaxf(fmaxf(s[g][0], s[g][1]), fmaxf(s[g][2], s[g][3])) * c2[g]);
      mt = max_xor16_32(mt);
      if (__ballot(mt > m[t] + kRescale) != 0) {
        const float mn = fmaxf(m[t], mt);
        const float alpha = (mn == -INFINITY) ? 1.f : fast_exp2(m[t] - mn);
        m[t] = mn;
        lsum[t] *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db) o[t][db] *= alpha;
      }
      const float mu = (m[t] == -INFINITY) ? 0.f : m[t];
      f32x4 p[kG];
#pragma unroll
      for (int g = 0; g < kG; ++g) {
        const float to = info.v_log[g] - mu;
#pragma unroll
        for (int r = 0; r < 4; ++r) p[g][r] = fast_exp2(fmaf(s[g][r], c2[g], to));
        lsum[t] = fmaf((p[g][0] + p[g][1]) + (p[g][2] + p[g][3]), info.v_inv[g], lsum[t]);
      }
#pragma unroll
      for (int h2 = 0; h2 < kG / 2; ++h2)
        pop[t][h2] = to_bf16x8(p[2 * h2][0], p[2 * h2][1], p[2 * h2][2], p[2 * h2][3], p[2 * h2 + 1][0], p[2 * h2 + 1][1],
                               p[2 * h2 + 1][2], p[2 * h2 + 1][3]);
    }
#pragma unroll
    for (int h2 = 0; h2 < kG / 2; ++h2)
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const bf16x8 va = kv.value_codes(vs, h2, db);
#pragma unroll
        for (int t = 0; t < RT; ++t) o[t][db] = mfma16(va, pop[t][h2], o[t][db]);
      }
  }

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    lsum[t] += shfl_xor(lsum[t], 16);
    lsum[t] = sum_xor32(lsum[t]);
  }
  constexpr int kStage = codes_stage<RT>;
  auto* ml = reinterpret_cast<MergeLds<NW, 16 * kStage>*>(smem);
#pragma unroll
  for (int t0 = 0; t0 < RT; t0 += kStage) {
    __syncthreads();  // the tiles, or the last stage's states, are reused
#pragma unroll
    for (int t = t0; t < t0 + kStage; ++t) {
      const int r = 16 * (t - t0) + l16;
#pragma unroll
      for (int db = 0; db < 4; ++db) *reinterpret_cast<f32x4*>(&ml->o[wave][r][16 * db + 4 * hq]) = o[t][db];
      if (hq == 0) {
        ml->m[wave][r] = m[t];
        ml->l[wave][r] = lsum[t];
      }
    }
    __syncthreads();
#pragma unroll 1
    for (int r0 = 0; r0 < 16 * kStage; r0 += 4 * NW)
      if (r0 + (tid >> 4) < 16 * kStage) ml->write_row(a, keys.ranges, it, r0 + (tid >> 4), 4 * (tid & 15), 16 * t0);
  }
}

template <int NW, int RT, int KC>
constexpr size_t codes_smem() {
  constexpr size_t v = (size_t)NW * 2 * KC * kHeadDim;
  return v > sizeof(MergeLds<NW, 16 * codes_stage<RT>>) ? v : sizeof(MergeLds<NW, 16 * codes_stage<RT>>);
}

// WPS: waves per SIMD that the registers leave room for.
template <int NW, int RT, int KC, int WPS, int POOL, bool COLS>
__global__ __launch_bounds__(NW * 64, WPS) void paged_codes_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[codes_smem<NW, RT, KC>()];
  for (int id = wg_x();; id += a.workgroups) {  // as in paged_rows_kernel
    const PagedItem<false, COLS> it(a, id);
    if (!it.found) return;
    if (!COLS || it.r0 < it.r1) paged_codes_item<NW, RT, KC, POOL, COLS>(a, it, smem);
    if (id + a.workgroups >= it.total) return;
    __syncthreads();
  }
}

template <int NW, int ROWS, bool COLS>
__global__ __launch_bounds__(NW * 64, ROWS == 16 ? 4 : NW == 4 ? 3 : 2) void paged_rows_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[chunk_smem<NW, ROWS>()];
  // The launch has about as many workgroups as there are items; those left over
  // (lengths that the caller's total did not tell) are taken in turn.
  for (int id = wg_x();; id += a.workgroups) {
    const PagedItem<false, COLS> it(a, id);
    if (!it.found) return;
    if (!COLS || it.r0 < it.r1) {
      if constexpr (ROWS == 16)
        paged16_item<NW, COLS>(a, it, smem);
      else
        paged32_item<NW, COLS>(a, it, smem);
    }
    if (id + a.workgroups >= it.total) return;
    __syncthreads();
  }
}

// 128-row tiles: four waves of 32 rows that share each 64-key K / V tile, which goes
// from the page to LDS directly (bd3_swz.h; two stages: the next tile loads during
// the current one). A wave loads 16 keys of a tile, which lie in one page, so its
// source is one scalar base and the same lane offsets for every full tile. SUBS sets
// of four waves take the tiles in turn, each through a ring of its own, and add up at
// the end: few, long items.
// S^T (keys x rows) = K Q^T, O^T += V^T P^T with P^T taken from the S^T registers;
// a wave skips tiles past its last row's keys and masks only those that its
// first row does not see whole. The running maximum is updated when it grew by
// more than kRescale (log2): a stale one leaves O / l exact and bounds P by 2^8.
// Full launches are bound by the softmax's VALU work beside the products (8 prompts
// of 2048 tokens, 12 heads: 74 us), short ones by a tile's own
// chain, ~1 us for a workgroup alone on its CU: three and four stages only cost
// occupancy (84 -> 95-107 us for prompts of 1507-4034 tokens, 28.5 -> 31-37 for 96 rows
// over 727-3871 keys).
// 8-bit pools: each wave loads the codes of its 16 keys to LDS during the step on the tile before,
// then converts them to bf16 into the other stage, once for the four waves; the tile's four scales
// enter as in paged_codes_item. (Held in registers during the step the codes spilled 4 to 40 of
// those: prompts of 1500-4096 tokens in int8 106 us.) The codes are there when a step ends (8 clocks of waiting); prompts of
// 1500-4096 tokens, 12 heads 74 us, 565 TFLOP/s, bound by VALU work: exponentials, and ~50 instructions of
// conversion a wave and tile. 24 sequences of 500-4000 keys, 32 tokens, 12 heads on 4: 23 us, 284 items of 3.5 us start-up
// and 3-6 steps of two tiles, 2.0 us each where the workgroup has its CU alone: most are done after 13 us, those of 5 and 6 steps
// on the 28 CUs that have two (up to 3.4 us a step) after 17-21.
template <int SUBS, int POOL>
__global__ __launch_bounds__(256 * SUBS, 4) void paged128_kernel(PagedArgs a) {
  constexpr bool kCodes = POOL != kPoolBf16;
  __shared__ __attribute__((aligned(1024))) __bf16 smem_all[SUBS][2][2][kSwTile];  // [set][stage][K | V]
  __shared__ __attribute__((aligned(1024))) uint8_t raw_all[kCodes ? SUBS : 1][kCodes ? 8 : 1][1024];  // [set][2 wave + K | V]
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform((tid >> 6) & 3);  // in its set
  const int sub = SUBS == 1 ? 0 : wave_uniform(tid >> 8);
  auto& smem = smem_all[sub];
  const int l32 = lane & 31;
  const int g = lane >> 5;

  // One item a workgroup; the launch has the most there can be, those without one at its end.
  int b, h, qt, split = 0;
  PagedSeq sq;
  if (a.sorted) {
    const int j = wave_uniform(fast_div(wg_x(), a.kv_heads_div));
    h = wg_x() - j * a.kv_heads;
    const TileItem it(a, j);
    if (!it.found) return;
    b = it.b;
    sq = it.sq;
    qt = (sq.rows + 127) / 128 - 1 - it.rank;
  } else {
    const PagedItem<true, false> it(a, wg_x());
    if (!it.found) return;
    b = it.b;
    h = it.h;
    sq = it.sq;
    qt = it.r0 / 128;
    split = it.split;
  }
  const int r0 = 128 * qt;
  const int key_end = sq.tile_end(a, r0);
  const KeySplit<true> cut(a, sq.kv);
  const int ranges = wave_uniform(cut.ranges(key_end));
  if (split >= ranges) return;
  const int lo = wave_uniform(split * cut.len);
  const int hi = split + 1 < ranges ? wave_uniform(lo + cut.len) : key_end;
  const int n_tiles = (hi - lo + kSwRows - 1) / kSwRows;  // 0: a tile that sees no key
  const int n_mine = n_tiles > sub ? (n_tiles - sub + SUBS - 1) / SUBS : 0;

  // Page entries of the set's next 16 tiles: lane 4 i + w holds that of wave w's keys
  // of the (base + i)-th one.
  const int32_t* table = a.table + (int64_t)b * a.table_s;
  auto entries = [&](int base) {
    const int key = lo + (sub + SUBS * (base + (lane >> 2))) * kSwRows + 16 * (lane & 3);
    return key < hi ? table[key >> a.page_shift] : -1;
  };
  int ids = entries(0), ids_next = -1;
  float k_scale = 1.f, v_log = 0.f, v_inv = 1.f;  // 8-bit pools: of the same tiles' 16-key groups, K's with the softmax's factor
  auto find_scales = [&](int base) {
    const int key = lo + (sub + SUBS * (base + (lane >> 2))) * kSwRows + 16 * (lane & 3);
    k_scale = 1.f;
    float v_scale = 1.f;
    if ((unsigned)ids < (unsigned)a.pages) {
      const int64_t at = ((int64_t)ids * a.kv_heads + h) * (a.page >> 4) + ((key & (a.page - 1)) >> 4);
      k_scale = a.k_scales[at] * a.scale_log2;
      v_scale = a.v_scales[at];
    }
    v_log = fast_log2(v_scale);
    v_inv = __builtin_amdgcn_rcpf(v_scale);
  };

  const int qrow0 = r0 + 32 * wave;
  const int myr = qrow0 + l32;
  const int row = myr < sq.rows ? myr : sq.rows - 1;
  const int tok = fast_div(row, a.group_div);
  const int64_t head = h * a.group + row - tok * a.group;
  const uint16_t* qp = a.q + (int64_t)(sq.q0 + tok) * a.sq_t + head * a.sq_h;
  bf16x8 qreg[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) qreg[c] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * c + 8 * g));

  uint64_t ok = __ballot((unsigned)ids < (unsigned)a.pages);

  uint32_t koff[2], voff[2];
  int lrow[2], lch[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    lrow[j] = 8 * j + (lane >> 3);
    lch[j] = 8 * ((lane & 7) ^ swz(16 * wave + lrow[j]));
    koff[j] = (uint32_t)(2 * (lrow[j] * (int)a.sk_s + lch[j]));
    voff[j] = (uint32_t)(2 * (lrow[j] * (int)a.sv_s + lch[j]));
  }
  const uint32_t lds_w = lds_addr(&smem[0][0][0]) + (uint32_t)wave * 2048u;
  const uint16_t* kh = static_cast<const uint16_t*>(a.k) + h * a.sk_h;
  const uint16_t* vh = static_cast<const uint16_t*>(a.v) + h * a.sv_h;
  uint32_t there = 0;  // quarters of the tile requested last whose page exists
  float ks_next[4], v_log_next[4], v_inv_next[4];  // and their scales
  const uint32_t raw_w = lds_addr(&raw_all[kCodes ? sub : 0][kCodes ? 2 * wave : 0][0]);
  const uint8_t* raw = &raw_all[kCodes ? sub : 0][kCodes ? 2 * wave : 0][16 * lane];
  auto read_scales = [&](int i) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      ks_next[q] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(k_scale), 4 * (i & 15) + q));
      v_log_next[q] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_log), 4 * (i & 15) + q));
      v_inv_next[q] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v_inv), 4 * (i & 15) + q));
    }
  };
  auto issue = [&](int i) {  // the set's i-th tile
    if ((i & 15) == 0 && i > 0) {
      ids = ids_next;
      ok = __ballot((unsigned)ids < (unsigned)a.pages);
      if constexpr (kCodes) find_scales(i);
    }
    if ((i & 15) == 8) ids_next = entries((i | 15) + 1);
    const int at = 4 * (i & 15) + wave;
    const int key = lo + (sub + SUBS * i) * kSwRows + 16 * wave;
    there = (uint32_t)(ok >> (4 * (i & 15))) & 15u;
    const uint32_t dst = lds_w + (uint32_t)(i & 1) * 16384u;
    const int lim = (ok >> at) & 1 ? sq.kv - 1 - key : -1;  // the last of its 16 rows that is a key
    const int64_t page = __builtin_amdgcn_readlane(ids, at);
    const int64_t slot = key & (a.page - 1);
    if constexpr (kCodes) {
      if (i > 0) read_scales(i);
      const int top = lim < 0 ? 0 : lim;  // rows past the last key re-read it
      const int r = (lane >> 2) < top ? lane >> 2 : top;
      const uint8_t* none = reinterpret_cast<const uint8_t*>(zero_row);
      const uint8_t* kb = lim >= 0 ? static_cast<const uint8_t*>(a.k) + h * a.sk_h + page * a.sk_p + slot * a.sk_s : none;
      const uint8_t* vb = lim >= 0 ? static_cast<const uint8_t*>(a.v) + h * a.sv_h + page * a.sv_p + slot * a.sv_s : none;
      dma16(kb, (uint32_t)(r * (int)a.sk_s + 16 * (lane & 3)), raw_w);
      dma16(vb, (uint32_t)(r * (int)a.sv_s + 16 * (lane & 3)), raw_w + 1024u);
      return;
    }
    const void* kb = lim >= 0 ? kh + page * a.sk_p + slot * a.sk_s : zero_row;
    const void* vb = lim >= 0 ? vh + page * a.sv_p + slot * a.sv_s : zero_row;
    if (lim >= 15) {
#pragma unroll
      for (int j = 0; j < 2; ++j) dma16(kb, koff[j], dst + 1024u * j);
#pragma unroll
      for (int j = 0; j < 2; ++j) dma16(vb, voff[j], dst + 8192u + 1024u * j);
    } else {  // rows past the last key re-read it
      const int top = lim < 0 ? 0 : lim;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = lrow[j] < top ? lrow[j] : top;
        dma16(kb, (uint32_t)(2 * (r * (int)a.sk_s + lch[j])), dst + 1024u * j);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = lrow[j] < top ? lrow[j] : top;
        dma16(vb, (uint32_t)(2 * (r * (int)a.sv_s + lch[j])), dst + 8192u + 1024u * j);
      }
    }
  };
  auto convert = [&](int i) {  // codes of the set's i-th tile to its stage
    const int r = 16 * wave + (lane >> 2), p = 2 * (lane & 3);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's codes are there
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(raw + 1024 * kv);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        *reinterpret_cast<bf16x8*>(&smem[i & 1][kv][64 * r + 8 * ((p + c) ^ swz(r))]) =
            cat8(codes4<POOL>(x[2 * c]), codes4<POOL>(x[2 * c + 1]));
    }
  };
  if (n_mine > 0) issue(0);
  if constexpr (kCodes) {  // the first tile's scales after its codes: asked for before them they were waited for first
    find_scales(0);
    read_scales(0);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) asm volatile("" ::"v"(qreg[c]));  // waits for Q here, not in the loop
  if constexpr (kCodes)
    if (n_mine > 0) convert(0);

  const int khi = sq.key_end(a, tok);  // the lane's row sees [0, khi)
  const int wave_last = qrow0 + 31 < sq.rows ? qrow0 + 31 : sq.rows - 1;
  const int emax = qrow0 < sq.rows ? wave_uniform(sq.key_end(a, fast_div(wave_last, a.group_div))) : 0;
  const int emin = qrow0 < sq.rows ? wave_uniform(sq.key_end(a, fast_div(qrow0, a.group_div))) : 0;

  f32x16 o[2] = {};  // O^T [d block]
  float mref = 0.f, lsum = 0.f;
  bool valid = false;  // the row has met a key
  const float c2 = a.scale_log2;
  float k_factor[4], v_to[4], v_back[4];  // 8-bit pools: the tile's
  auto step = [&](int k0, uint32_t seen, const __bf16* ks, const __bf16* vs) {
    f32x16 s[2];
#pragma unroll
    for (int sb = 0; sb < 2; ++sb) s[sb] = mfma32(sw_row_op(ks, 32 * sb, 0, lane), qreg[0], f32x16{});
#pragma unroll
    for (int c = 1; c < 4; ++c)
#pragma unroll
      for (int sb = 0; sb < 2; ++sb) s[sb] = mfma32(sw_row_op(ks, 32 * sb, c, lane), qreg[c], s[sb]);
    if (k0 + kSwRows > emin || seen != 15u) {
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * sb + 8 * (r >> 2) + 4 * g + (r & 3);
          s[sb][r] = key < khi && ((seen >> (2 * sb + (r >> 3))) & 1) ? s[sb][r] : -INFINITY;
        }
    }
    float mt;
    if constexpr (kCodes) {
      float mrow[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int r = 0; r < 16; r += 2)
          mrow[2 * sb + (r >> 3)] = fmaxf(fmaxf(mrow[2 * sb + (r >> 3)], s[sb][r]), s[sb][r + 1]);
      mt = max_xor32(fmaxf(fmaxf(mrow[0] * k_factor[0], mrow[1] * k_factor[1]),
                           fmaxf(mrow[2] * k_factor[2], mrow[3] * k_factor[3]))) - mref;
    } else {
      float mrow = -INFINITY;
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) mrow = fmaxf(fmaxf(mrow, s[sb][r]), s[sb][r + 1]);
      mt = fmaf(max_xor32(mrow), c2, -mref);
    }
    if (__ballot(!valid || mt > kRescale) != 0) {
      const float delta = valid ? fmaxf(mt, 0.f) : (mt == -INFINITY ? 0.f : mt);
      const float alpha = valid ? fast_exp2(-delta) : 1.f;
      valid = valid || mt != -INFINITY;
      mref += delta;
      lsum *= alpha;
      o[0] *= alpha;
      o[1] *= alpha;
    }
#pragma unroll
    for (int sb = 0; sb < 2; ++sb) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r)
        p[r] = kCodes ? fast_exp2(fmaf(s[sb][r], k_factor[2 * sb + (r >> 3)], v_to[2 * sb + (r >> 3)] - mref))
                      : fast_exp2(fmaf(s[sb][r], c2, -mref));
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const bf16x8 pop = to_bf16x8(p[8 * kc], p[8 * kc + 1], p[8 * kc + 2], p[8 * kc + 3], p[8 * kc + 4],
                                     p[8 * kc + 5], p[8 * kc + 6], p[8 * kc + 7]);
        const float sum = ((p[8 * kc] + p[8 * kc + 1]) + (p[8 * kc + 2] + p[8 * kc + 3])) +
                          ((p[8 * kc + 4] + p[8 * kc + 5]) + (p[8 * kc + 6] + p[8 * kc + 7]));
        lsum = kCodes ? fmaf(sum, v_back[2 * sb + kc], lsum) : lsum + sum;
#pragma unroll
        for (int db = 0; db < 2; ++db) o[db] = mfma32(sw_tr_op(vs, 32 * sb + 16 * kc, 32 * db, lane), pop, o[db]);
      }
    }
  };

  uint32_t seen = there;
  auto take_factors = [&] {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      k_factor[q] = ks_next[q];
      v_to[q] = v_log_next[q];
      v_back[q] = v_inv_next[q];
    }
  };
  if constexpr (kCodes) {
    take_factors();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  vm_wait_barrier<0>();
  const int steps = (n_tiles + SUBS - 1) / SUBS;  // of the set with the most tiles
  for (int i = 0; i < steps; ++i) {
    if (i + 1 < n_mine) issue(i + 1);
    const int k0 = lo + (sub + SUBS * i) * kSwRows;
    if (i < n_mine && k0 < emax) step(k0, seen, smem[i & 1][0], smem[i & 1][1]);
    seen = there;
    if constexpr (kCodes) {
      if (i + 1 < n_mine) convert(i + 1);
      take_factors();
    }
    // The next tile is there, and this wave's reads of this one are done before
    // any wave requests the tile after it into the same stage.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    vm_wait_barrier<0>();
  }

  float ltot = sum_xor32(lsum);
  if constexpr (SUBS > 1) {
    // The other sets hand their state to set 0 through LDS (every wave is past its
    // last read of the rings); a set that met no key of a row has l = 0.
    constexpr int kWave = 34 * 64, kSet = 4 * kWave;
    static_assert((SUBS - 1) * kSet * 4 <= (int)sizeof(smem_all), "hand-over fits the rings");
    float* ex = reinterpret_cast<float*>(&smem_all[0][0][0][0]) + wave * kWave + lane;
    if (sub > 0) {
      float* my = ex + (sub - 1) * kSet;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        my[r * 64] = o[0][r];
        my[(16 + r) * 64] = o[1][r];
      }
      my[32 * 64] = mref;
      my[33 * 64] = ltot;
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int t = 0; t < SUBS - 1; ++t, ex += kSet) {
      const float m1 = ex[32 * 64], l1 = ex[33 * 64];
      const float m = l1 > 0.f ? (ltot > 0.f ? fmaxf(mref, m1) : m1) : mref;
      const float w0 = ltot > 0.f ? fast_exp2(mref - m) : 0.f, w1 = l1 > 0.f ? fast_exp2(m1 - m) : 0.f;
      mref = m;
      ltot = ltot * w0 + l1 * w1;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        o[0][r] = o[0][r] * w0 + ex[r * 64] * w1;
        o[1][r] = o[1][r] * w0 + ex[(16 + r) * 64] * w1;
      }
    }
  }
  if (myr >= sq.rows) return;
  const bool any = ltot > 0.f;
  const float inv = any ? 1.f / ltot : 0.f;
  if (ranges == 1) {
    uint16_t* op = a.o + (int64_t)(sq.q0 + tok) * a.so_t + head * a.so_h;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<bf16x4*>(op + 32 * db + 8 * q4 + 4 * g) =
            to_bf16x4(o[db][4 * q4] * inv, o[db][4 * q4 + 1] * inv, o[db][4 * q4 + 2] * inv, o[db][4 * q4 + 3] * inv);
  } else {
    const int at = sq.part_row(a, h, split, myr);
    float* po = a.part_o + at * kHeadDim;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4*>(po + 32 * db + 8 * q4 + 4 * g) =
            f32x4{o[db][4 * q4] * inv, o[db][4 * q4 + 1] * inv, o[db][4 * q4 + 2] * inv, o[db][4 * q4 + 3] * inv};
    if (g == 0) a.part_lse[at] = any ? mref + fast_log2(ltot) : -INFINITY;
  }
}

// Merges the ranges of the tiles that were cut: weights exp2(lse_s - max lse), 16
// threads a row, 4 outputs each; the loads of 8 ranges are issued before their
// first use. Grid: (KV head, 16 packed rows), the head fastest as in the first launch,
// which leaves more of the partials in the L2 that reads them (5 sequences of 247-6958
// keys, 8 heads, 16 rows: 13.8 us with the rows fastest, 13.4 so; 13.9 with 32 rows to a
// workgroup).
__global__ __launch_bounds__(16 * kMergeRows) void paged_combine_kernel(PagedArgs a) {
  const int slot = fast_div(wg_x(), a.kv_heads_div);
  const int h = wg_x() - slot * a.kv_heads;
  const int at = slot * kMergeRows + (wi_x() >> 4);
  const int lane = wi_x() & 63;
  const int tok = fast_div(at, a.group_div);
  // The share that holds the row's token, from the lane that has it: a lane a
  // sequence, four rows to a wave, mostly of one sequence. Every lane stays in the
  // loop, it holds a share.
  const int t0 = __builtin_amdgcn_readlane(tok, 0), t3 = __builtin_amdgcn_readlane(tok, 48);
  PagedSeq sq = {};
  for (int s0 = 0; s0 < a.seqs; s0 += 64) {
    PagedSeq mine = {};
    if (s0 + lane < a.seqs) mine = PagedSeq(a, s0 + lane);
    const uint64_t all = __ballot(mine.q0 <= t0 && t3 - mine.q0 < mine.n);
    if (all != 0) {
      sq = mine.of_lane(__builtin_ctzll(all));
      break;
    }
    int from = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = __builtin_amdgcn_readlane(tok, 16 * k);
      const uint64_t has = __ballot(mine.q0 <= t && t - mine.q0 < mine.n);
      if ((lane >> 4) == k && has != 0) from = __builtin_ctzll(has);
    }
    const int q0 = __builtin_amdgcn_ds_bpermute(4 * from, mine.q0), n = __builtin_amdgcn_ds_bpermute(4 * from, mine.n);
    const int kv = __builtin_amdgcn_ds_bpermute(4 * from, mine.kv), rows = __builtin_amdgcn_ds_bpermute(4 * from, mine.rows);
    if (from >= 0 && sq.n == 0) {
      sq.q0 = q0;
      sq.n = n;
      sq.kv = kv;
      sq.rows = rows;
    }
  }
  const int row = at - sq.q0 * a.group;
  if (row >= sq.rows) return;  // of no sequence, or past the caller's bound
  const int r0 = fast_div(row, a.tile_div) * a.tile;
  const int keys = a.columns != nullptr
                       ? sq.listed_keys(a)
                       : sq.key_end(a, fast_div((r0 + a.tile < sq.rows ? r0 + a.tile : sq.rows) - 1, a.group_div));
  const int ranges = a.tile == 128 ? KeySplit<true>(a, sq.kv).ranges(keys) : KeySplit<false>(a, sq.kv).ranges(keys);
  if (ranges <= 1) return;
  const int d0 = 4 * (wi_x() & 15);
  const int part0 = (h * a.part_rows + at) * a.n_splits;
  const float* lp = a.part_lse + part0;
  const float* pp = a.part_o + part0 * kHeadDim + d0;
  constexpr int kG = 8;
  float mm = -INFINITY, wt = 0.f;
  f32x4 acc = {};
  for (int s0 = 0; s0 < ranges; s0 += kG) {
    float l[kG];
    f32x4 po[kG];
#pragma unroll
    for (int k = 0; k < kG; ++k) {
      l[k] = s0 + k < ranges ? lp[s0 + k] : -INFINITY;
      po[k] = s0 + k < ranges ? *reinterpret_cast<const f32x4*>(pp + (s0 + k) * kHeadDim) : f32x4{};
    }
    float mg = mm;
#pragma unroll
    for (int k = 0; k < kG; ++k) mg = fmaxf(mg, l[k]);
    const float base = mg == -INFINITY ? 0.f : mg;
    const float old = fast_exp2(mm - base);  // 0 while no key was met
    wt *= old;
    acc *= old;
    mm = mg;
#pragma unroll
    for (int k = 0; k < kG; ++k) {
      const float w = fast_exp2(l[k] - base);
      wt += w;
      acc += w * po[k];
    }
  }
  const float inv = wt > 0.f ? 1.f / wt : 0.f;
  *reinterpret_cast<bf16x4*>(a.o + (int64_t)tok * a.so_t + (int64_t)(h * a.group + at - tok * a.group) * a.so_h + d0) =
      to_bf16x4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

template <int POOL, bool COLS>
hipError_t launch_paged_tiles(const PagedArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.workgroups);
  if (a.tile == 128) {
    if constexpr (!COLS) {
      if (a.subs == 4)
        hipLaunchKernelGGL((paged128_kernel<4, POOL>), grid, dim3(1024), 0, stream, a);
      else if (a.subs == 2)
        hipLaunchKernelGGL((paged128_kernel<2, POOL>), grid, dim3(512), 0, stream, a);
      else if (a.subs == 1)
        hipLaunchKernelGGL((paged128_kernel<1, POOL>), grid, dim3(256), 0, stream, a);
    } else {
      return hipErrorInvalidValue;
    }
  } else if constexpr (POOL != kPoolBf16) {
    if (a.tile == 16 && a.subs == 2)
      hipLaunchKernelGGL((paged_codes_kernel<8, 1, 32, 4, POOL, COLS>), grid, dim3(512), 0, stream, a);
    else if (a.tile == 16)
      hipLaunchKernelGGL((paged_codes_kernel<4, 1, 32, 3, POOL, COLS>), grid, dim3(256), 0, stream, a);
    else if (a.tile == 32 && a.subs == 2)
      hipLaunchKernelGGL((paged_codes_kernel<8, 2, 32, 3, POOL, COLS>), grid, dim3(512), 0, stream, a);
    else if (a.tile == 32)
      hipLaunchKernelGGL((paged_codes_kernel<4, 2, 64, 2, POOL, COLS>), grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL((paged_codes_kernel<4, 3, 64, 2, POOL, COLS>), grid, dim3(256), 0, stream, a);
  } else {
    if (a.tile == 16)
      hipLaunchKernelGGL((paged_rows_kernel<8, 16, COLS>), grid, dim3(512), 0, stream, a);
    else if (a.subs == 2)
      hipLaunchKernelGGL((paged_rows_kernel<8, 32, COLS>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((paged_rows_kernel<4, 32, COLS>), grid, dim3(256), 0, stream, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_splits == 1) return e;
  hipLaunchKernelGGL(paged_combine_kernel, dim3((unsigned)(a.kv_heads * a.part_slots)), dim3(16 * kMergeRows), 0, stream, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace bd3
