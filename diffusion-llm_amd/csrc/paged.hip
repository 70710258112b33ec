// paged.hip - attention of ragged batches over a paged KV cache, and the
// attention inputs written into its pages.
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
// Pages cost 11% against a contiguous cache in full launches: 32 sequences x 12 heads,
// 16 rows over 4112 keys, 70 us at 16- to 256-key pages (5.8 TB/s) against 63; short
// ones pay two dependent reads (lengths, table entries) before the first key.
#include "bd3_device.h"
#include "bd3_launch.h"
#include "bd3_swz.h"

namespace bd3 {
namespace {

constexpr int kQT = 32;       // rows of the 32-row tile
constexpr int kSub = 32;      // keys per wave step
constexpr int kStride = 72;   // padded LDS row (bf16)
constexpr int kMergeRow = kHeadDim + 4;

__device__ __attribute__((aligned(128))) uint16_t zero_row[kHeadDim];

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

// The 32-key chunks of one key range that one of NW waves takes in turn (chunks
// wave, wave + NW, ...): from the pages to registers, the next chunk's loads in
// flight while the last one, staged in the wave's LDS tiles, is computed.
template <int NW>
struct ChunkStream {
  const PagedArgs& a;
  const int32_t* table;
  const uint16_t *kh, *vh;  // the head's rows of page 0
  int lo, hi, wave, lane, mine;
  int ids;        // lane 2 i + half: page of the half's 16 keys (a page holds at least 16) of chunk base + i
  uint64_t ok;    // which of them exist
  u32x4 kr[4], vr[4];  // lane + 64 j -> key row 8 j + lane / 8 of the chunk, 16-byte part lane % 8
  uint32_t there;      // halves of the loaded chunk whose page exists

  __device__ __forceinline__ ChunkStream(const PagedArgs& a_, int b, int h, int lo_, int hi_, int wave_, int lane_)
      : a(a_), lo(lo_), hi(hi_), wave(wave_), lane(lane_), there(0) {
    table = a.table + (int64_t)b * a.table_s;
    kh = a.k + h * a.sk_h;
    vh = a.v + h * a.sv_h;
    const int n = hi > lo ? (hi - lo + kSub - 1) / kSub : 0;
    mine = n > wave ? (n - wave + NW - 1) / NW : 0;
  }
  __device__ __forceinline__ int first_key(int i) const { return lo + (wave + NW * i) * kSub; }
  __device__ __forceinline__ void load(int i) {
    if ((i & 31) == 0) {
      const int key = first_key(i + (lane >> 1)) + 16 * (lane & 1);
      ids = key < hi ? table[key >> a.page_shift] : -1;
      ok = __ballot((unsigned)ids < (unsigned)a.pages);
    }
    there = (uint32_t)(ok >> (2 * (i & 31))) & 3u;
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int at = 2 * (i & 31) + hh;
      const int key = first_key(i) + 16 * hh;
      const bool is = (there >> hh) & 1;
      const int64_t page = __builtin_amdgcn_readlane(ids, at);
      const int64_t slot = key & (a.page - 1);
      const uint64_t kb = (uint64_t)(uintptr_t)(is ? kh + page * a.sk_p + slot * a.sk_s : zero_row);
      const uint64_t vb = (uint64_t)(uintptr_t)(is ? vh + page * a.sv_p + slot * a.sv_s : zero_row);
      const int last = is ? hi - 1 - key : 0;  // rows past the range's end re-read its last one
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = (lane >> 3) + 8 * j < last ? (lane >> 3) + 8 * j : last;
        kr[2 * hh + j] = __builtin_nontemporal_load(
            (global_u32x4*)(kb + (uint32_t)(2 * (r * (int)a.sk_s + 8 * (lane & 7)))));
        vr[2 * hh + j] = __builtin_nontemporal_load(
            (global_u32x4*)(vb + (uint32_t)(2 * (r * (int)a.sv_s + 8 * (lane & 7)))));
      }
    }
  }
  __device__ __forceinline__ void stage(__bf16* ks, __bf16* vs) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int off = ((lane >> 3) + 8 * j) * kStride + 8 * (lane & 7);
      *reinterpret_cast<u32x4*>(&ks[off]) = kr[j];
      *reinterpret_cast<u32x4*>(&vs[off]) = vr[j];
    }
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

// Item `id` of the list: KV head (fastest), row tile, range, in the order of the
// sequences. Every sequence has items of its own number, so the list
// is made here from the lengths, a lane a sequence: a launch of the most items that
// the bounds allow spent about 1 ns on each empty workgroup (32 sequences of
// 100-8192 keys, 12 heads: 67 us at the best range length, 55 with the list).
template <bool EVEN>
struct PagedItem {
  int b, h, qt, split;
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
        tiles = (mine.rows + a.tile - 1) / a.tile;
        items = tiles * KeySplit<EVEN>(a, mine.kv).ranges(mine.kv);
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
        qt = rem;
        found = true;
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
  __device__ __forceinline__ void write_row(const PagedArgs& a, int ranges, const PagedItem<false>& it, int rt,
                                            int d) const {
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
    const int row = it.qt * ROWS + rt;
    if (ranges == 1) {
      if (row < it.sq.rows) {
        const int t = fast_div(row, a.group_div);
        *reinterpret_cast<bf16x4*>(a.o + (int64_t)(it.sq.q0 + t) * a.so_t +
                                   (int64_t)(it.h * a.group + row - t * a.group) * a.so_h + d) =
            to_bf16x4(ot[0] * inv, ot[1] * inv, ot[2] * inv, ot[3] * inv);
      }
    } else {
      if (row >= it.sq.rows) return;
      const int at = it.sq.part_row(a, it.h, it.split, row);
      *reinterpret_cast<f32x4*>(&a.part_o[at * kHeadDim + d]) = ot * inv;
      if (d == 0) a.part_lse[at] = lt > 0.f ? mm + fast_log2(lt) : -INFINITY;
    }
  }
};
template <int NW, int ROWS>
constexpr size_t chunk_smem() {
  constexpr size_t v = sizeof(__bf16) * NW * 2 * kSub * kStride;
  return v > sizeof(MergeLds<NW, ROWS>) ? v : sizeof(MergeLds<NW, ROWS>);
}

// 32-row tiles: NW waves share the key chunks of a range. S^T (32 keys x 32 rows) =
// K Q^T on v_mfma_f32_32x32x16_bf16 with the K tile's rows as A operands; O^T += V^T
// P^T with V read transposed. Eight waves for few items (one workgroup a CU at 160
// registers), four for many (three a CU), each at its best ranges: 32 rows over 500-2000
// keys of 8 sequences 13.9 us against 15.1; over 4032 keys of 48 sequences 111, 104.
// At four waves per SIMD it spills (43 -> 50 us). Full launches are bound by HBM (32
// sequences x 4128 keys 73 us, 5.6 TB/s; contiguous 65).
template <int NW>
__device__ __forceinline__ void paged32_item(const PagedArgs& a, const PagedItem<false>& it, char* smem) {
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform(tid >> 6);
  const int l32 = lane & 31;
  const int g = lane >> 5;
  __bf16* ks = reinterpret_cast<__bf16*>(smem) + wave * 2 * kSub * kStride;
  __bf16* vs = ks + kSub * kStride;

  const PagedSeq& sq = it.sq;
  const int r0 = it.qt * kQT;
  const int key_end = sq.tile_end(a, r0);
  const KeySplit<false> cut(a, sq.kv);
  const int ranges = cut.ranges(key_end);
  if (it.split >= ranges) return;
  const int lo = it.split << cut.shift;
  const int hi = it.split + 1 < ranges ? lo + cut.len : key_end;
  ChunkStream<NW> kv(a, it.b, it.h, lo, hi, wave, lane);
  if (kv.mine > 0) kv.load(0);

  // Q^T B operand: lane holds row r0 + l32 (clamped), d = 16c + 8g .. +7.
  const int row = r0 + l32 < sq.rows ? r0 + l32 : sq.rows - 1;
  const int tok = fast_div(row, a.group_div);
  const uint16_t* qp = a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(it.h * a.group + row - tok * a.group) * a.sq_h;
  bf16x8 qreg[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) qreg[c] = __builtin_bit_cast(bf16x8, ld16(qp + 16 * c + 8 * g));
  const int ends = sq.key_end(a, tok);
  const int khi = ends < hi ? ends : hi;
  const int kfull = wave_uniform(sq.key_end(a, fast_div(r0, a.group_div)));  // every row of the tile sees these

  f32x16 oacc[2] = {};
  float m = -INFINITY, lsum = 0.f;
  const int tr_row = (lane & 15) >> 2;
  const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  for (int i = 0; i < kv.mine; ++i) {
    const int c0 = kv.first_key(i);
    const uint32_t there = kv.there;
    kv.stage(ks, vs);
    if (i + 1 < kv.mine) kv.load(i + 1);
    // A = K rows from the tile (lane: key l32, d 16c + 8g .. +7).
    f32x16 s = {};
#pragma unroll
    for (int c = 0; c < 4; ++c)
      s = mfma32(*reinterpret_cast<const bf16x8*>(&ks[l32 * kStride + 16 * c + 8 * g]), qreg[c], s);
    if (c0 + kSub > kfull || c0 + kSub > hi || there != 3) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int key = c0 + 8 * (r >> 2) + 4 * g + (r & 3);
        s[r] = key < khi && ((there >> (r >> 3)) & 1) ? s[r] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = max_xor32(mx);
    const float mt = mx * a.scale_log2;
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
  for (int t0 = 0; t0 < kQT; t0 += NW * 4) ml->write_row(a, ranges, it, t0 + (tid >> 4), 4 * (tid & 15));
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
template <int NW>
__device__ __forceinline__ void paged16_item(const PagedArgs& a, const PagedItem<false>& it, char* smem) {
  constexpr int kRows = 16;
  const int tid = wi_x();
  const int lane = tid & 63;
  const int wave = wave_uniform(tid >> 6);
  const int l16 = lane & 15;
  const int hq = lane >> 4;
  __bf16* ks = reinterpret_cast<__bf16*>(smem) + wave * 2 * kSub * kStride;
  __bf16* vs = ks + kSub * kStride;

  const PagedSeq& sq = it.sq;
  const int key_end = sq.tile_end(a, 0);
  const KeySplit<false> cut(a, sq.kv);
  const int ranges = cut.ranges(key_end);
  if (it.split >= ranges) return;
  const int lo = it.split << cut.shift;
  const int hi = it.split + 1 < ranges ? lo + cut.len : key_end;
  ChunkStream<NW> kv(a, it.b, it.h, lo, hi, wave, lane);
  if (kv.mine > 0) kv.load(0);

  const int row = l16 < sq.rows ? l16 : sq.rows - 1;
  const int tok = fast_div(row, a.group_div);
  const uint16_t* qp = a.q + (int64_t)(sq.q0 + tok) * a.sq_t + (int64_t)(it.h * a.group + row - tok * a.group) * a.sq_h;
  bf16x8 qreg[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) qreg[c] = __builtin_bit_cast(bf16x8, ld16(qp + 32 * c + 8 * hq));
  const int ends = sq.key_end(a, tok);
  const int khi = ends < hi ? ends : hi;
  const int kfull = wave_uniform(sq.key_end(a, 0));  // every row sees these

  f32x4 o[4] = {};  // O^T [16-d block]: lane (row l16, hq) holds d 16 db + 4 hq + r
  float m = -INFINITY, lsum = 0.f;
  const int tr_row = l16 >> 2;
  const int tr_col = 4 * (lane & 3);
  for (int i = 0; i < kv.mine; ++i) {
    const int c0 = kv.first_key(i);
    const uint32_t there = kv.there;
    kv.stage(ks, vs);
    if (i + 1 < kv.mine) kv.load(i + 1);
    f32x4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const __bf16* kt = &ks[(16 * kb + l16) * kStride + 8 * hq];
      s[kb] = mfma16(*reinterpret_cast<const bf16x8*>(kt), qreg[0], f32x4{});
      s[kb] = mfma16(*reinterpret_cast<const bf16x8*>(kt + 32), qreg[1], s[kb]);
    }
    if (c0 + kSub > kfull || c0 + kSub > hi || there != 3) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[kb][r] = c0 + 16 * kb + 4 * hq + r < khi && ((there >> kb) & 1) ? s[kb][r] : -INFINITY;
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = fmaxf(mx, shfl_xor(mx, 16));
    mx = max_xor32(mx);
    const float mt = mx * a.scale_log2;
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
  if (tid < 16 * kRows) ml->write_row(a, ranges, it, tid >> 4, 4 * (tid & 15));
}

template <int NW, int ROWS>
__global__ __launch_bounds__(NW * 64, ROWS == 16 ? 4 : NW == 4 ? 3 : 2) void paged_rows_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[chunk_smem<NW, ROWS>()];
  // The launch has about as many workgroups as there are items; those left over
  // (lengths that the caller's total did not tell) are taken in turn.
  for (int id = wg_x();; id += a.workgroups) {
    const PagedItem<false> it(a, id);
    if (!it.found) return;
    if constexpr (ROWS == 16)
      paged16_item<NW>(a, it, smem);
    else
      paged32_item<NW>(a, it, smem);
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
constexpr float kRescale = 8.0f;

template <int SUBS>
__global__ __launch_bounds__(256 * SUBS, 4) void paged128_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(1024))) __bf16 smem_all[SUBS][2][2][kSwTile];  // [set][stage][K | V]
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
    const PagedItem<true> it(a, wg_x());
    if (!it.found) return;
    b = it.b;
    h = it.h;
    sq = it.sq;
    qt = it.qt;
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
  const uint16_t* kh = a.k + h * a.sk_h;
  const uint16_t* vh = a.v + h * a.sv_h;
  uint32_t there = 0;  // quarters of the tile requested last whose page exists
  auto issue = [&](int i) {  // the set's i-th tile
    if ((i & 15) == 0 && i > 0) {
      ids = ids_next;
      ok = __ballot((unsigned)ids < (unsigned)a.pages);
    }
    if ((i & 15) == 8) ids_next = entries((i | 15) + 1);
    const int at = 4 * (i & 15) + wave;
    const int key = lo + (sub + SUBS * i) * kSwRows + 16 * wave;
    there = (uint32_t)(ok >> (4 * (i & 15))) & 15u;
    const uint32_t dst = lds_w + (uint32_t)(i & 1) * 16384u;
    const int lim = (ok >> at) & 1 ? sq.kv - 1 - key : -1;  // the last of its 16 rows that is a key
    const int64_t page = __builtin_amdgcn_readlane(ids, at);
    const int64_t slot = key & (a.page - 1);
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
  if (n_mine > 0) issue(0);
#pragma unroll
  for (int c = 0; c < 4; ++c) asm volatile("" ::"v"(qreg[c]));  // waits for Q here, not in the loop

  const int khi = sq.key_end(a, tok);  // the lane's row sees [0, khi)
  const int wave_last = qrow0 + 31 < sq.rows ? qrow0 + 31 : sq.rows - 1;
  const int emax = qrow0 < sq.rows ? wave_uniform(sq.key_end(a, fast_div(wave_last, a.group_div))) : 0;
  const int emin = qrow0 < sq.rows ? wave_uniform(sq.key_end(a, fast_div(qrow0, a.group_div))) : 0;

  f32x16 o[2] = {};  // O^T [d block]
  float mref = 0.f, lsum = 0.f;
  bool valid = false;  // the row has met a key
  const float c2 = a.scale_log2;
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
    float mrow = -INFINITY;
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int r = 0; r < 16; r += 2) mrow = fmaxf(fmaxf(mrow, s[sb][r]), s[sb][r + 1]);
    const float mt = fmaf(max_xor32(mrow), c2, -mref);
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
      for (int r = 0; r < 16; ++r) p[r] = fast_exp2(fmaf(s[sb][r], c2, -mref));
#pragma unroll
      for (int kc = 0; kc < 2; ++kc) {
        const bf16x8 pop = to_bf16x8(p[8 * kc], p[8 * kc + 1], p[8 * kc + 2], p[8 * kc + 3], p[8 * kc + 4],
                                     p[8 * kc + 5], p[8 * kc + 6], p[8 * kc + 7]);
        lsum += ((p[8 * kc] + p[8 * kc + 1]) + (p[8 * kc + 2] + p[8 * kc + 3])) +
                ((p[8 * kc + 4] + p[8 * kc + 5]) + (p[8 * kc + 6] + p[8 * kc + 7]));
#pragma unroll
        for (int db = 0; db < 2; ++db) o[db] = mfma32(sw_tr_op(vs, 32 * sb + 16 * kc, 32 * db, lane), pop, o[db]);
      }
    }
  };

  uint32_t seen = there;
  vm_wait_barrier<0>();
  const int steps = (n_tiles + SUBS - 1) / SUBS;  // of the set with the most tiles
  for (int i = 0; i < steps; ++i) {
    if (i + 1 < n_mine) issue(i + 1);
    const int k0 = lo + (sub + SUBS * i) * kSwRows;
    if (i < n_mine && k0 < emax) step(k0, seen, smem[i & 1][0], smem[i & 1][1]);
    seen = there;
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
  const int r0 = row & -a.tile;
  const int keys = sq.key_end(a, fast_div((r0 + a.tile < sq.rows ? r0 + a.tile : sq.rows) - 1, a.group_div));
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
    dst = kh < a.kv_heads ? a.k + (int64_t)page * a.sk_p + (int64_t)kh * a.sk_h + slot * a.sk_s
                          : a.v + (int64_t)page * a.sv_p + (int64_t)(kh - a.kv_heads) * a.sv_h + slot * a.sv_s;
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

hipError_t launch_paged_attn(const PagedArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.workgroups);
  if (a.tile == 128) {
    if (a.subs == 4)
      hipLaunchKernelGGL(paged128_kernel<4>, grid, dim3(1024), 0, stream, a);
    else if (a.subs == 2)
      hipLaunchKernelGGL(paged128_kernel<2>, grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL(paged128_kernel<1>, grid, dim3(256), 0, stream, a);
  } else {
    if (a.tile == 16)
      hipLaunchKernelGGL((paged_rows_kernel<8, 16>), grid, dim3(512), 0, stream, a);
    else if (a.subs == 2)
      hipLaunchKernelGGL((paged_rows_kernel<8, 32>), grid, dim3(512), 0, stream, a);
    else
      hipLaunchKernelGGL((paged_rows_kernel<4, 32>), grid, dim3(256), 0, stream, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.n_splits == 1) return e;
  hipLaunchKernelGGL(paged_combine_kernel, dim3((unsigned)(a.kv_heads * a.part_slots)), dim3(16 * kMergeRows), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_rope(const PagedRopeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(paged_rope_kernel, dim3((unsigned)((a.total + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace bd3
