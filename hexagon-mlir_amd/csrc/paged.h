// What the kernels of a paged cache share: whole-number division by an argument, the tokens of a batch, where a position stands.
#pragma once
#include "hexmi_common.h"

namespace hexmi {

// n / d for 0 <= n < 2^31, by a product (d from 1): with l = ceil(log2 d), m = ceil(2^(31 + l) / d) is below 2^32 and exceeds
// 2^(31 + l) / d by less than 2^l / d <= 2^(31 + l) / (d n), so the floor is right.
struct Divider {
  uint32_t m, shift;
};
inline Divider divider(int64_t d) {
  uint32_t l = 0;
  while ((int64_t(1) << l) < d) ++l;
  return {(uint32_t)(((uint64_t(1) << (31 + l)) + (uint64_t)d - 1) / (uint64_t)d), 31 + l};
}
#if defined(__HIPCC__)
__device__ __forceinline__ int divided(int n, const Divider& d) { return (int)(((uint64_t)(uint32_t)n * d.m) >> d.shift); }
#endif

// hexmi_paged_batch as the kernels take it: sizes below 2^31 (batch_fits), strides in elements.
struct Pages {
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
  const int32_t *table, *lengths, *starts;
  int64_t table_row;
  int num_pages, page_size, table_cols, sequences, tokens, kv_heads;
  Divider size;
};
inline Pages pages_of(const hexmi_paged_batch& b) {
  return {b.k_page, b.k_head, b.k_slot, b.v_page, b.v_head, b.v_slot, b.page_table, b.lengths, b.starts, b.table_row, (int)b.num_pages,
          (int)b.page_size, (int)b.table_cols, (int)b.sequences, (int)b.tokens, (int)b.kv_heads, divider(b.page_size)};
}
// HEXMI_OK, or why a batch is refused (pointers aside)
inline int check_batch(const hexmi_paged_batch& b) {
  if (b.num_pages < 1 || b.page_size < 1 || b.kv_heads < 1 || b.dim < 1 || b.table_cols < 0 || b.sequences < 0 || b.tokens < 0 ||
      (b.sequences > 1 && b.table_row < b.table_cols))
    return HEXMI_EINVAL;
  if (!b.starts && b.sequences != b.tokens) return HEXMI_EINVAL;
  constexpr int64_t most = 0x7fffffff;
  if (b.num_pages > most || b.page_size > most || b.kv_heads > 65535 || b.table_cols > most || b.sequences > most / 2 || b.tokens > most / 2 ||
      (b.table_cols > 0 && b.page_size > (most - 1024) / b.table_cols))
    return HEXMI_ENOTSUP;
  return HEXMI_OK;
}

#if defined(__HIPCC__)
// The sequence of row t: the last b with starts[b] <= t, by the 64 lanes of a wave together (t the same for all): 64 places are asked
// at once, so 64 sequences take one read and 4096 two. -1: none (below starts[0], from starts[sequences] on).
__device__ __forceinline__ int sequence_of(const Pages& p, int t, int lane) {
  int lo = 0, hi = p.sequences + 1;                       // among starts[0 .. sequences]
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const bool below = at < hi && p.starts[at] <= t;
    const int n = __popcll(__ballot(below));
    if (n == 0) return -1;
    lo += (n - 1) * step;
    hi = lo + step < hi ? lo + step : hi;
    if (step == 1) break;
  }
  return lo < p.sequences && p.starts[lo] <= t ? lo : -1;
}

// The rows of sequence b, from the first of them to the first of b + 1: -1 and `sequences` are the rows of no sequence before the first and
// behind the last; all within the operands, whatever starts holds. A sequence's end, and so its tokens' positions, go by this everywhere.
__device__ __forceinline__ int first_row(const Pages& p, int b) {
  const int s = b < 0 ? 0 : b > p.sequences ? p.tokens : p.starts ? p.starts[b] : b;
  return s < 0 ? 0 : s < p.tokens ? s : p.tokens;
}
__device__ __forceinline__ int new_tokens_of(const Pages& p, int b) { return p.starts ? first_row(p, b + 1) - first_row(p, b) : 1; }

// The positions of sequence b that have a place in the table, whatever lengths holds.
__device__ __forceinline__ int length_of(const Pages& p, int b) {
  const int most = p.table_cols * p.page_size, n = p.lengths[b];
  return n < 0 ? 0 : n < most ? n : most;
}
#endif

// How attention holds a head: D columns of a row in LDS, COLS <= D of them multiplied (a multiple of 32), PADDED: the head is narrower than COLS.
template <int D_, int COLS_, bool PADDED_> struct HeadWidth {
  static constexpr int D = D_, COLS = COLS_;
  static constexpr bool PADDED = PADDED_;
};
template <int D, int COLS, typename F> int with_columns(int64_t dim, F&& f) {
  return dim == COLS ? f(HeadWidth<D, COLS, false>{}) : f(HeadWidth<D, COLS, true>{});
}
// f of the width that heads of dim columns go by, up to MOST (128 or 256)
template <int MOST, typename F> int with_width(int64_t dim, F&& f) {
  if (dim <= 64) return with_columns<64, 64>(dim, f);
  if (dim <= 96) return with_columns<128, 96>(dim, f);
  if constexpr (MOST == 128) return with_columns<128, 128>(dim, f);
  else return dim <= 128 ? with_columns<128, 128>(dim, f) : with_columns<256, 256>(dim, f);
}
// The first of the eight columns that a tile copies to where columns c .. c + 7 of an LDS row stand. The row is wider than the head where
// the head is padded, and where fewer columns than the row's are multiplied (heads of 96): what stands behind the head there is no part
// of it, and nobody multiplies it or stores what comes of it, so the head's first columns are copied.
template <int D, int COLS, bool PADDED> constexpr int copied_column(int c, int dim) { return (PADDED || COLS < D) && c >= dim ? 0 : c; }

// How far (log2) the reference of a softmax stands below the largest score when it is set: probabilities, which go to the matrix cores
// rounded to T, are 2^kLift there, and up to 2^(kLift + kRescaleLag) before it is set again. fp16 has no more than 2^-24 below 1, so without
// it a key of 2^-25 of the largest one's weight was nothing, and 2^17 of them with it; 2^15 is as far as fp16 goes, and the step is 2^-31 of the
// largest weight so. bf16 has the exponents of fp32.
template <typename T> constexpr float kLift = 0.0f;
template <> inline constexpr float kLift<f16> = 7.0f;

// What attention over the pages takes beside them (paged_attn.hip, paged_decode.hip).
struct PagedAttnArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_token, q_head, out_token, out_head;
  const int32_t* shared;                       // the pages of the positions below `prefix`
  int prefix, heads, group, dim;               // group: query heads of a key head
  float scale;                                 // sm_scale * log2 e
  Divider by_group;
};
// Sums that several workgroups hold of a row: slot i of row (token * heads + head) has the row's unnormalised output, dim floats at
// o + (i * rows + row) * dim, and (maximum in log2 units, sum) at ml[i * rows + row]; sum 0: no key, and o is not written.
struct RowSums {
  float* o;
  float2* ml;
  int64_t rows;
  int slots;
};
// One launch: the prefix for all rows (the first workgroups), and every sequence's keys behind it.
struct TileArgs {
  bool deep;                                   // DeepTile (paged_tile.h), or WideTile
  bool workers;                                // sequences of one new token are the workers' (paged_decode.h)
  int shared_tiles, shared_splits;             // tiles of a key head; parts of the prefix, whose sums go to slots 0 .. (0: no prefix)
  int tiles, splits;                           // of the sequences' own keys, whose sums go to the slots behind (0: decode, not here)
  RowSums sums;                                // slots 0: the result goes to out
};

// One new token a sequence: how the keys are shared out (workers; 0: every unit of sequence, key head and 16 query heads whole).
struct PagedDecodePlan {
  int workers, row_tiles, rows;
};
// A unit that a worker begins and others go on with: its sequence, unit and last worker (none: last < 0).
struct BegunUnit {
  int sequence, unit, last, pad;
};
struct DecodeArgs {
  float* part_o;                               // [workers][2][16][dim]
  float2* part_ml;                             // [workers][2][16]
  BegunUnit* begun;                               // [workers]
  int workers, row_tiles;
  RowSums sums;                                // slots 0: rows go to out
  int own;                                     // otherwise the slot of the sequences' own keys
  bool join_all;                               // own is the last slot, and every unit is joined with the prefix's sums
};
PagedDecodePlan plan_paged_decode(const hexmi_paged_batch& b, int64_t heads, int64_t prefix);
int64_t paged_decode_workspace(const PagedDecodePlan& plan, int64_t dim);
// One new token a sequence, or those sequences of a batch that have one, with the tiles (none: splits and shared_splits 0) of the prefix and the
// others. Rows whose sums are to be joined (tiles.sums) are left there, but for one token a sequence throughout.
int paged_decode(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, int dtype, void* workspace, const TileArgs& tiles,
                 hipStream_t s);
// tiles and `grid` workers in one launch (paged_shared.hip)
int paged_shared_decode(const PagedAttnArgs& a, const Pages& p, const TileArgs& tiles, const DecodeArgs& w, unsigned grid, int dtype,
                        hipStream_t s);

}  // namespace hexmi
