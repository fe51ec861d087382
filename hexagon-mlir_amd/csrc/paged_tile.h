// A tile of query rows over the pages of a cache (paged_attn.hip, paged_shared.hip).
//
// The query rows of a key head, (token, head of its group) one behind the other, are cut into tiles of kRows; a workgroup of four waves
// takes a tile, 32 rows a wave, and walks the keys up to its last token's own in blocks of 64, as flash_attn.hip does: S^T = K Q^T with
// v_mfma_f32_32x32x16, online softmax in registers, O^T += V^T P^T with V read transposed from LDS. What differs is where things stand:
// a block's 64 pages are looked up a block ahead, a lane each, a key's row is copied into LDS from wherever its page is, and a block
// carries a bit a key that says whether it is one. Heads that share their keys share a tile, so a step of decode in a batch with
// prompts reads its keys once too; a wave whose rows are none only copies.
//
// The prefix is one sequence that all rows of the batch attend: its keys go through LDS once for kRows rows, whatever sequences they are
// of. Its sums, and those of tiles whose keys are cut over several workgroups because there are few, go through the workspace.
//
// What bounds it. Prompts of 4 x 4096, 32 heads over 8 of 128, bf16: 587 us, 0.93 PFLOP/s (a matrix product of 8192^3 1.12). Without the
// copies it takes 432 us, with nothing but them 332: a wave reads all of a block out of LDS for its 32 rows, as many cycles as the matrix
// instructions take, and two workgroups a compute unit hide that in part. Measured on the way: copies that the compiler knows of (it waits
// for them before it reads LDS transposed) 609; a lane's own address for every row 687. Few rows are bound by what is one behind the other:
// launch and look-up about 5 us, 1 to 2 us a block (its copies are all waited for before the next block is begun), the join 4 to 5.
#pragma once
#include "flash_attn_tiles.h"
#include "paged.h"

namespace hexmi {
namespace {

// KEYS a block, ROW_WAVES waves of 32 rows each, GROUPS of such waves that take every GROUPS-th block each, with LDS of their own.
template <int KEYS, int ROW_WAVES, int GROUPS> struct TileShape {
  static constexpr int kKeys = KEYS, kRowWaves = ROW_WAVES, kGroups = GROUPS, kRows = ROW_WAVES * 32, kThreads = ROW_WAVES * GROUPS * kWave;
  // LDS of D columns of 16 bits: K and V of two blocks a group, later the groups' sums in 32 bits
  static constexpr int lds_elements(int d) { return GROUPS * 4 * KEYS * d; }
  static_assert(4 * KEYS * 2 == kRows * 4, "a group's sums take the place of its blocks");
};
typedef TileShape<64, 4, 1> WideTile;          // many tiles: 128 rows; two workgroups a compute unit (heads of 64 three)
typedef TileShape<32, 2, 2> DeepTile;          // few: 64 rows, the chain of a tile's keys half as long

// The tiles of a key head: those of sequence b are numbered from first_tile(b) on, b = -1 .. sequences (first_row).
// floor(x / r) + 1 >= ceil(n / r) + floor(x0 / r) for x = x0 + n, so a sequence's tiles end before the next one's begin; some numbers are
// no tile.
template <int ROWS>
__device__ __forceinline__ int first_tile(const Pages& p, int group, int b) { return b < 0 ? 0 : first_row(p, b) * group / ROWS + b + 1; }
template <int ROWS>
__device__ __forceinline__ int sequence_of_tile(const Pages& p, int group, int tile, int lane) {
  int lo = -1, hi = p.sequences + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const int n = __popcll(__ballot(at < hi && first_tile<ROWS>(p, group, at) <= tile));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
    if (step == 1) break;
  }
  return lo;
}

// The sequence of a tile, its rows from `first` to `next`, and its length. Where the sequences are a lane each, starts and lengths come in
// one trip to memory.
struct Run {
  int sequence, first, next;
  int64_t length;
};
template <int ROWS>
__device__ __forceinline__ Run run_of_tile(const Pages& p, int group, int tile, int lane) {
  Run run;
  if (p.sequences > 0 && p.sequences <= kWave - 3) {                // lanes of -1 .. sequences + 1
    const int at = lane - 1, s = p.starts[at < 0 ? 0 : at < p.sequences ? at : p.sequences];
    const int length = p.lengths[at < 0 ? 0 : at < p.sequences ? at : p.sequences - 1];
    const int row = at < 0 || s < 0 ? 0 : at > p.sequences || s > p.tokens ? p.tokens : s;
    const int n = __popcll(__ballot(at <= p.sequences && (at < 0 ? 0 : row * group / ROWS + at + 1) <= tile));      // lane 0 is one
    run = {n - 2, __builtin_amdgcn_readlane(row, n - 1), __builtin_amdgcn_readlane(row, n), __builtin_amdgcn_readlane(length, n - 1)};
  } else {
    const int b = __builtin_amdgcn_readfirstlane(sequence_of_tile<ROWS>(p, group, tile, lane));
    run = {b, first_row(p, b), first_row(p, b + 1), b >= 0 && b < p.sequences ? p.lengths[b] : 0};
  }
  return run;
}

// keys that token i of a sequence's n sees, whatever the index tensors hold
__device__ __forceinline__ int keys_of(int64_t length, int n, int i, int most) {
  const int64_t keys = length - n + i + 1;
  return keys < 0 ? 0 : keys < most ? (int)keys : most;
}

// D, COLS, PADDED: HeadWidth. A lane whose columns lie past the head copies the head's first ones instead (copied_column): the query has
// zeros there or they are not multiplied, and what comes of V there is not stored.
// A workgroup's tile: number block_id of a launch whose tiles are `grid` workgroups; lds: Shape::lds_elements(D); m_lds, l_lds: of every
// group's rows.
template <typename T, int D, int COLS, bool PADDED, typename Shape>
__device__ __forceinline__ void paged_tile(const PagedAttnArgs& a, const Pages& p, const TileArgs& w, unsigned block_id, unsigned grid,
                                           T* lds, float (*m_lds)[Shape::kRows], float (*l_lds)[Shape::kRows]) {
  typedef typename MfmaT<T>::Frag Frag;
  constexpr int kKeys = Shape::kKeys, kRowWaves = Shape::kRowWaves, kGroups = Shape::kGroups, kRows = Shape::kRows, JT = kKeys / 32;
  constexpr int DS = COLS / 16, DT = COLS / 32, CPR = D / 8;
  constexpr int NI = kKeys * CPR / kWave / kRowWaves, kRowStep = kRowWaves * kWave / CPR;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32;
  const int group = wave / kRowWaves, row_wave = wave % kRowWaves;
  constexpr int kTile = kKeys * D;
  T *k_lds0 = lds + group * 4 * kTile, *k_lds1 = k_lds0 + kTile, *v_lds0 = k_lds1 + kTile, *v_lds1 = v_lds0 + kTile;
  const int dim = PADDED ? a.dim : COLS;

  // Workgroup -> (prefix or not, key head, tile, part). Workgroup ids go round robin to the 8 XCDs (one L2 each): every XCD gets a run of
  // the list, key head by key head, a sequence's last (longest) tiles first.
  const unsigned shared_grid = (unsigned)(w.shared_tiles * w.shared_splits * p.kv_heads);
  const bool shared = block_id < shared_grid;
  const int tiles = shared ? w.shared_tiles : w.tiles, splits = shared ? w.shared_splits : w.splits;
  const unsigned id = shared ? block_id : block_id - shared_grid, count = shared ? shared_grid : grid - shared_grid;
  const unsigned xcd = id % 8, each = count / 8, more = count % 8;
  const unsigned unit = xcd * each + (xcd < more ? xcd : more) + id / 8;
  const int part = unit % splits, tile = tiles - 1 - (int)(unit / splits % tiles), kvh = unit / splits / tiles;

  int token0 = 0, rows, row0, new_tokens = 0, begin = 0, end;
  int64_t length = 0;
  bool none = false;                                                // rows of no sequence
  const int most = p.table_cols * p.page_size;
  const int32_t* table;
  if (shared) {
    row0 = tile * kRows;
    rows = p.tokens * a.group;
    end = a.prefix;
    table = a.shared;
  } else {
    const Run run = run_of_tile<kRows>(p, a.group, tile, lane);
    const int b = run.sequence;
    token0 = run.first;
    new_tokens = run.next - token0;
    row0 = (tile - (b < 0 ? 0 : token0 * a.group / kRows + b + 1)) * kRows;
    rows = new_tokens * a.group;                                    // negative where starts fall: nothing
    if (row0 < 0 || row0 >= rows) return;
    none = b < 0 || b >= p.sequences;
    if (w.workers && new_tokens == 1 && !none) return;
    if (!none) length = run.length;
    const int last = row0 + kRows < rows ? row0 + kRows - 1 : rows - 1;
    end = none ? 0 : keys_of(length, new_tokens, divided(last, a.by_group), most);
    begin = a.prefix;
    table = p.table + (none ? 0 : b) * p.table_row;
  }
  end = __builtin_amdgcn_readfirstlane(end);
  const int blocks = end > begin ? (end - begin + kKeys - 1) / kKeys : 0, share = (blocks + splits - 1) / splits;
  const int block0 = part * share, block1 = block0 + share < blocks ? block0 + share : blocks;

  const int first = block0 + group;                                 // this group's blocks: first, first + kGroups, ..

  // ---- copies: instruction j of a wave takes kRowsOfOne rows, a lane 16 bytes of one
  const T* k_head = static_cast<const T*>(a.k) + kvh * p.k_head;
  const T* v_head = static_cast<const T*>(a.v) + kvh * p.v_head;
  const int lin = row_wave * kWave + lane, copy_row = lin / CPR, lds_at = row_wave * kWave * 8;
  // The table's entry for key kKeys block + lane. No branch: it is asked for a block ahead, and what it is worth is looked at then (a load
  // behind a branch would be waited for where the branch ends).
  auto find = [&](int block) __attribute__((always_inline)) {
    const int key = begin + block * kKeys + lane % kKeys;
    return table[divided(key < end ? key : end - 1, p.size)];       // end > begin: only asked then
  };
  auto page_at = [&](int block, int entry) __attribute__((always_inline)) {     // -1: no key there
    return block < block1 && begin + block * kKeys + lane % kKeys < end && entry >= 0 && entry < p.num_pages ? entry : -1;
  };
  // One block into LDS, by copies that the compiler does not know of: it would wait for all of them before it reads LDS transposed, in the
  // middle of the block before. They are waited for ahead of the barrier that ends that block. Where every key is there and the rows of an
  // instruction share a page, the page, and so the place, is the wave's (scalar arithmetic), and a lane adds what it is off in it; any other
  // block goes row by row.
  constexpr int kRowsOfOne = kWave / CPR;
  const bool one_page = p.page_size % kRowsOfOne == 0;
  auto column = [&](bool v, int r) __attribute__((always_inline)) {
    const int c = ((lin % CPR) ^ (v ? swz_vtile<D == 64 ? 64 : 128>(r) : swz_ktile<D == 64 ? 64 : 128>(r))) * 8;
    return copied_column<D, COLS, PADDED>(c, dim);
  };
  auto copy = [&](int block, int page_of_lane, T* k_dst, T* v_dst) __attribute__((always_inline)) {
    if (one_page && __ballot(page_of_lane >= 0) == ~0ull) {
      // a lane works out where its key stands, for all of the block's at once; an instruction takes its first row's
      const int key_of_lane = begin + block * kKeys + lane % kKeys, slot_of_lane = key_of_lane - divided(key_of_lane, p.size) * p.page_size;
      const int64_t k_at = page_of_lane * p.k_page + slot_of_lane * p.k_slot, v_at = page_of_lane * p.v_page + slot_of_lane * p.v_slot;
      auto first_of = [&](int64_t at, int j) __attribute__((always_inline)) {
        const int row = row_wave * kRowsOfOne + j * kRowStep;
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)at, row), hi = __builtin_amdgcn_readlane((int)(at >> 32), row);
        return (int64_t)((uint64_t)hi << 32 | lo);
      };
      constexpr int kStep = kRowWaves * kWave * 16;                 // bytes of LDS between a wave's instructions
#pragma unroll
      for (int v = 0; v < 2; ++v)
#pragma unroll
        for (int j = 0; j < NI; j += 2) {
          const T* head = v ? v_head : k_head;
          const int64_t at = v ? v_at : k_at;
          const int step = lane / CPR * (int)(v ? p.v_slot : p.k_slot);
          copy_two_to_lds_asm<kStep>(reinterpret_cast<const char*>(head + first_of(at, j)), (step + column(v, copy_row + j * kRowStep)) * 2,
                                     reinterpret_cast<const char*>(head + first_of(at, j + 1)),
                                     (step + column(v, copy_row + (j + 1) * kRowStep)) * 2,
                                     reinterpret_cast<char*>((v ? v_dst : k_dst) + lds_at) + j * kStep);
        }
      return;
    }
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int r = copy_row + j * kRowStep, key = begin + block * kKeys + r, page = __shfl(page_of_lane, r);
      const int slot = key - divided(key, p.size) * p.page_size;
      T *k_to = k_dst + lds_at + j * (kRowWaves * kWave * 8), *v_to = v_dst + lds_at + j * (kRowWaves * kWave * 8);
      if (page >= 0) {
        copy_ptr_to_lds_asm(reinterpret_cast<const char*>(k_head + page * p.k_page + slot * p.k_slot + column(false, r)), reinterpret_cast<char*>(k_to));
        copy_ptr_to_lds_asm(reinterpret_cast<const char*>(v_head + page * p.v_page + slot * p.v_slot + column(true, r)), reinterpret_cast<char*>(v_to));
      } else {                                                      // no key: whatever the cache holds, zeros of V (its score is dropped)
        *reinterpret_cast<u32x4*>(v_to + lane * 8) = u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  int page = -1, next = -1;
  if (block0 < block1) {                                            // on their way while the rows are looked up
    page = find(first);
    next = find(first + kGroups);
    page = page_at(first, page);
    if (first < block1) copy(first, page, k_lds0, v_lds0);
  }

  // this lane's row: its token, its queries and the keys it sees
  const int wave_row = row0 + row_wave * 32, row = wave_row + lane % 32;
  const bool live = row < rows;
  const int in_seq = divided(live ? row : rows - 1, a.by_group), head = kvh * a.group + (live ? row : rows - 1) - in_seq * a.group;
  const int token = token0 + in_seq;
  Frag qf[DS];                                                      // row lane % 32, columns 16 ds + 8 half ..
  {
    const T* q = static_cast<const T*>(a.q) + token * a.q_token + head * a.q_head;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      const int c = ds * 16 + half * 8;
      if (!PADDED || c < dim) qf[ds] = *reinterpret_cast<const Frag*>(q + c);
      else qf[ds] = Frag{};
    }
  }
  int keys = 0;
  if (shared) {
    int s = token;                                                  // the row's sequence: this lane's own search
    if (p.starts) {
      int lo = 0, hi = p.sequences + 1;                             // the last one with starts[s] <= token, among 0 .. sequences
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.starts[mid] <= token) lo = mid;
        else hi = mid;
      }
      s = lo < p.sequences && p.starts[lo] <= token ? lo : -1;
    }
    if (live && s >= 0) keys = keys_of(p.lengths[s], first_row(p, s + 1) - token, 0, most);
    keys = keys < a.prefix ? keys : a.prefix;
  } else if (live && !none) {
    keys = keys_of(length, new_tokens, in_seq, most);
  }
  // the wave's rows together: beyond the most that one sees a block is nothing to it, up to the least none is hidden
  int most_keys = keys, least_keys = live ? keys : 0x7fffffff;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) {
    const int m1 = __shfl_xor(most_keys, x), m2 = __shfl_xor(least_keys, x);
    most_keys = most_keys > m1 ? most_keys : m1;
    least_keys = least_keys < m2 ? least_keys : m2;
  }
  most_keys = __builtin_amdgcn_readfirstlane(most_keys);
  least_keys = __builtin_amdgcn_readfirstlane(least_keys);

  f32x16 o_acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[dt][r] = 0.0f;
  float m_i = -INFINITY, neg_m = 0.0f, l_i = 0.0f;

  auto process = [&](int block, uint64_t there, int next_page, const T* k_src, const T* v_src, T* k_dst, T* v_dst) __attribute__((always_inline)) {
    const int key0 = begin + block * kKeys;
    if (block + kGroups < block1) copy(block + kGroups, next_page, k_dst, v_dst);
    if (block >= block1 || key0 >= most_keys) return;               // wave-uniform; the barriers are outside
    f32x16 s[JT];
#pragma unroll
    for (int jt = 0; jt < JT; ++jt)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[jt][r] = 0.0f;
    {
      constexpr int kAhead = 3;
      auto read_k = [&](int jt, int ds) __attribute__((always_inline)) {
        const int r = jt * 32 + lane % 32, c = (ds * 2 + half) ^ swz_ktile<D == 64 ? 64 : 128>(r);
        return *reinterpret_cast<const Frag*>(k_src + (r * CPR + c) * 8);
      };
      Frag kf[JT][DS];
#pragma unroll
      for (int ds = 0; ds < kAhead && ds < DS; ++ds)
#pragma unroll
        for (int jt = 0; jt < JT; ++jt) kf[jt][ds] = read_k(jt, ds);
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        if (ds + kAhead < DS)
#pragma unroll
          for (int jt = 0; jt < JT; ++jt) kf[jt][ds + kAhead] = read_k(jt, ds + kAhead);
#pragma unroll
        for (int jt = 0; jt < JT; ++jt) s[jt] = MfmaT<T>::run(kf[jt][ds], qf[ds], s[jt]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // fragments of V: of a 32-key tile they are read ahead of its probabilities, but for heads of 256 columns, whose registers they are
    constexpr int kPieces = D == 256 ? 1 : 2 * DT;
    struct VFrags { Frag f[kPieces]; };
    auto read_piece = [&](int jt, int piece) __attribute__((always_inline)) {
      const int g = lane / 16, i16 = lane % 16, hf = piece / DT, dt = piece % DT;
      union { i16x4 h[2]; Frag f; } u;
#pragma unroll
      for (int pp = 0; pp < 2; ++pp) {
        const int r = jt * 32 + hf * 16 + 8 * pp + 4 * (g >> 1) + (i16 >> 2), col = dt * 32 + (g & 1) * 16 + (i16 & 3) * 4;
        const int c = (col / 8) ^ swz_vtile<D == 64 ? 64 : 128>(r);
        u.h[pp] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(v_src + (r * CPR + c) * 8 + col % 8));
      }
      return u.f;
    };
    auto read_v = [&](int jt, VFrags& vf) __attribute__((always_inline)) {
      if constexpr (kPieces > 1) {
#pragma unroll
        for (int piece = 0; piece < kPieces; ++piece) vf.f[piece] = read_piece(jt, piece);
      }
    };
    VFrags vf0, vf1;
    read_v(0, vf0);
    __builtin_amdgcn_sched_barrier(0);
    // s[jt][r] is the score of key key0 + 32 jt + 8 (r / 4) + 4 half + r % 4
    if (there != ~0ull || key0 + kKeys > least_keys) {
      const uint32_t bits[2] = {(uint32_t)there >> (4 * half), (uint32_t)(there >> 32) >> (4 * half)};
#pragma unroll
      for (int jt = 0; jt < JT; ++jt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int at = 8 * (r / 4) + r % 4;
          if (!(bits[jt] >> at & 1) || key0 + jt * 32 + at + 4 * half >= keys) s[jt][r] = -INFINITY;
        }
    }
    float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[0][r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) mx1 = fmaxf(mx1, s[JT - 1][r]);
    mx = fmaxf(mx, mx1);
    mx = fmaxf(mx, other_half(mx)) * a.scale;
    const bool grow = mx > m_i + (kLift<T> + kRescaleLag);          // the reference may lag (flash_attn.hip)
    if (__ballot(grow) != 0) {
      const float m_new = grow ? mx - kLift<T> : m_i, alpha = grow ? __builtin_amdgcn_exp2f(m_i - m_new) : 1.0f;
      l_i *= alpha;
      m_i = m_new;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[dt][r] *= alpha;
      neg_m = m_i == -INFINITY ? 0.0f : -m_i;
    }
    Frag pf[2];
    auto exp_tile = [&](const f32x16& t) __attribute__((always_inline)) {
      float pr[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) pr[r] = __builtin_amdgcn_exp2f(fmaf(t[r], a.scale, neg_m));
      // Rounded to T, as the matrix instruction takes them beside V: a second product with what the rounding leaves would be half as much
      // again of the arithmetic. Off from 64 bits by 1.2 to 1.4 times what the result's own rounding is (fp16 2.9e-4 and 2.1e-4 of the
      // result, bf16 2.1e-3 and 1.7e-3).
      pf[0] = MfmaT<T>::pack(&pr[0]);
      pf[1] = MfmaT<T>::pack(&pr[8]);
      l_i += MfmaT<T>::sum8(pf[1], MfmaT<T>::sum8(pf[0], 0.0f));    // the sum of what the product multiplies, these keys' first: two at a
                                                                    // time to a sum 2^25 times as large are nothing
    };
    auto pv = [&](int jt, const VFrags& vf) __attribute__((always_inline)) {
#pragma unroll
      for (int piece = 0; piece < 2 * DT; ++piece) {
        o_acc[piece % DT] = MfmaT<T>::run(kPieces > 1 ? vf.f[piece % kPieces] : read_piece(jt, piece), pf[piece / DT], o_acc[piece % DT]);
        if (kPieces == 1 && piece % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    };
    if constexpr (JT == 2) read_v(1, vf1);
    exp_tile(s[0]);
    pv(0, vf0);
    if constexpr (JT == 2) {
      exp_tile(s[1]);
      pv(1, vf1);
    }
  };

  // the queries are here before the walk begins: their first use must not wait inside it, with copies on their way
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) {
    u32x4 f = __builtin_bit_cast(u32x4, qf[ds]);
    asm volatile("" : "+v"(f));
    qf[ds] = __builtin_bit_cast(Frag, f);
  }
  for (int block = first, at = block0; at < block1; block += 2 * kGroups, at += 2 * kGroups) {      // as many turns for every group
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint64_t there = __ballot(page >= 0);
    page = page_at(block + kGroups, next);
    next = find(block + 2 * kGroups);
    process(block, there, page, k_lds0, v_lds0, k_lds1, v_lds1);
    if (at + kGroups >= block1) break;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    there = __ballot(page >= 0);
    page = page_at(block + 2 * kGroups, next);
    next = find(block + 3 * kGroups);
    process(block + kGroups, there, page, k_lds1, v_lds1, k_lds0, v_lds0);
  }
  __syncthreads();

  // ---- o_acc[dt][r] is column 32 dt + 8 (r / 4) + 4 half + r % 4 of the row's sum. A lane holds four columns of its row at a time; they
  // leave as whole rows, through the LDS that held the blocks (16-byte chunks XOR swizzled by the row), where the groups' sums meet.
  const float l = l_i + other_half(l_i);
  const bool parts = w.sums.slots != 0;
  const float own = kGroups > 1 || parts ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
  const int64_t slot = (int64_t)(part + (shared ? 0 : w.shared_splits)) * w.sums.rows;
  float* sums = reinterpret_cast<float*>(lds);
  auto at_lds = [&](int g, int r, int chunk) __attribute__((always_inline)) {
    return sums + (g * kRows + r) * D + (chunk ^ (r & (D == 64 ? 15 : 31))) * 4;
  };
  if (kGroups > 1 || wave_row < rows) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4*>(at_lds(group, row_wave * 32 + lane % 32, dt * 8 + 2 * q4 + half)) =
            f32x4{o_acc[dt][q4 * 4] * own, o_acc[dt][q4 * 4 + 1] * own, o_acc[dt][q4 * 4 + 2] * own, o_acc[dt][q4 * 4 + 3] * own};
  }
  if constexpr (kGroups > 1) {
    if (half == 0) {
      m_lds[group][row_wave * 32 + lane] = m_i;
      l_lds[group][row_wave * 32 + lane] = l;
    }
    __syncthreads();
  } else {
    if (parts && live && half == 0) w.sums.ml[slot + (int64_t)token * a.heads + head] = float2{m_i, l};
    asm volatile("" ::: "memory");                                  // a wave's LDS accesses are in order
  }
  constexpr int kLanes = D / 8, kRowsAtOnce = kWave / kLanes, kWaveRows = kRows / (kRowWaves * kGroups);      // eight columns a lane
  const int d = lane % kLanes * 8;
#pragma unroll 2
  for (int r0 = 0; r0 < kWaveRows; r0 += kRowsAtOnce) {
    const int r = wave * kWaveRows + r0 + lane / kLanes, at = row0 + r;
    if (at >= rows || d >= dim) continue;
    const int i = divided(at, a.by_group), t = token0 + i, h = kvh * a.group + at - i * a.group;
    const int64_t to = slot + (int64_t)t * a.heads + h;
    float v[8];
    if constexpr (kGroups == 1) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(at_lds(0, r, d / 4)), hi = *reinterpret_cast<const f32x4*>(at_lds(0, r, d / 4 + 1));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = lo[e];
        v[e + 4] = hi[e];
      }
    } else {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) top = fmaxf(top, m_lds[g][r]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      const float base = top == -INFINITY ? 0.0f : top;             // no key: sums of 0; a NaN among the scores stays one
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const float f = __builtin_amdgcn_exp2f(m_lds[g][r] - base);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(at_lds(g, r, d / 4)), hi = *reinterpret_cast<const f32x4*>(at_lds(g, r, d / 4 + 1));
        sum = fmaf(l_lds[g][r], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = fmaf(lo[e], f, v[e]);
          v[e + 4] = fmaf(hi[e], f, v[e + 4]);
        }
      }
      if (parts && d == 0) w.sums.ml[to] = float2{top, sum};
      const float inv = parts ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= inv;
    }
    if (parts) {
      float* out = w.sums.o + to * dim + d;
      *reinterpret_cast<f32x4*>(out) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(out + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      *reinterpret_cast<Frag*>(static_cast<T*>(a.out) + t * a.out_token + h * a.out_head + d) = MfmaT<T>::pack(v);
    }
  }
}

}  // namespace
}  // namespace hexmi
