// Attention over a paged cache of keys and values (fp16 / bf16): runs of new tokens of many sequences over the positions before them, and
// the prefix that all sequences share.
//
// The query rows of a key head, (token, head of its group) one behind the other, are cut into tiles of kRows; a workgroup of four waves
// takes a tile, 32 rows a wave, and walks the keys up to its last token's own in blocks of 64, as flash_attn.hip does: S^T = K Q^T with
// v_mfma_f32_32x32x16, online softmax in registers, O^T += V^T P^T with V read transposed from LDS. What differs is where things stand:
// a block's 64 pages are looked up a block ahead, a lane each, a key's row is copied into LDS from wherever its page is, and a block
// carries a bit a key that says whether it is one. Heads that share their keys share a tile, so a step of decode in a batch with
// prompts reads its keys once too; a wave whose rows are none only copies.
//
// The prefix (SHARED mode) is one sequence that all rows of the batch attend: its keys go through LDS once for kRows rows, whatever sequences they
// are of. Its sums, and those of tiles whose keys are cut over several workgroups because there are few, go through the workspace.
#include "flash_attn_tiles.h"
#include "paged.h"

namespace hexmi {
namespace {

constexpr int kTileWaves = 4, kRows = kTileWaves * 32;

// One launch: the prefix for all rows (the first workgroups), and every sequence's keys behind it.
struct TileArgs {
  int shared_tiles, shared_splits;             // tiles of a key head; parts of the prefix, whose sums go to slots 0 .. (0: no prefix)
  int tiles, splits;                           // of the sequences' own keys, whose sums go to the slots behind (0: decode, not here)
  RowSums sums;                                // slots 0: the result goes to out
};

// The tiles of a key head: those of sequence b are numbered from first_tile(b) on, b = -1 .. sequences, where -1 and `sequences` are the
// rows of no sequence before the first and behind the last. floor(x / r) + 1 >= ceil(n / r) + floor(x0 / r) for x = x0 + n, so
// a sequence's tiles end before the next one's begin; some numbers are no tile.
__device__ __forceinline__ int first_row(const Pages& p, int b) {
  const int s = b < 0 ? 0 : b > p.sequences ? p.tokens : p.starts[b];
  return s < 0 ? 0 : s < p.tokens ? s : p.tokens;
}
__device__ __forceinline__ int first_tile(const Pages& p, int group, int b) { return b < 0 ? 0 : first_row(p, b) * group / kRows + b + 1; }
__device__ __forceinline__ int sequence_of_tile(const Pages& p, int group, int tile, int lane) {
  int lo = -1, hi = p.sequences + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const int n = __popcll(__ballot(at < hi && first_tile(p, group, at) <= tile));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
    if (step == 1) break;
  }
  return lo;
}

// keys that token i of a sequence's n sees, whatever the index tensors hold
__device__ __forceinline__ int keys_of(int64_t length, int n, int i, int most) {
  const int64_t keys = length - n + i + 1;
  return keys < 0 ? 0 : keys < most ? (int)keys : most;
}

// D: columns of a row in LDS; COLS <= D, a multiple of 32: columns that are multiplied; PADDED: a head is narrower than COLS. A lane whose
// columns lie past the head copies the head's first ones instead: the query has zeros there, and what comes of V there is not stored.
template <typename T, int D, int COLS, bool PADDED>
__global__ __launch_bounds__(kTileWaves * kWave, D == 256 ? 1 : 2)
void paged_tile_kernel(PagedAttnArgs a, Pages p, TileArgs w) {
  typedef typename MfmaT<T>::Frag Frag;
  constexpr int DS = COLS / 16, DT = COLS / 32, CPR = D / 8;
  constexpr int NI = kBlockN * CPR / kWave / kTileWaves, kRowStep = kTileWaves * kWave / CPR;
  __shared__ __attribute__((aligned(16))) T k_lds0[kBlockN * D];
  __shared__ __attribute__((aligned(16))) T k_lds1[kBlockN * D];
  __shared__ __attribute__((aligned(16))) T v_lds0[kBlockN * D];
  __shared__ __attribute__((aligned(16))) T v_lds1[kBlockN * D];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), half = lane / 32;
  const int dim = PADDED ? a.dim : COLS;

  // Workgroup -> (prefix or not, key head, tile, part). Workgroup ids go round robin to the 8 XCDs (one L2 each): every XCD gets a run of
  // the list, key head by key head, a sequence's last (longest) tiles first.
  const unsigned shared_grid = (unsigned)(w.shared_tiles * w.shared_splits * p.kv_heads);
  const bool shared = blockIdx.x < shared_grid;
  const int tiles = shared ? w.shared_tiles : w.tiles, splits = shared ? w.shared_splits : w.splits;
  const unsigned id = shared ? blockIdx.x : blockIdx.x - shared_grid, count = shared ? shared_grid : gridDim.x - shared_grid;
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
    const int b = __builtin_amdgcn_readfirstlane(sequence_of_tile(p, a.group, tile, lane));
    token0 = first_row(p, b);
    new_tokens = first_row(p, b + 1) - token0;
    row0 = (tile - first_tile(p, a.group, b)) * kRows;
    rows = new_tokens * a.group;                                    // negative where starts fall: nothing
    if (row0 < 0 || row0 >= rows) return;
    none = b < 0 || b >= p.sequences;
    if (!none) length = p.lengths[b];
    const int last = row0 + kRows < rows ? row0 + kRows - 1 : rows - 1;
    end = none ? 0 : keys_of(length, new_tokens, divided(last, a.by_group), most);
    begin = a.prefix;
    table = p.table + (none ? 0 : b) * p.table_row;
  }
  end = __builtin_amdgcn_readfirstlane(end);
  const int blocks = end > begin ? (end - begin + kBlockN - 1) / kBlockN : 0, share = (blocks + splits - 1) / splits;
  const int block0 = part * share, block1 = block0 + share < blocks ? block0 + share : blocks;

  // ---- copies: instruction j of a wave takes kRowStep / 4 rows, a lane 16 bytes of one
  const T* k_head = static_cast<const T*>(a.k) + kvh * p.k_head;
  const T* v_head = static_cast<const T*>(a.v) + kvh * p.v_head;
  const int lin = wave * kWave + lane, copy_row = lin / CPR, lds_at = wave * kWave * 8;
  auto find = [&](int block) __attribute__((always_inline)) {       // the page of key 64 block + lane, -1: none
    const int key = begin + block * kBlockN + lane;
    if (block >= block1 || key >= end) return -1;
    const int page = table[divided(key, p.size)];
    return page < p.num_pages ? page : -1;
  };
  auto copy = [&](int j, bool v, int block, int page_of_lane, T* lds) __attribute__((always_inline)) {
    const int r = copy_row + j * kRowStep, key = begin + block * kBlockN + r, page = __shfl(page_of_lane, r);
    int c = ((lin % CPR) ^ (v ? swz_vtile<D == 64 ? 64 : 128>(r) : swz_ktile<D == 64 ? 64 : 128>(r))) * 8;
    if (PADDED && c >= dim) c = 0;
    T* to = lds + lds_at + j * (kTileWaves * kWave * 8);
    if (page >= 0) {
      const int slot = key - divided(key, p.size) * p.page_size;
      const T* from = v ? v_head + page * p.v_page + slot * p.v_slot + c : k_head + page * p.k_page + slot * p.k_slot + c;
      __builtin_amdgcn_global_load_lds(HEXMI_GLB(from), HEXMI_LDS(to), 16, 0, 0);
    } else if (v) {                                                 // no key: whatever the cache holds, zeros of V (its score is dropped)
      *reinterpret_cast<u32x4*>(to + lane * 8) = u32x4{0u, 0u, 0u, 0u};
    }
  };
  int page = -1, next = -1;
  if (block0 < block1) {                                            // on their way while the rows are looked up
    page = find(block0);
    next = find(block0 + 1);
#pragma unroll
    for (int j = 0; j < NI; ++j) copy(j, false, block0, page, k_lds0);
#pragma unroll
    for (int j = 0; j < NI; ++j) copy(j, true, block0, page, v_lds0);
  }

  // this lane's row: its token, its queries and the keys it sees
  const int wave_row = row0 + wave * 32, row = wave_row + lane % 32;
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
    if (live && s >= 0) keys = keys_of(p.lengths[s], p.starts ? p.starts[s + 1] - token : 1, 0, most);
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
    const int key0 = begin + block * kBlockN;
    if (block + 1 < block1) {
#pragma unroll
      for (int j = 0; j < NI; ++j) copy(j, false, block + 1, next_page, k_dst);
#pragma unroll
      for (int j = 0; j < NI; ++j) copy(j, true, block + 1, next_page, v_dst);
    }
    if (key0 >= most_keys) return;                                  // wave-uniform; the barriers are outside
    f32x16 s[2];
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[jt][r] = 0.0f;
    {
      constexpr int kAhead = 3;
      auto read_k = [&](int jt, int ds) __attribute__((always_inline)) {
        const int r = jt * 32 + lane % 32, c = (ds * 2 + half) ^ swz_ktile<D == 64 ? 64 : 128>(r);
        return *reinterpret_cast<const Frag*>(k_src + (r * CPR + c) * 8);
      };
      Frag kf[2][DS];
#pragma unroll
      for (int ds = 0; ds < kAhead && ds < DS; ++ds) {
        kf[0][ds] = read_k(0, ds);
        kf[1][ds] = read_k(1, ds);
      }
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        if (ds + kAhead < DS) {
          kf[0][ds + kAhead] = read_k(0, ds + kAhead);
          kf[1][ds + kAhead] = read_k(1, ds + kAhead);
        }
        s[0] = MfmaT<T>::run(kf[0][ds], qf[ds], s[0]);
        s[1] = MfmaT<T>::run(kf[1][ds], qf[ds], s[1]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    struct VFrags { Frag f[2][DT]; };
    auto read_v = [&](int jt, VFrags& vf) __attribute__((always_inline)) {
      const int g = lane / 16, i16 = lane % 16;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          union { i16x4 h[2]; Frag f; } u;
#pragma unroll
          for (int pp = 0; pp < 2; ++pp) {
            const int r = jt * 32 + hf * 16 + 8 * pp + 4 * (g >> 1) + (i16 >> 2), col = dt * 32 + (g & 1) * 16 + (i16 & 3) * 4;
            const int c = (col / 8) ^ swz_vtile<D == 64 ? 64 : 128>(r);
            u.h[pp] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(v_src + (r * CPR + c) * 8 + col % 8));
          }
          vf.f[hf][dt] = u.f;
        }
    };
    VFrags vf0, vf1;
    read_v(0, vf0);
    __builtin_amdgcn_sched_barrier(0);
    // s[jt][r] is the score of key key0 + 32 jt + 8 (r / 4) + 4 half + r % 4
    if (there != ~0ull || key0 + kBlockN > least_keys) {
      const uint32_t bits[2] = {(uint32_t)there >> (4 * half), (uint32_t)(there >> 32) >> (4 * half)};
#pragma unroll
      for (int jt = 0; jt < 2; ++jt)
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
    for (int r = 0; r < 16; ++r) mx1 = fmaxf(mx1, s[1][r]);
    mx = fmaxf(mx, mx1);
    mx = fmaxf(mx, other_half(mx)) * a.scale;
    const bool grow = mx > m_i + kRescaleLag;                       // the reference maximum may lag (flash_attn.hip)
    if (__ballot(grow) != 0) {
      const float m_new = grow ? mx : m_i, alpha = grow ? __builtin_amdgcn_exp2f(m_i - m_new) : 1.0f;
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
      pf[0] = MfmaT<T>::pack(&pr[0]);
      pf[1] = MfmaT<T>::pack(&pr[8]);
      l_i = MfmaT<T>::sum8(pf[1], MfmaT<T>::sum8(pf[0], l_i));      // the sum of what the product multiplies
    };
    auto pv = [&](const VFrags& vf) __attribute__((always_inline)) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o_acc[dt] = MfmaT<T>::run(vf.f[hf][dt], pf[hf], o_acc[dt]);
    };
    read_v(1, vf1);
    exp_tile(s[0]);
    pv(vf0);
    exp_tile(s[1]);
    pv(vf1);
  };

  for (int block = block0; block < block1; block += 2) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint64_t there = __ballot(page >= 0);
    page = next;
    next = find(block + 2);
    process(block, there, page, k_lds0, v_lds0, k_lds1, v_lds1);
    if (block + 1 >= block1) break;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    there = __ballot(page >= 0);
    page = next;
    next = find(block + 3);
    process(block + 1, there, page, k_lds1, v_lds1, k_lds0, v_lds0);
  }

  // ---- o_acc[dt][r] is column 32 dt + 8 (r / 4) + 4 half + r % 4 of the row's sum
  const float l = l_i + other_half(l_i);
  if (!live) return;
  if (w.sums.slots) {
    const int64_t at = (int64_t)(part + (shared ? 0 : w.shared_splits)) * w.sums.rows + (int64_t)token * a.heads + head;
    if (half == 0) w.sums.ml[at] = float2{m_i, l};
    if (!(l > 0.0f)) return;
    float* out = w.sums.o + at * dim;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d = dt * 32 + 8 * q4 + 4 * half;
        if (!PADDED || d < dim) store4<float>(out + d, o_acc[dt][q4 * 4], o_acc[dt][q4 * 4 + 1], o_acc[dt][q4 * 4 + 2], o_acc[dt][q4 * 4 + 3]);
      }
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d = dt * 32 + 8 * q4 + 4 * half;
      if (!PADDED || d < dim)
        store4o<T>(out + d, o_acc[dt][q4 * 4] * inv, o_acc[dt][q4 * 4 + 1] * inv, o_acc[dt][q4 * 4 + 2] * inv, o_acc[dt][q4 * 4 + 3] * inv);
    }
}

// A row's sums of all slots (at most 32) joined: 32 threads a row, a thread the columns d and, past 128, d + 128.
template <typename T>
__global__ __launch_bounds__(256)
void paged_join_kernel(PagedAttnArgs a, RowSums sums) {
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= sums.rows) return;
  const int d = threadIdx.x % 32 * 4;
  // lane x of the 32 has slot x's maximum and sum, and all four slots' columns are asked for at once
  constexpr int kSlots = 4;
  const int lane = threadIdx.x % kWave, own = lane % 32;
  const float2 ml = own < sums.slots ? sums.ml[own * sums.rows + row] : float2{-INFINITY, 0.0f};
  float top = ml.y > 0.0f ? ml.x : -INFINITY;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  const float f = ml.y > 0.0f ? __builtin_amdgcn_exp2f(ml.x - top) : 0.0f;
  float sum = ml.y * f;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) sum += __shfl_xor(sum, x);
  f32x4 out[2] = {};
  for (int x0 = 0; x0 < sums.slots; x0 += kSlots) {
    f32x4 o[kSlots][2];
    float fx[kSlots];
#pragma unroll
    for (int x = 0; x < kSlots; ++x) {
      fx[x] = __shfl(f, (lane & 32) + x0 + x);                      // 0: nothing there, and its columns are not read
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[x][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (fx[x] > 0.0f && d + h * 128 < a.dim)
          o[x][h] = *reinterpret_cast<const f32x4*>(sums.o + ((x0 + x) * sums.rows + row) * a.dim + d + h * 128);
      }
    }
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[h][e] = fmaf(o[x][h][e], fx[x], out[h][e]);
  }
  const int token = (int)(row / a.heads), head = (int)(row - (int64_t)token * a.heads);
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  T* to = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (d + h * 128 < a.dim) store4o<T>(to + d + h * 128, out[h][0] * inv, out[h][1] * inv, out[h][2] * inv, out[h][3] * inv);
}

template <typename T>
int launch_tiles(const PagedAttnArgs& a, const Pages& p, const TileArgs& w, hipStream_t s) {
  const unsigned grid = (unsigned)(((int64_t)w.tiles * w.splits + (int64_t)w.shared_tiles * w.shared_splits) * p.kv_heads);
#define HEXMI_PAGED_TILE(D, COLS)                                                                                                         \
  do {                                                                                                                                    \
    if (a.dim == COLS) hipLaunchKernelGGL((paged_tile_kernel<T, D, COLS, false>), dim3(grid), dim3(kTileWaves * kWave), 0, s, a, p, w);   \
    else hipLaunchKernelGGL((paged_tile_kernel<T, D, COLS, true>), dim3(grid), dim3(kTileWaves * kWave), 0, s, a, p, w);                  \
  } while (0)
  if (a.dim <= 64) HEXMI_PAGED_TILE(64, 64);
  else if (a.dim <= 96) HEXMI_PAGED_TILE(128, 96);
  else if (a.dim <= 128) HEXMI_PAGED_TILE(128, 128);
  else HEXMI_PAGED_TILE(256, 256);
#undef HEXMI_PAGED_TILE
  return launch_status();
}

// What a call launches: the prefix's tiles (prefix_splits 0: none), then one token a sequence (decode) or tiles of the sequences' own keys
// (splits), then the join of the tiles' sums.
struct Plan {
  bool decode;
  int prefix_tiles, prefix_splits, splits;
  int64_t tiles;
  PagedDecodePlan one;
  int64_t rows, sum_bytes, decode_bytes;
  int slots() const { return prefix_splits == 0 && (decode || splits == 1) ? 0 : prefix_splits + (decode ? 1 : splits); }
};
// Parts of the keys for tiles of which there are `units`: two workgroups a compute unit, no part below four blocks. A row has 32 slots for
// the sums of its parts, of the prefix and its own together.
int parts_of(int64_t units, int64_t keys) {
  const int64_t blocks = (keys + kBlockN - 1) / kBlockN, wanted = 2 * (int64_t)hexmi_num_cus() / units;
  const int64_t most = blocks / 4 < 16 ? blocks / 4 : 16;
  return (int)(wanted < most ? (wanted > 1 ? wanted : 1) : (most > 1 ? most : 1));
}
Plan plan_of(const hexmi_paged_batch& b, int64_t heads, int64_t shared) {
  Plan plan = {};
  const int64_t group = heads / b.kv_heads, prefix = shared * b.page_size, rows = b.tokens * group;
  const int64_t own = b.table_cols * b.page_size - prefix, full = (rows + kRows - 1) / kRows;
  plan.decode = b.starts == nullptr;
  plan.rows = b.tokens * heads;
  if (shared > 0) {
    plan.prefix_tiles = (int)full;
    plan.prefix_splits = parts_of(full * b.kv_heads, prefix);
  }
  if (plan.decode) {
    plan.one = plan_paged_decode(b, heads, prefix);
    plan.decode_bytes = (paged_decode_workspace(plan.one, b.dim) + 15) / 16 * 16;
  } else {
    plan.tiles = rows / kRows + b.sequences + 2;
    plan.splits = parts_of(full * b.kv_heads, own);
  }
  plan.sum_bytes = plan.slots() * plan.rows * (b.dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
  return plan;
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

namespace {
int check(const hexmi_paged_batch& b, int64_t heads, int64_t shared) {
  const int rc = check_batch(b);
  if (rc != HEXMI_OK) return rc;
  if (heads < 1 || heads % b.kv_heads != 0 || shared < 0 || shared > b.table_cols) return HEXMI_EINVAL;
  if (b.dim % 8 != 0 || b.dim > 256 || heads > 65535) return HEXMI_ENOTSUP;
  // rows, the blocks of all sequences and heads, and a launch's threads stay below 2^31
  const int64_t group = heads / b.kv_heads, limit = 0x7fffffff, units = b.kv_heads * ((group + 15) / 16);
  const int64_t blocks = (b.table_cols * b.page_size + 127) / 128 + 1;
  if (b.tokens > limit / heads || b.sequences > limit / units / blocks) return HEXMI_ENOTSUP;
  if (!b.starts) return b.sequences <= limit / 256 / units ? HEXMI_OK : HEXMI_ENOTSUP;
  const Plan plan = plan_of(b, heads, shared);
  return (plan.tiles * plan.splits + (int64_t)plan.prefix_tiles * plan.prefix_splits) * b.kv_heads <= limit / (kTileWaves * kWave) ? HEXMI_OK : HEXMI_ENOTSUP;
}
}  // namespace

extern "C" int64_t hexmi_paged_attention_workspace(const hexmi_paged_batch* batch, int64_t heads, int64_t shared) {
  if (!batch || check(*batch, heads, shared) != HEXMI_OK || batch->tokens == 0) return 0;
  const Plan plan = plan_of(*batch, heads, shared);
  return plan.decode_bytes + plan.sum_bytes;
}

extern "C" int hexmi_paged_attention(const hexmi_head_rows* q, const hexmi_paged_batch* batch, const int32_t* shared_pages, int64_t shared,
                                     float sm_scale, int dtype, void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  if (!q || !batch || (shared > 0 && !shared_pages) || workspace_bytes < 0) return HEXMI_EINVAL;
  int rc = check(*batch, q->heads, shared);
  if (rc != HEXMI_OK) return rc;
  if (!(sm_scale > 0.0f) || sm_scale > 2e38f) return HEXMI_EINVAL;
  if (dtype != HEXMI_F16 && dtype != HEXMI_BF16) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (!q->x || !q->out || !batch->k_pages || !batch->v_pages ||
      (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))))
    return HEXMI_EINVAL;
  const int64_t strides[] = {q->token, q->head, q->out_token, q->out_head, batch->k_page, batch->k_head, batch->k_slot, batch->v_page,
                             batch->v_head, batch->v_slot};
  for (int64_t s : strides)
    if (s % 8 != 0) return HEXMI_ENOTSUP;
  if (!aligned_to(q->x, 16) || !aligned_to(q->out, 16) || !aligned_to(batch->k_pages, 16) || !aligned_to(batch->v_pages, 16)) return HEXMI_ENOTSUP;
  const Plan plan = plan_of(*batch, q->heads, shared);
  const int64_t need = plan.decode_bytes + plan.sum_bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return HEXMI_EINVAL;
  const int64_t group = q->heads / batch->kv_heads;
  const PagedAttnArgs a = {q->x, batch->k_pages, batch->v_pages, q->out, q->token, q->head, q->out_token, q->out_head, shared_pages,
                           (int)(shared * batch->page_size), (int)q->heads, (int)group, (int)batch->dim, sm_scale * kLog2e, divider(group)};
  const Pages p = pages_of(*batch);
  float* o = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.decode_bytes);
  const RowSums sums = {o, reinterpret_cast<float2*>(o + plan.slots() * plan.rows * batch->dim), plan.rows, plan.slots()};
  hipStream_t s = as_stream(stream);
  begin_call();
  auto tiles = [&](const TileArgs& w) { return dtype == HEXMI_F16 ? launch_tiles<f16>(a, p, w, s) : launch_tiles<bf16>(a, p, w, s); };
  if (plan.decode) {
    if (plan.prefix_splits > 0 && (rc = tiles({plan.prefix_tiles, plan.prefix_splits, 0, 0, sums})) != HEXMI_OK) return rc;
    return paged_decode(plan.one, a, p, dtype, workspace, sums, s);
  }
  if ((rc = tiles({plan.prefix_tiles, plan.prefix_splits, (int)plan.tiles, plan.splits, sums})) != HEXMI_OK || sums.slots == 0) return rc;
  const unsigned blocks = (unsigned)((plan.rows + 7) / 8);
  if (dtype == HEXMI_F16) hipLaunchKernelGGL((paged_join_kernel<f16>), dim3(blocks), dim3(256), 0, s, a, sums);
  else hipLaunchKernelGGL((paged_join_kernel<bf16>), dim3(blocks), dim3(256), 0, s, a, sums);
  return launch_status();
}
