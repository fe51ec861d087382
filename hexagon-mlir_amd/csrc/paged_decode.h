// A worker of a decode step over the pages of a cache (paged_decode.hip, paged_shared.hip).
//
// Bound by HBM: every key and value of a sequence is read once, for all the query heads that share its key head. Those heads (up to 16)
// are the columns of v_mfma_f32_16x16x32: a wave takes 32 keys at a time,
//   S^T = K Q^T    a lane's A operand is 16 bytes of a key's row, straight from its page to registers; a lane then holds 8 scores of one head
//   O^T += V^T P^T the probabilities go from the score registers to the B operand as they are (which key stands in which slot of the
//                  product is free: slot 8 g + 4 t + i is key 16 t + 4 g + i); V passes through a wave's own LDS and is read transposed
//                  (ds_read_b64_tr_b16).
// Keys and values of the next 32 are asked for as soon as the registers of these are free, so a wave has 16 KiB (heads of 128) on the way
// at nearly all times, eight waves a compute unit: 16 sequences x 2048 keys x 32 heads of 128 97 us, 5.5 TB/s (a copy reaches 5.1, read and
// written), 64 of 100 to 16384 over 8 heads 177. Two tiles ahead, twelve waves a compute unit, and rows of keys fetched whole through LDS
// changed nothing there.
//
// The work is cut evenly whatever the lengths are: the blocks of keys of all sequences and key heads, one behind the other,
// are dealt to the workers (workgroups) in equal runs. A worker that has all of a unit (sequence, key head, 16 query heads) writes
// its rows; of a unit that several share every worker leaves its sums, at most two sets, which a second launch joins in the order of
// the keys. Nothing is added atomically.
#pragma once
#include "flash_attn_tiles.h"
#include "paged.h"

namespace hexmi {
namespace {

constexpr int kWaves = 4;                      // of a workgroup that only decodes
constexpr int kTileKeys = 32;                  // of a wave; a workgroup's W waves take a block of W * kTileKeys
constexpr int kBlockKeys = kWaves * kTileKeys;

template <typename T> struct Mfma16;
template <> struct Mfma16<f16> {
  static __device__ __forceinline__ f32x4 run(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma16<bf16> {
  static __device__ __forceinline__ f32x4 run(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ float max_of_quarters(float v) {        // over the lanes of one head: lane % 16
  float a, b;
  swap16(v, a, b);
  v = fmaxf(a, b);
  swap32(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_of_quarters(float v) {
  float a, b;
  swap16(v, a, b);
  v = a + b;
  swap32(v, a, b);
  return a + b;
}

// blocks of a sequence's unit: one at least, so that a row without keys is written too
template <int W> __device__ __forceinline__ int blocks_of_keys(int keys) {
  return keys > W * kTileKeys ? (keys + W * kTileKeys - 1) / (W * kTileKeys) : 1;
}
// of sequence b, none where it has other than one new token (the tiles take those)
// View: the most keys that its token sees, and the blocks that a unit counts for beside its own when the work is dealt: to begin one costs
// a worker about the time of a block in 8 bits. None / 1 / 2, us: 64 sequences of 100 to 16384 over 8 heads 99.1 / 93.5 / 95.5, 128 of 50 to 2000
// 53.4 / 45.6 / 46.5, 8 of 100 to 4000 14.0 / 13.7 / 13.5, heads of 80 45.0 / 43.5 / 46.6; the other way round heads of 64 78.6 / 80.8 / 80.8 and
// lengths that are all the same, 32 x 1000 19.9 / 21.0 / 21.6 (16 x 2048 x 32 heads 65.5 / 65.3 / 65.5).
struct Dealt {
  int view, extra;
};
constexpr int kExtraBlocks = 1;                // of a cache in 8 bits; in 16, none
__device__ __forceinline__ int at_most(int n, int most) { return n < most ? n : most; }
template <int W> __device__ __forceinline__ int dealt_blocks(int length, int prefix, const Dealt& d) {
  return blocks_of_keys<W>(at_most(length, d.view) - prefix) + d.extra;
}
template <int W> __device__ __forceinline__ int blocks_of(const Pages& p, int b, int prefix, const Dealt& d) {
  return new_tokens_of(p, b) == 1 ? dealt_blocks<W>(length_of(p, b), prefix, d) : 0;
}
// the sum over the lanes up to this one
__device__ __forceinline__ int sum_up_to(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);     // row_shr:1, 2, 4, 8: within 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);    // row_bcast:15 into the second and fourth 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);    // row_bcast:31 into the upper 32
  return v;
}
__device__ __forceinline__ int of_last_lane(int v) { return __builtin_amdgcn_readlane(v, kWave - 1); }

// The list of all blocks, sequence by sequence: lengths, blocks and sums of blocks of the first 64 sequences are a lane's each, read once;
// those of further ones are read again where they are needed.
struct BlockList {
  int length, blocks, up_to;                   // lane b: of sequence b (no blocks: not a worker's), and of all up to it
  int of_64, all;                              // blocks of the first 64 sequences, of all (one unit's)
};
template <int W>
__device__ __forceinline__ BlockList block_list(const Pages& p, int prefix, const Dealt& d, int lane) {
  BlockList l;
  l.length = lane < p.sequences ? length_of(p, lane) : 0;
  l.blocks = lane < p.sequences && new_tokens_of(p, lane) == 1 ? dealt_blocks<W>(l.length, prefix, d) : 0;
  l.up_to = sum_up_to(l.blocks);
  l.of_64 = of_last_lane(l.up_to);
  int more = 0;
  for (int b0 = kWave; b0 < p.sequences; b0 += kWave) more += b0 + lane < p.sequences ? blocks_of<W>(p, b0 + lane, prefix, d) : 0;
  l.all = l.of_64 + (p.sequences > kWave ? of_last_lane(sum_up_to(more)) : 0);
  return l;
}
// The sequence that block `at` of the list belongs to, with `units` units a sequence, and the blocks (of one unit) before it.
template <int W>
__device__ __forceinline__ int sequence_at(const BlockList& l, const Pages& p, int prefix, const Dealt& d, int units, int at, int lane, int& before) {
  before = 0;
  for (int b0 = 0;; b0 += kWave) {
    const int n = b0 == 0 ? l.blocks : b0 + lane < p.sequences ? blocks_of<W>(p, b0 + lane, prefix, d) : 0, sum = b0 == 0 ? l.up_to : sum_up_to(n);
    const uint64_t past = __ballot((before + sum) * units > at);
    if (past || b0 + kWave >= p.sequences) {   // `at` is below the end: there is one
      const int first = past ? __ffsll((unsigned long long)past) - 1 : 0;
      before += __builtin_amdgcn_readlane(sum - n, first);
      return b0 + first;
    }
    before += of_last_lane(sum);
  }
}
__device__ __forceinline__ int length_at(const BlockList& l, const Pages& p, int b) {
  return __builtin_amdgcn_readfirstlane(b < kWave ? __builtin_amdgcn_readlane(l.length, b & (kWave - 1)) : length_of(p, b));
}
template <int W> __device__ __forceinline__ int blocks_at(const BlockList& l, const Pages& p, int prefix, const Dealt& d, int b) {
  return __builtin_amdgcn_readfirstlane(b < kWave ? __builtin_amdgcn_readlane(l.blocks, b & (kWave - 1)) : blocks_of<W>(p, b, prefix, d));
}
// worker w's run of `total` blocks
__device__ __forceinline__ int run_start(int total, int workers, int w) {
  const int each = total / workers, more = total % workers;
  return w * each + (w < more ? w : more);
}
__device__ __forceinline__ int worker_of(int total, int workers, int at) {
  const int each = total / workers, more = total % workers, long_end = more * (each + 1);
  return at < long_end ? at / (each + 1) : more + (at - long_end) / each;
}

// the 16-byte chunks of a V row in LDS are XOR swizzled in pairs, so that 8 rows at one pair of chunks (a transposing read takes 16 rows x
// 32 bytes) stand on all banks once
template <int D> __device__ __forceinline__ int swz_pairs(int row) { return D == 64 ? ((row >> 1) & 3) << 1 : (row & 7) << 1; }

// LDS of a wave: 32 rows of V, later 16 rows of sums; a whole number of rows of V
constexpr int decode_wave_bytes(int d, int cols) {
  const int sums = (16 * (cols + 4) * 4 + d * 2 - 1) / (d * 2) * (d * 2), tile = kTileKeys * d * 2;
  return tile > sums ? tile : sums;
}

// A row's four columns from d on into the slot for sequences' own keys; of the slots behind it, which only tiles fill, that they are empty.
__device__ __forceinline__ void keep_sums(const DecodeArgs& w, int64_t row, int dim, int d, const f32x4& out, float2 ml) {
  const int64_t at = w.own * w.sums.rows + row;
  *reinterpret_cast<f32x4*>(w.sums.o + at * dim + d) = out;
  if (d != 0) return;
  w.sums.ml[at] = ml;
  for (int x = w.own + 1; x < w.sums.slots; ++x) w.sums.ml[x * w.sums.rows + row] = float2{-INFINITY, 0.0f};
}

// D, COLS, PADDED: HeadWidth. A lane whose columns lie past the head reads the head's first ones instead: the query has zeros there, and what
// comes of V there is not stored.
// worker: of w.workers, or the unit where that is 0.
// The keys that a token sees within a window are its sinks and the last of its sequence, gone through as if they stood side by side.
// A scaled cache: keys and values are widened to T (exact, see kLeastExponent) on the way from their registers to the matrix cores and to LDS.
// A lane's 16 bytes are 16 columns of a row, so where a head is whole 64s the columns go to the products in another order, the query's too.
template <typename T, typename Kind, int D, int COLS, bool PADDED, int W>
__device__ __forceinline__ void paged_decode_worker(const PagedAttnArgs& a, const Pages& p, const DecodeArgs& w, unsigned worker, char* lds,
                                                    float (*m_lds)[16], float (*l_lds)[16]) {
  typedef typename MfmaT<T>::Frag Frag;
  constexpr int DS = COLS / 32, DT = COLS / 16, kPitch = COLS + 4;
  constexpr bool kWide = Kind::kScaled && COLS % 64 == 0 && !PADDED;
  constexpr int LS = kWide ? DS / 2 : DS;                           // loads of a row
  typedef std::conditional_t<Kind::kScaled && !kWide, u32x2, u32x4> Raw;
  typedef std::conditional_t<Kind::kScaled, uint8_t, T> Held;
  const Dealt dealt = {Kind::kWindow ? a.view : kNoWindow, Kind::kScaled ? kExtraBlocks : 0};
  constexpr int kWaveBytes = decode_wave_bytes(D, COLS), kBlock = W * kTileKeys;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane / 16, n = lane % 16;
  const int dim = PADDED ? a.dim : COLS;
  // This lane's bytes of V in LDS, rows of D columns in 16-byte chunks: chunk g of row n, where it puts, and columns 4 (n % 4) .. of row
  // 4 g + n / 4, from where it takes (ds_read_b64_tr_b16: a group of 16 lanes asks for 4 rows x 16 columns, and a lane gets a column).
  // Other chunks are these with the chunk's number XORed in.
  const int put_at = wave * kWaveBytes + n * (D * 2) + ((kWide ? 2 * g : g) ^ swz_pairs<D>(n)) * 16;
  const int take_row = 4 * g + (n >> 2), take_at = wave * kWaveBytes + take_row * (D * 2) + (((n & 3) >> 1) ^ swz_pairs<D>(take_row)) * 16 + (n & 1) * 8;
  float* o_lds = reinterpret_cast<float*>(lds + wave * kWaveBytes);
  const int units = p.kv_heads * w.row_tiles;

  BlockList list;
  int cur, end, b, before = 0, total = 0;
  int unit = 0;
  if (w.workers == 0) {                        // a unit each
    b = worker / units;
    unit = worker - b * units;
    list.length = 0;
    cur = 0;
    end = __builtin_amdgcn_readfirstlane(blocks_of<W>(p, b, a.prefix, dealt));
  } else {
    list = block_list<W>(p, a.prefix, dealt, lane);
    total = list.all * units;
    cur = run_start(total, w.workers, worker);
    end = run_start(total, w.workers, worker + 1);
    if (wave == 0 && lane == 0) w.begun[worker].last = -1;
    if (cur >= end) return;
    b = sequence_at<W>(list, p, a.prefix, dealt, units, cur, lane, before);
  }
  const int start = cur;

  while (cur < end) {
    const int whole_length = w.workers ? length_at(list, p, b) : __builtin_amdgcn_readfirstlane(length_of(p, b));
    const int length = at_most(whole_length, dealt.view), skip = whole_length - length;      // keys that are seen; those between the sinks and the others
    const int blocks = w.workers ? blocks_at<W>(list, p, a.prefix, dealt, b) : end - cur, local = cur - before * units;
    if (local >= blocks * units) {             // on to the next sequence
      before += blocks;
      ++b;
      continue;
    }
    const int in_list = local / blocks, u = w.workers ? in_list : unit, block0 = local - in_list * blocks;
    const int count = end - cur < blocks - block0 ? end - cur : blocks - block0;
    const int kvh = u / w.row_tiles, row0 = (u - kvh * w.row_tiles) * 16;
    const int rows = a.group - row0 < 16 ? a.group - row0 : 16;
    const int head0 = kvh * a.group + row0;
    const int token = __builtin_amdgcn_readfirstlane(first_row(p, b));

    // ---- queries: the B operand, head n's columns 32 ds + 8 g ..
    Frag qf[DS];
    int col[DS];
    {
      const T* q = static_cast<const T*>(a.q) + token * a.q_token + (head0 + (n < rows ? n : rows - 1)) * a.q_head;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const int c = kWide ? ds / 2 * 64 + g * 16 + ds % 2 * 8 : ds * 32 + g * 8;
        const bool live = !PADDED || c < dim;
        col[ds] = live ? c : 0;
        qf[ds] = *reinterpret_cast<const Frag*>(q + col[ds]);
        if (!live) qf[ds] = Frag{};
      }
    }
    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, neg_m = 0.0f, l = 0.0f;

    // ---- keys: this wave's tiles of the run
    auto own_block = [&](int block) __attribute__((always_inline)) { return block > dealt.extra ? block - dealt.extra : 0; };
    const int key_first = a.prefix + (own_block(block0) * W + wave) * kTileKeys;
    int key_end = a.prefix + own_block(block0 + count) * kBlock;
    key_end = key_end < length ? key_end : length;
    const int32_t* table = p.table + b * p.table_row;
    const Held* k_head = static_cast<const Held*>(a.k) + kvh * p.k_head;
    const Held* v_head = static_cast<const Held*>(a.v) + kvh * p.v_head;
    // where keys key0 + n and key0 + 16 + n stand; past the end: the last key again, without weight
    struct Keys { int page[2]; };
    auto clamped = [&](int key) __attribute__((always_inline)) {
      const int c = key < key_end ? key : key_end - 1;
      return Kind::kWindow ? c + (c >= a.sinks ? skip : 0) : c;
    };
    auto find = [&](int key0) __attribute__((always_inline)) {
      Keys k;
#pragma unroll
      for (int t = 0; t < 2; ++t) k.page[t] = table[divided(clamped(key0 + t * 16 + n), p.size)];
      return k;
    };
    auto there = [&](int page) __attribute__((always_inline)) { return page >= 0 && page < p.num_pages; };
    // strides of a scaled cache are below 2^32
    auto place = [&](int page, int64_t page_stride, int at, int64_t stride) __attribute__((always_inline)) {
      if constexpr (Kind::kScaled) return (int64_t)((uint64_t)(uint32_t)page * (uint32_t)page_stride + (uint64_t)(uint32_t)at * (uint32_t)stride);
      else return page * page_stride + at * stride;
    };
    auto load = [&](const Keys& at, int key0, const Held* base, int64_t page_stride, int64_t slot_stride, Raw (*r)[LS]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = clamped(key0 + t * 16 + n), slot = key - divided(key, p.size) * p.page_size;
        const Held* row = base + place(there(at.page[t]) ? at.page[t] : 0, page_stride, slot, slot_stride);
#pragma unroll
        for (int i = 0; i < LS; ++i) r[t][i] = *reinterpret_cast<const Raw*>(row + col[kWide ? 2 * i : i]);
      }
    };
    // Scales: a lane asks for one of its row's four, g % 2 the row (n, 16 + n), g / 2 keys' or values'; the swaps give all to all.
    const uint8_t* scale_head = nullptr;
    int64_t scale_page = 0, scale_block = 0;
    if constexpr (Kind::kScaled) {
      const Scales& sc = a.scales;
      scale_head = g < 2 ? sc.k + kvh * sc.k_head : sc.v + kvh * sc.v_head;
      scale_page = g < 2 ? sc.k_page : sc.v_page;
      scale_block = g < 2 ? sc.k_block : sc.v_block;
    }
    auto load_scale = [&](const Keys& at, int key0) __attribute__((always_inline)) {
      const int key = clamped(key0 + (g & 1) * 16 + n), slot = key - divided(key, p.size) * p.page_size;
      auto pick = [](bool second, int v0, int v1) { return second ? v1 : v0; };      // (values, not places: no scratch)
      const int page = pick(g & 1, at.page[0], at.page[1]);
      return (uint32_t)scale_head[place(there(page) ? page : 0, scale_page, divided(slot, a.scales.by_block), scale_block)];
    };
    if (key_first < key_end) {
      Raw kr[2][LS], vr[2][LS];
      Keys now = find(key_first), next = find(key_first + kBlock);
      uint32_t own_scale = 0;
      if constexpr (Kind::kScaled) own_scale = load_scale(now, key_first);
      load(now, key_first, k_head, p.k_page, p.k_slot, kr);
      load(now, key_first, v_head, p.v_page, p.v_slot, vr);
      for (int key0 = key_first; key0 < key_end; key0 += kBlock) {
        __builtin_amdgcn_sched_barrier(0);
        // what the constants of a chunk are XORed into; kept from becoming a register each
        int to = put_at, from = take_at;
        asm volatile("" : "+v"(to), "+v"(from));
        float k_scale0 = 1.0f, k_scale1 = 1.0f, v_scale0 = 1.0f, v_scale1 = 1.0f;
        if constexpr (Kind::kScaled) {
          float first, second;
          swap16(__builtin_bit_cast(float, own_scale << 23), first, second);
          swap32(first, k_scale0, v_scale0);
          swap32(second, k_scale1, v_scale1);
        }
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < LS; ++i)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if constexpr (Kind::kScaled) {
#pragma unroll
              for (int h = 0; h < (kWide ? 2 : 1); ++h)
                s[t] = Mfma16<T>::run(widened<T>(kr[t][i][2 * h], kr[t][i][2 * h + 1], t ? k_scale1 : k_scale0), qf[kWide ? 2 * i + h : i], s[t]);
            } else {
              s[t] = Mfma16<T>::run(__builtin_bit_cast(Frag, kr[t][i]), qf[i], s[t]);
            }
          }
        const bool ok0 = there(now.page[0]) && key0 + n < key_end, ok1 = there(now.page[1]) && key0 + 16 + n < key_end;
        const bool whole = __ballot(ok0 && ok1) == ~0ull;
        __builtin_amdgcn_sched_barrier(0);
        load(next, key0 + kBlock, k_head, p.k_page, p.k_slot, kr);
        if constexpr (Kind::kScaled) own_scale = load_scale(next, key0 + kBlock);
        __builtin_amdgcn_sched_barrier(0);
        if (!whole) {                                                // what stands where no key is may be anything: no weight, and zeros of V
          const uint32_t k0 = (uint32_t)__ballot(ok0), k1 = (uint32_t)__ballot(ok1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!(k0 >> (4 * g + i) & 1)) s[0][i] = -INFINITY;
            if (!(k1 >> (4 * g + i) & 1)) s[1][i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < LS; ++i) {
            if (!ok0) vr[0][i] = Raw{};
            if (!ok1) vr[1][i] = Raw{};
          }
          if (!ok0) v_scale0 = 1.0f;                                 // (a scale may be a NaN's)
          if (!ok1) v_scale1 = 1.0f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < LS; ++i) {
            if constexpr (Kind::kScaled) {
#pragma unroll
              for (int h = 0; h < (kWide ? 2 : 1); ++h)
                *reinterpret_cast<Frag*>(lds + (to ^ (kWide ? i * 128 + h * 16 : i * 64)) + t * (16 * D * 2)) =
                    widened<T>(vr[t][i][2 * h], vr[t][i][2 * h + 1], t ? v_scale1 : v_scale0);
            } else {
              *reinterpret_cast<u32x4*>(lds + (to ^ (i * 64)) + t * (16 * D * 2)) = vr[t][i];
            }
          }
        __builtin_amdgcn_sched_barrier(0);
        load(next, key0 + kBlock, v_head, p.v_page, p.v_slot, vr);
        __builtin_amdgcn_sched_barrier(0);
        // online softmax, the reference up to kRescaleLag further behind the true maximum than it was set (flash_attn.hip)
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_of_quarters(mx) * a.scale;
        const bool grow = mx > m + (kLift<T> + kRescaleLag);
        if (__ballot(grow) != 0) {
          const float m_new = grow ? mx - kLift<T> : m, alpha = grow ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
          l *= alpha;
          m = m_new;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[dt][i] *= alpha;
          neg_m = m == -INFINITY ? 0.0f : -m;
        }
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) pr[i] = __builtin_amdgcn_exp2f(fmaf(s[i / 4][i % 4], a.scale, neg_m));
        const Frag pf = MfmaT<T>::pack(pr);                          // 16 bits: paged_tile.h
        l += MfmaT<T>::sum8(pf, 0.0f);                               // the sum of what the product multiplies (these keys' first, paged_tile.h)
        asm volatile("" ::: "memory");                               // the reads below stay behind the writes above (LDS is in order)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          union { i16x4 h[2]; Frag f; } v;
#pragma unroll
          for (int t = 0; t < 2; ++t)
            v.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(lds + (from ^ (dt * 32)) + t * (16 * D * 2)));
          o[dt] = Mfma16<T>::run(v.f, pf, o[dt]);
          if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);      // no more than four pieces of V in registers
        }
        asm volatile("" ::: "memory");
        now = next;
        next = find(key0 + 2 * kBlock);
      }
    }

    // ---- the waves' sums meet: o[dt][i] is column 16 dt + 4 g + i of head n
    l = sum_of_quarters(l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(o_lds + n * kPitch + dt * 16 + 4 * g) = o[dt];
    if (g == 0) {
      m_lds[wave][n] = m;
      l_lds[wave][n] = l;
    }
    __syncthreads();
    const bool mine = block0 == 0 && count == blocks;
    const int slot = worker * 2 + (block0 != 0 ? 0 : 1);         // what another began, or what it begins
    if (threadIdx.x == 0 && w.workers && block0 == 0 && !mine)
      w.begun[worker] = BegunUnit{b, u, worker_of(total, w.workers, cur + blocks - 1), 0};
    for (int i = threadIdx.x; i < rows * (COLS / 4); i += W * kWave) {
      const int r = i / (COLS / 4), d = i % (COLS / 4) * 4;
      if (PADDED && d >= dim) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int x = 0; x < W; ++x) top = fmaxf(top, m_lds[x][r]);
      f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
      const float base = top == -INFINITY ? 0.0f : top;             // no key: sums of 0; a NaN among the scores stays one
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float f = __builtin_amdgcn_exp2f(m_lds[x][r] - base);
        const f32x4 ox = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * kWaveBytes) + r * kPitch + d);
        sum = fmaf(l_lds[x][r], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = fmaf(ox[e], f, out[e]);
      }
      if (!mine) {
        *reinterpret_cast<f32x4*>(w.part_o + ((int64_t)slot * 16 + r) * dim + d) = out;
        if (d == 0) w.part_ml[slot * 16 + r] = float2{top, sum};
        continue;
      }
      if (w.sums.slots) {                                            // to be joined with others
        keep_sums(w, (int64_t)token * a.heads + head0 + r, dim, d, out, float2{top, sum});
        continue;
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      store4o<T>(static_cast<T*>(a.out) + token * a.out_token + (head0 + r) * a.out_head + d, out[0] * inv, out[1] * inv, out[2] * inv, out[3] * inv);
    }
    __syncthreads();                                                 // before the LDS holds V again
    cur += count;
  }
}

template <typename T, typename Kind, int D, int COLS, bool PADDED>
__global__ __launch_bounds__(kWaves * kWave, D == 256 ? 1 : 2)
void paged_decode_kernel(PagedAttnArgs a, Pages p, DecodeArgs w) {
  __shared__ __attribute__((aligned(16))) char lds[kWaves * decode_wave_bytes(D, COLS)];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
  paged_decode_worker<T, Kind, D, COLS, PADDED, kWaves>(a, p, w, blockIdx.x, lds, m_lds, l_lds);
}

}  // namespace

template <typename Kind>
int launch_paged_workers(const PagedAttnArgs& a, const Pages& p, const DecodeArgs& w, unsigned grid, int dtype, hipStream_t s) {
  return with_width<256>(a.dim, [&](auto width) {
    typedef decltype(width) W;
    if (dtype == HEXMI_F16)
      hipLaunchKernelGGL((paged_decode_kernel<f16, Kind, W::D, W::COLS, W::PADDED>), dim3(grid), dim3(kWaves * kWave), 0, s, a, p, w);
    else
      hipLaunchKernelGGL((paged_decode_kernel<bf16, Kind, W::D, W::COLS, W::PADDED>), dim3(grid), dim3(kWaves * kWave), 0, s, a, p, w);
    return launch_status();
  });
}

}  // namespace hexmi
