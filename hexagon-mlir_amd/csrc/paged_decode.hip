// Attention of one new token a sequence over the pages of its sequence (fp16 / bf16): a decode step of a batch.
//
// Bound by HBM: every key and value of a sequence is read once, for all the query heads that share its key head. Those heads (up to 16)
// are the columns of v_mfma_f32_16x16x32: a wave takes 32 keys at a time,
//   S^T = K Q^T    a lane's A operand is 16 bytes of a key's row, straight from its page to registers; a lane then holds 8 scores of one head
//   O^T += V^T P^T the probabilities go from the score registers to the B operand as they are (which key stands in which slot of the
//                  product is free: slot 8 g + 4 t + i is key 16 t + 4 g + i); V passes through a wave's own LDS and is read transposed
//                  (ds_read_b64_tr_b16).
// Keys and values of the next 32 are asked for as soon as the registers of these are free, so a wave has 16 KiB (heads of 128) on the way
// at nearly all times, eight waves a compute unit.
//
// The work is cut evenly whatever the lengths are: the blocks of kBlockKeys keys of all sequences and key heads, one behind the other,
// are dealt to the workers (workgroups) in equal runs. A worker that has all of a unit (sequence, key head, 16 query heads) writes
// its rows; of a unit that several share every worker leaves its sums, at most two sets, which a second launch joins in the order of
// the keys. Nothing is added atomically.
#include "flash_attn_tiles.h"
#include "paged.h"

namespace hexmi {
namespace {

constexpr int kWaves = 4, kTileKeys = 32, kBlockKeys = kWaves * kTileKeys;

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
__device__ __forceinline__ int blocks_of_keys(int keys) { return keys > kBlockKeys ? (keys + kBlockKeys - 1) / kBlockKeys : 1; }
__device__ __forceinline__ int blocks_of(const Pages& p, int b, int prefix) { return blocks_of_keys(length_of(p, b) - prefix); }
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
  int length, blocks, up_to;                   // lane b: of sequence b, and of all up to it
  int of_64, all;                              // blocks of the first 64 sequences, of all (one unit's)
};
__device__ __forceinline__ BlockList block_list(const Pages& p, int prefix, int lane) {
  BlockList l;
  l.length = lane < p.sequences ? length_of(p, lane) : 0;
  l.blocks = lane < p.sequences ? blocks_of_keys(l.length - prefix) : 0;
  l.up_to = sum_up_to(l.blocks);
  l.of_64 = of_last_lane(l.up_to);
  int more = 0;
  for (int b0 = kWave; b0 < p.sequences; b0 += kWave) more += b0 + lane < p.sequences ? blocks_of(p, b0 + lane, prefix) : 0;
  l.all = l.of_64 + (p.sequences > kWave ? of_last_lane(sum_up_to(more)) : 0);
  return l;
}
// The sequence that block `at` of the list belongs to, with `units` units a sequence, and the blocks (of one unit) before it.
__device__ __forceinline__ int sequence_at(const BlockList& l, const Pages& p, int prefix, int units, int at, int lane, int& before) {
  before = 0;
  for (int b0 = 0;; b0 += kWave) {
    const int n = b0 == 0 ? l.blocks : b0 + lane < p.sequences ? blocks_of(p, b0 + lane, prefix) : 0, sum = b0 == 0 ? l.up_to : sum_up_to(n);
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

// A unit that a worker begins and others go on with: its sequence, unit and last worker (none: last < 0).
struct Shared {
  int sequence, unit, last, pad;
};
struct DecodeArgs {
  float* part_o;                               // [workers][2][16][dim]
  float2* part_ml;                             // [workers][2][16]
  Shared* begun;                               // [workers]
  int workers, row_tiles;
  RowSums prefix;
};

// D: columns of a row in LDS; COLS <= D, a multiple of 32: columns that are multiplied; PADDED: a head is narrower than COLS. A lane whose
// columns lie past the head reads the head's first ones instead: the query has zeros there, and what comes of V there is not stored.
template <typename T, int D, int COLS, bool PADDED>
__global__ __launch_bounds__(kWaves * kWave, D == 256 ? 1 : 2)
void paged_decode_kernel(PagedAttnArgs a, Pages p, DecodeArgs w) {
  typedef typename MfmaT<T>::Frag Frag;
  constexpr int DS = COLS / 32, DT = COLS / 16, CPR = D / 8, kPitch = COLS + 4;
  constexpr int kSumBytes = (16 * kPitch * 4 + D * 2 - 1) / (D * 2) * (D * 2);      // a wave's part starts at a row's multiple
  constexpr int kWaveBytes = kTileKeys * D * 2 > kSumBytes ? kTileKeys * D * 2 : kSumBytes;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWaveBytes];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane / 16, n = lane % 16;
  const int dim = PADDED ? a.dim : COLS;
  // This lane's bytes of V in LDS, rows of D columns in 16-byte chunks: chunk g of row n, where it puts, and columns 4 (n % 4) .. of row
  // 4 g + n / 4, from where it takes (ds_read_b64_tr_b16: a group of 16 lanes asks for 4 rows x 16 columns, and a lane gets a column).
  // Other chunks are these with the chunk's number XORed in.
  const int put_at = wave * kWaveBytes + n * (D * 2) + (g ^ swz_pairs<D>(n)) * 16;
  const int take_row = 4 * g + (n >> 2), take_at = wave * kWaveBytes + take_row * (D * 2) + (((n & 3) >> 1) ^ swz_pairs<D>(take_row)) * 16 + (n & 1) * 8;
  float* o_lds = reinterpret_cast<float*>(lds + wave * kWaveBytes);
  const int units = p.kv_heads * w.row_tiles;

  BlockList list;
  int cur, end, b, before = 0, total = 0;
  if (w.workers == 0) {                        // a unit each
    b = blockIdx.x / units;
    list.length = 0;
    const int u = blockIdx.x - b * units, blocks = __builtin_amdgcn_readfirstlane(blocks_of(p, b, a.prefix));
    cur = u * blocks;
    end = cur + blocks;
  } else {
    list = block_list(p, a.prefix, lane);
    total = list.all * units;
    cur = run_start(total, w.workers, blockIdx.x);
    end = run_start(total, w.workers, blockIdx.x + 1);
    if (wave == 0 && lane == 0) w.begun[blockIdx.x].last = -1;
    if (cur >= end) return;
    b = sequence_at(list, p, a.prefix, units, cur, lane, before);
  }
  const int start = cur;

  while (cur < end) {
    const int length = w.workers ? length_at(list, p, b) : __builtin_amdgcn_readfirstlane(length_of(p, b));
    const int blocks = blocks_of_keys(length - a.prefix), local = cur - before * units;
    if (local >= blocks * units) {             // on to the next sequence
      before += blocks;
      ++b;
      continue;
    }
    const int u = local / blocks, block0 = local - u * blocks;
    const int count = end - cur < blocks - block0 ? end - cur : blocks - block0;
    const int kvh = u / w.row_tiles, row0 = (u - kvh * w.row_tiles) * 16;
    const int rows = a.group - row0 < 16 ? a.group - row0 : 16;
    const int head0 = kvh * a.group + row0;

    // ---- queries: the B operand, head n's columns 32 ds + 8 g ..
    Frag qf[DS];
    int col[DS];
    {
      const T* q = static_cast<const T*>(a.q) + b * a.q_token + (head0 + (n < rows ? n : rows - 1)) * a.q_head;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) {
        const int c = ds * 32 + g * 8;
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
    const int key_first = a.prefix + (block0 * kWaves + wave) * kTileKeys;
    int key_end = a.prefix + (block0 + count) * kBlockKeys;
    key_end = key_end < length ? key_end : length;
    const int32_t* table = p.table + b * p.table_row;
    const T* k_head = static_cast<const T*>(a.k) + kvh * p.k_head;
    const T* v_head = static_cast<const T*>(a.v) + kvh * p.v_head;
    // where keys key0 + n and key0 + 16 + n stand; past the end: the last key again, without weight
    struct Keys { int page[2]; };
    auto clamped = [&](int key) __attribute__((always_inline)) { return key < key_end ? key : key_end - 1; };
    auto find = [&](int key0) __attribute__((always_inline)) {
      Keys k;
#pragma unroll
      for (int t = 0; t < 2; ++t) k.page[t] = table[divided(clamped(key0 + t * 16 + n), p.size)];
      return k;
    };
    auto there = [&](int page) __attribute__((always_inline)) { return page >= 0 && page < p.num_pages; };
    auto load = [&](const Keys& at, int key0, const T* base, int64_t page_stride, int64_t slot_stride, u32x4 (*r)[DS]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = clamped(key0 + t * 16 + n), slot = key - divided(key, p.size) * p.page_size;
        const T* row = base + (there(at.page[t]) ? at.page[t] : 0) * page_stride + slot * slot_stride;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) r[t][ds] = *reinterpret_cast<const u32x4*>(row + col[ds]);
      }
    };
    if (key_first < key_end) {
      u32x4 kr[2][DS], vr[2][DS];
      Keys now = find(key_first), next = find(key_first + kBlockKeys);
      load(now, key_first, k_head, p.k_page, p.k_slot, kr);
      load(now, key_first, v_head, p.v_page, p.v_slot, vr);
      for (int key0 = key_first; key0 < key_end; key0 += kBlockKeys) {
        __builtin_amdgcn_sched_barrier(0);
        // what the constants of a chunk are XORed into; kept from becoming a register each
        int to = put_at, from = take_at;
        asm volatile("" : "+v"(to), "+v"(from));
        f32x4 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
          for (int t = 0; t < 2; ++t) s[t] = Mfma16<T>::run(__builtin_bit_cast(Frag, kr[t][ds]), qf[ds], s[t]);
        const bool ok0 = there(now.page[0]) && key0 + n < key_end, ok1 = there(now.page[1]) && key0 + 16 + n < key_end;
        const bool whole = __ballot(ok0 && ok1) == ~0ull;
        __builtin_amdgcn_sched_barrier(0);
        load(next, key0 + kBlockKeys, k_head, p.k_page, p.k_slot, kr);
        __builtin_amdgcn_sched_barrier(0);
        if (!whole) {                                                // what stands where no key is may be anything: no weight, and zeros of V
          const uint32_t k0 = (uint32_t)__ballot(ok0), k1 = (uint32_t)__ballot(ok1);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!(k0 >> (4 * g + i) & 1)) s[0][i] = -INFINITY;
            if (!(k1 >> (4 * g + i) & 1)) s[1][i] = -INFINITY;
          }
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) {
            if (!ok0) vr[0][ds] = u32x4{0u, 0u, 0u, 0u};
            if (!ok1) vr[1][ds] = u32x4{0u, 0u, 0u, 0u};
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int ds = 0; ds < DS; ++ds) *reinterpret_cast<u32x4*>(lds + (to ^ (ds * 64)) + t * (16 * D * 2)) = vr[t][ds];
        __builtin_amdgcn_sched_barrier(0);
        load(next, key0 + kBlockKeys, v_head, p.v_page, p.v_slot, vr);
        __builtin_amdgcn_sched_barrier(0);
        // online softmax, the reference maximum up to kRescaleLag behind the true one (flash_attn.hip)
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_of_quarters(mx) * a.scale;
        const bool grow = mx > m + kRescaleLag;
        if (__ballot(grow) != 0) {
          const float m_new = grow ? mx : m, alpha = grow ? __builtin_amdgcn_exp2f(m - m_new) : 1.0f;
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
        const Frag pf = MfmaT<T>::pack(pr);
        l = MfmaT<T>::sum8(pf, l);                                   // the sum of what the product multiplies
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
        next = find(key0 + 2 * kBlockKeys);
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
    const int slot = blockIdx.x * 2 + (block0 != 0 ? 0 : 1);         // what another began, or what it begins
    if (threadIdx.x == 0 && w.workers && block0 == 0 && !mine)
      w.begun[blockIdx.x] = Shared{b, u, worker_of(total, w.workers, cur + blocks - 1), 0};
    for (int i = threadIdx.x; i < rows * (COLS / 4); i += kWaves * kWave) {
      const int r = i / (COLS / 4), d = i % (COLS / 4) * 4;
      if (PADDED && d >= dim) continue;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) top = fmaxf(top, m_lds[x][r]);
      f32x4 out = {0.0f, 0.0f, 0.0f, 0.0f};
      if (top != -INFINITY) {
#pragma unroll
        for (int x = 0; x < kWaves; ++x) {
          const float f = __builtin_amdgcn_exp2f(m_lds[x][r] - top);
          const f32x4 ox = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * kWaveBytes) + r * kPitch + d);
          sum = fmaf(l_lds[x][r], f, sum);
#pragma unroll
          for (int e = 0; e < 4; ++e) out[e] = fmaf(ox[e], f, out[e]);
        }
      }
      if (!mine) {
        *reinterpret_cast<f32x4*>(w.part_o + ((int64_t)slot * 16 + r) * dim + d) = out;
        if (d == 0) w.part_ml[slot * 16 + r] = float2{top, sum};
        continue;
      }
      if (w.prefix.slots) {                                          // to be joined with the prefix's
        const int64_t at = (w.prefix.slots - 1) * w.prefix.rows + (int64_t)b * a.heads + head0 + r;
        *reinterpret_cast<f32x4*>(w.prefix.o + at * dim + d) = out;
        if (d == 0) w.prefix.ml[at] = float2{top, sum};
        continue;
      }
      const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
      store4o<T>(static_cast<T*>(a.out) + b * a.out_token + (head0 + r) * a.out_head + d, out[0] * inv, out[1] * inv, out[2] * inv, out[3] * inv);
    }
    __syncthreads();                                                 // before the LDS holds V again
    cur += count;
  }
}

// The units that several workers share: block (w, row) takes the one that worker w began. Behind a prefix every unit is joined with its
// sums: block (unit, row).
template <typename T>
__global__ __launch_bounds__(256)
void paged_decode_join_kernel(PagedAttnArgs a, Pages p, DecodeArgs w) {
  __shared__ float o_lds[8][256 + 4];
  __shared__ float m_lds[8], l_lds[8];
  const int units = p.kv_heads * w.row_tiles, r = blockIdx.y;
  int b, u, w0 = 0, w1 = 0;
  if (w.prefix.slots) {
    b = blockIdx.x / units;
    u = blockIdx.x - b * units;
    if (w.workers) {
      const int lane = threadIdx.x % kWave;
      const BlockList list = block_list(p, a.prefix, lane);
      int before = 0;
      for (int x = lane; x < b; x += kWave) before += x < kWave ? list.blocks : blocks_of(p, x, a.prefix);
      const int blocks = blocks_of_keys(length_at(list, p, b) - a.prefix), total = list.all * units;
      const int first = of_last_lane(sum_up_to(before)) * units + u * blocks;
      w0 = worker_of(total, w.workers, first);
      w1 = worker_of(total, w.workers, first + blocks - 1);
    }
  } else {
    const Shared begun = w.begun[blockIdx.x];
    if (begun.last < 0) return;
    b = begun.sequence;
    u = begun.unit;
    w0 = blockIdx.x;
    w1 = begun.last;
  }
  const int kvh = u / w.row_tiles, row0 = (u - kvh * w.row_tiles) * 16;
  if (r >= a.group - row0) return;
  const int head = kvh * a.group + row0 + r;
  const int64_t row = (int64_t)b * a.heads + head;
  // eight groups of 32 threads take every eighth set of sums, a thread the columns d and, past 128, d + 128
  const int group = threadIdx.x / 32, d = threadIdx.x % 32 * 4;
  float top = -INFINITY, sum = 0.0f;
  f32x4 out[2] = {};
  auto take = [&](float2 ml, const float* o) __attribute__((always_inline)) {
    if (!(ml.y > 0.0f)) return;
    const float new_top = fmaxf(top, ml.x), f = __builtin_amdgcn_exp2f(ml.x - new_top), old = __builtin_amdgcn_exp2f(top - new_top);
    sum = fmaf(ml.y, f, sum * old);
    top = new_top;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (d + h * 128 < a.dim) {
        const f32x4 ox = *reinterpret_cast<const f32x4*>(o + d + h * 128);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[h][e] = fmaf(ox[e], f, out[h][e] * old);
      }
  };
  for (int x = w0 + group; x <= w1 && w0 < w1; x += 8) {
    const int64_t slot = (int64_t)x * 2 + (x == w0 ? 1 : 0);
    take(w.part_ml[slot * 16 + r], w.part_o + (slot * 16 + r) * a.dim);
  }
  for (int x = group; x < w.prefix.slots - (w0 < w1 ? 1 : 0); x += 8) take(w.prefix.ml[x * w.prefix.rows + row], w.prefix.o + (x * w.prefix.rows + row) * a.dim);
#pragma unroll
  for (int h = 0; h < 2; ++h) *reinterpret_cast<f32x4*>(&o_lds[group][d + h * 128]) = out[h];
  if (d == 0) {
    m_lds[group] = top;
    l_lds[group] = sum;
  }
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= a.dim) return;
  top = -INFINITY;
  for (int x = 0; x < 8; ++x) top = fmaxf(top, m_lds[x]);
  float l = 0.0f, o = 0.0f;
  if (top != -INFINITY)
    for (int x = 0; x < 8; ++x) {
      const float f = __builtin_amdgcn_exp2f(m_lds[x] - top);
      l = fmaf(l_lds[x], f, l);
      o = fmaf(o_lds[x][c], f, o);
    }
  static_cast<T*>(a.out)[b * a.out_token + head * a.out_head + c] = from_f32<T>(l > 0.0f ? o / l : 0.0f);
}

template <typename T>
int launch(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, const DecodeArgs& w, hipStream_t s) {
  const unsigned grid = plan.workers ? plan.workers : (unsigned)((int64_t)p.sequences * p.kv_heads * plan.row_tiles);
#define HEXMI_PAGED_DECODE(D, COLS)                                                                                                      \
  do {                                                                                                                                   \
    if (a.dim == COLS) hipLaunchKernelGGL((paged_decode_kernel<T, D, COLS, false>), dim3(grid), dim3(kWaves * kWave), 0, s, a, p, w);    \
    else hipLaunchKernelGGL((paged_decode_kernel<T, D, COLS, true>), dim3(grid), dim3(kWaves * kWave), 0, s, a, p, w);                   \
  } while (0)
  if (a.dim <= 64) HEXMI_PAGED_DECODE(64, 64);
  else if (a.dim <= 96) HEXMI_PAGED_DECODE(128, 96);
  else if (a.dim <= 128) HEXMI_PAGED_DECODE(128, 128);
  else HEXMI_PAGED_DECODE(256, 256);
#undef HEXMI_PAGED_DECODE
  const int rc = launch_status();
  if (rc != HEXMI_OK || (plan.workers < 2 && w.prefix.slots == 0)) return rc;
  const unsigned joins = w.prefix.slots ? (unsigned)((int64_t)p.sequences * p.kv_heads * plan.row_tiles) : plan.workers - 1;
  hipLaunchKernelGGL((paged_decode_join_kernel<T>), dim3(joins, plan.rows), dim3(256), 0, s, a, p, w);
  return launch_status();
}

}  // namespace

PagedDecodePlan plan_paged_decode(const hexmi_paged_batch& b, int64_t heads, int64_t prefix) {
  const int64_t group = heads / b.kv_heads, tiles = (group + 15) / 16, units = b.sequences * b.kv_heads * tiles;
  const int64_t most = b.table_cols * b.page_size - prefix, blocks = most > kBlockKeys ? (most + kBlockKeys - 1) / kBlockKeys : 1;
  const int rows = (int)(group < 16 ? group : 16);
  if (blocks <= 1) return {0, (int)tiles, rows};
  // A block each while they are fewer than the compute units; then four and more, so that a worker's sums are few beside its keys, on as
  // many workgroups as a compute unit holds. One and two a compute unit, heads of 128: 1 sequence x 16000 keys x 8 heads 21.9 / 24.5 us,
  // 3 x 5000 15.2 / 17.0; 128 x 500 58 / 52, 16 x 2048 x 32 97.7 / 93.5. Heads of 256, of which it holds one: 16 x 2048 x 8 56 / 60.
  const int64_t cus = hexmi_num_cus(), all = units * blocks, held = cus * (b.dim <= 96 ? 3 : b.dim <= 128 ? 2 : 1);
  const int64_t fours = all / 4 < cus ? cus : all / 4, workers = all < cus ? all : fours < held ? fours : held;
  return {(int)(workers < 1 ? 1 : workers), (int)tiles, rows};
}

int64_t paged_decode_workspace(const PagedDecodePlan& plan, int64_t dim) {
  return (int64_t)plan.workers * (2 * 16 * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2)) + (int64_t)sizeof(Shared));
}

int paged_decode(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, int dtype, void* workspace, const RowSums& prefix,
                 hipStream_t s) {
  float* o = static_cast<float*>(workspace);
  float2* ml = reinterpret_cast<float2*>(o + (int64_t)plan.workers * 2 * 16 * a.dim);
  const DecodeArgs w = {o, ml, reinterpret_cast<Shared*>(ml + (int64_t)plan.workers * 2 * 16), plan.workers, plan.row_tiles, prefix};
  return dtype == HEXMI_F16 ? launch<f16>(plan, a, p, w, s) : launch<bf16>(plan, a, p, w, s);
}

}  // namespace hexmi
