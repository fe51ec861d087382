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
__device__ __forceinline__ int blocks_of(const Pages& p, int b, int prefix) {
  const int keys = length_of(p, b) - prefix;
  return keys > kBlockKeys ? (keys + kBlockKeys - 1) / kBlockKeys : 1;
}
__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int x = 1; x < kWave; x *= 2) v += __shfl_xor(v, x);
  return v;
}
__device__ __forceinline__ int all_blocks(const Pages& p, int prefix, int lane) {
  int n = 0;
  for (int b = lane; b < p.sequences; b += kWave) n += blocks_of(p, b, prefix);
  return wave_sum_int(n);
}
// The sequence that block `at` of the list of all blocks belongs to, with `units` units a sequence, and the blocks (of one unit)
// before it.
__device__ __forceinline__ int sequence_at(const Pages& p, int prefix, int units, int at, int lane, int& before) {
  before = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += kWave) {
    const int b = b0 + lane, n = b < p.sequences ? blocks_of(p, b, prefix) : 0;
    int sum = n;
#pragma unroll
    for (int x = 1; x < kWave; x *= 2) {
      const int below = __shfl_up(sum, x);
      if (lane >= x) sum += below;
    }
    const uint64_t past = __ballot((before + sum) * units > at);
    if (past) {
      const int first = __ffsll((unsigned long long)past) - 1;
      before += __shfl(sum - n, first);
      return b0 + first;
    }
    before += __shfl(sum, kWave - 1);
  }
  return p.sequences;                          // at is past the end: callers do not ask
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

struct DecodeArgs {
  float* part_o;                               // [workers][2][16][dim]
  float2* part_ml;                             // [workers][2][16]
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
  constexpr int kWaveBytes = kTileKeys * D * 2 > 16 * kPitch * 4 ? kTileKeys * D * 2 : 16 * kPitch * 4;
  __shared__ __attribute__((aligned(16))) char lds[kWaves * kWaveBytes];
  __shared__ float m_lds[kWaves][16], l_lds[kWaves][16];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int g = lane / 16, n = lane % 16;
  const int dim = PADDED ? a.dim : COLS;
  T* v_lds = reinterpret_cast<T*>(lds + wave * kWaveBytes);
  float* o_lds = reinterpret_cast<float*>(lds + wave * kWaveBytes);
  const int units = p.kv_heads * w.row_tiles;

  int cur, end, b, before, start = 0;
  if (w.workers == 0) {                        // a unit each
    b = blockIdx.x / units;
    before = 0;
    const int u = blockIdx.x - b * units, blocks = blocks_of(p, b, a.prefix);
    cur = u * blocks;
    end = cur + blocks;
    start = cur;
  } else {
    const int total = all_blocks(p, a.prefix, lane) * units;
    cur = run_start(total, w.workers, blockIdx.x);
    end = run_start(total, w.workers, blockIdx.x + 1);
    if (cur >= end) return;
    start = cur;
    b = sequence_at(p, a.prefix, units, cur, lane, before);
  }
  b = __builtin_amdgcn_readfirstlane(b);
  before = __builtin_amdgcn_readfirstlane(before);

  while (cur < end) {
    const int length = length_of(p, b), blocks = blocks_of(p, b, a.prefix), local = cur - before * units;
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
    struct Keys { int page[2], slot[2]; };
    auto find = [&](int key0) __attribute__((always_inline)) {       // where keys key0 + n and key0 + 16 + n stand
      Keys k;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        int key = key0 + t * 16 + n;
        key = key < key_end ? key : key_end - 1;                     // past the end: the last key again, without weight
        const int column = divided(key, p.size);
        k.page[t] = table[column];
        k.slot[t] = key - column * p.page_size;
      }
      return k;
    };
    auto there = [&](int page) __attribute__((always_inline)) { return page >= 0 && page < p.num_pages; };
    u32x4 kr[2][DS], vr[2][DS];
    auto load = [&](const Keys& at, const T* base, int64_t page, int64_t slot, u32x4 (*r)[DS]) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const T* row = base + (there(at.page[t]) ? at.page[t] : 0) * page + at.slot[t] * slot;
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) r[t][ds] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row + col[ds]));
      }
    };
    if (key_first < key_end) {
      Keys now = find(key_first), next = find(key_first + kBlockKeys);
      load(now, k_head, p.k_page, p.k_slot, kr);
      load(now, v_head, p.v_page, p.v_slot, vr);
      for (int key0 = key_first; key0 < key_end; key0 += kBlockKeys) {
        __builtin_amdgcn_sched_barrier(0);
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
        load(next, k_head, p.k_page, p.k_slot, kr);                  // past the last tile: its last key again
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
          for (int ds = 0; ds < DS; ++ds) {
            const int row = t * 16 + n;
            *reinterpret_cast<u32x4*>(v_lds + (row * CPR + ((ds * 4 + g) ^ swz_pairs<D>(row))) * 8) = vr[t][ds];
          }
        __builtin_amdgcn_sched_barrier(0);
        load(next, v_head, p.v_page, p.v_slot, vr);
        now = next;
        next = find(key0 + 2 * kBlockKeys);
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
          for (int t = 0; t < 2; ++t) {
            const int row = t * 16 + 4 * g + (n >> 2), c = (dt * 2 + ((n & 3) >> 1)) ^ swz_pairs<D>(row);
            v.h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) i16x4*)(v_lds + (row * CPR + c) * 8 + (n & 1) * 4));
          }
          o[dt] = Mfma16<T>::run(v.f, pf, o[dt]);
        }
        asm volatile("" ::: "memory");
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
    const int slot = blockIdx.x * 2 + (cur == start && block0 != 0 ? 0 : 1);
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

// The units that several workers share: block (w, row) looks at the boundary between workers w and w + 1, and takes the unit that it
// falls into if no earlier boundary does. Behind a prefix every unit is joined with its sums: block (unit, row).
template <typename T>
__global__ __launch_bounds__(256)
void paged_decode_join_kernel(PagedAttnArgs a, Pages p, DecodeArgs w) {
  __shared__ float o_lds[8][256 + 4];
  __shared__ float m_lds[8], l_lds[8];
  const int lane = threadIdx.x % kWave, units = p.kv_heads * w.row_tiles;
  int total = 0, b, u, first = 0, blocks = 1;
  if (w.prefix.slots) {
    b = blockIdx.x / units;
    u = blockIdx.x - b * units;
    if (w.workers) {
      int before = 0;
      for (int x = lane; x < p.sequences; x += kWave) {
        const int n = blocks_of(p, x, a.prefix);
        total += n;
        if (x < b) before += n;
      }
      total = wave_sum_int(total) * units;
      blocks = blocks_of(p, b, a.prefix);
      first = wave_sum_int(before) * units + u * blocks;
    }
  } else {
    total = all_blocks(p, a.prefix, lane) * units;
    const int at = run_start(total, w.workers, blockIdx.x + 1);
    if (at >= total) return;
    int before;
    b = sequence_at(p, a.prefix, units, at, lane, before);
    blocks = blocks_of(p, b, a.prefix);
    u = (at - before * units) / blocks;
    first = before * units + u * blocks;
    if (at == first || run_start(total, w.workers, blockIdx.x) > first) return;
  }
  const int kvh = u / w.row_tiles, row0 = (u - kvh * w.row_tiles) * 16, r = blockIdx.y;
  if (r >= a.group - row0) return;
  const int head = kvh * a.group + row0 + r;
  const int w0 = w.workers ? worker_of(total, w.workers, first) : 0, w1 = w.workers ? worker_of(total, w.workers, first + blocks - 1) : 0;
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
  const int64_t workers = 2 * (int64_t)hexmi_num_cus();
  return {(int)(units * blocks < workers ? units * blocks : workers), (int)tiles, rows};
}

int64_t paged_decode_workspace(const PagedDecodePlan& plan, int64_t dim) {
  return (int64_t)plan.workers * 2 * 16 * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
}

int paged_decode(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, int dtype, void* workspace, const RowSums& prefix,
                 hipStream_t s) {
  float* o = static_cast<float*>(workspace);
  const DecodeArgs w = {o, reinterpret_cast<float2*>(o + (int64_t)plan.workers * 2 * 16 * a.dim), plan.workers, plan.row_tiles, prefix};
  return dtype == HEXMI_F16 ? launch<f16>(plan, a, p, w, s) : launch<bf16>(plan, a, p, w, s);
}

}  // namespace hexmi
