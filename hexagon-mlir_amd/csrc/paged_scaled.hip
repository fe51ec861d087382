// Keys and values of new tokens into a paged cache in 8 bits: rows normed and turned as head_rows.hip has them, rounded to e4m3 with one
// power-of-two scale for each block of slots and head; the queries' rows beside them.
//
// A block's scale is known when all of the call's rows in it are, so a workgroup takes the new tokens of one block of one sequence and a share
// of the heads: the angles of its tokens are worked out once, into LDS, and a wave takes a head's keys or values of the block, held in registers
// while the largest value is found. A scale is a power of two so that it can rise while a block fills: older numbers keep their bits then, but
// for what falls below e4m3's normal numbers.
// Bound by its launch up to some hundred tokens (64 tokens x 32 + 8 heads of 128 5.1 us), then by rows in flight: prompts of 8100 tokens, normed
// and turned, 46.8 us (3.6 TB/s; a copy of that size 34). That is with blocks of 16: 32 and 64 slots, which a wave does not hold and goes through
// twice, take 65 and 79 us, heads of 256 76 in blocks of 16 and 212 of 64; 600 tokens 10 us, in blocks of 64 32.
#include "head_rows.h"

namespace hexmi {
namespace {

// Workgroups wanted for keys and values: a unit's heads are shared while they are fewer. 1024 / 2048 / 4096: prompts of 8100 tokens 46.5 / 50.9 /
// 51.2 us (every share works out the angles again); keys and values by workgroups of their own 51 (their rows stand side by side). 512 / 1024 / 2048
// over other batches, us: 32 x 100 25.8 / 21.9 / 22.5, blocks of 64 81.5 / 77.1 / 77.3, up to 600 tokens and one key head level; the other way round
// 32 key heads of 64 76 / 59 / 54, 16000 tokens 92.0 / 92.2 / 87.8, heads of 256 68.5 / 73.5 / 73.2.
constexpr int kUnitGroups = 1024;

// Units (a sequence's new tokens of one block): those of sequence b are numbered from first_unit(b) on, b = -1 .. sequences (first_row). n
// tokens stand in at most floor((n - 2) / block) + 2 blocks and floor(x1 / block) - floor(x0 / block) >= floor(n / block) for x1 = x0 + n, so
// two more for each sequence are enough; some numbers are no unit.
__device__ __forceinline__ int first_unit(const Pages& p, const Scales& s, int b) { return b < 0 ? 0 : divided(first_row(p, b), s.by_block) + 2 * (b + 1); }
__device__ __forceinline__ int sequence_of_unit(const Pages& p, const Scales& s, int unit, int lane) {
  int lo = -1, hi = p.sequences + 1;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const int n = __popcll(__ballot(at < hi && first_unit(p, s, at) <= unit));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
    if (step == 1) break;
  }
  return lo;
}

// the largest over the LPR lanes of a row, in all of them
template <int LPR>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  float a, b;
  if constexpr (LPR >= 16) v = fmaxf(v, dpp_move<0x140>(v));
  if constexpr (LPR >= 32) {
    swap16(v, a, b);
    v = fmaxf(a, b);
  }
  return v;
}

// Eight values, ones that are not finite as NaN, over 2^e, rounded to e4m3. Numbers end at 240 times T's largest exponent, which is within 448 2^e
// where e is below that; where an older exponent leaves fewer bits of it than there are, at the next multiple of 2^(e - 9) below.
template <typename T>
__device__ __forceinline__ u32x2 to_codes(const float* y, int e) {
  constexpr int kOver = kMostExponent<T> + 14;
  constexpr float kMost = 240.0f * (kMostExponent<T> == 8 ? 0x1p8f : 0x1p120f);
  static_assert(kMostExponent<T> == 8 || kMostExponent<T> == 120);
  const float by = __builtin_amdgcn_ldexpf(1.0f, -e);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fabsf(y[i]) < INFINITY ? fminf(fmaxf(y[i], -kMost), kMost) * by : NAN;
  if constexpr (kOver < 128) {
    if (e >= kOver) {
      const float most = floorf(kMost * by * 512.0f) * 0x1p-9f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] > most ? most : v[i] < -most ? -most : v[i];
    }
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return u32x2{(uint32_t)lo, (uint32_t)hi};
}
// eight numbers of e4m3 times f (at most 1, or NaN), rounded again
__device__ __forceinline__ u32x2 codes_again(u32x2 c, float f) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
    c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, lo, true);
  }
  return c;
}

// Where a unit's tokens stand: rows token0 .. token0 + n - 1 (n <= 0: none) at positions from `position` on, all in one block of a page.
struct Unit {
  int token0, n, page, slot, block, old;       // old: slots of the block, before `slot`, that older tokens of the sequence have
  int64_t position;
};
__device__ __forceinline__ Unit unit_at(const Pages& p, const Scales& sc, int unit, int lane) {
  Unit u = {0, 0, -1, 0, 0, 0, 0};
  int b = unit, n = 1, nth = 0;
  if (p.starts) {
    b = __builtin_amdgcn_readfirstlane(sequence_of_unit(p, sc, unit, lane));
    if (b < 0 || b >= p.sequences) return u;
    u.token0 = first_row(p, b);
    n = first_row(p, b + 1) - u.token0;
    nth = unit - first_unit(p, sc, b);
    if (n <= 0) return u;                      // starts may fall
  } else {
    u.token0 = b;
  }
  const int64_t first = (int64_t)p.lengths[b] - n;
  const int r = first >= 0 ? (int)first - divided((int)first, sc.by_block) * sc.block : (int)((first % sc.block + sc.block) % sc.block);
  const int skip = nth > 0 ? nth * sc.block - r : 0, next = (nth + 1) * sc.block - r;       // tokens before the unit's own, up to its last
  u.token0 += skip;
  u.n = (next < n ? next : n) - skip;
  u.position = first + skip;
  if (u.n <= 0 || u.position < 0 || u.position >= (int64_t)p.table_cols * p.page_size) return u;
  const int column = divided((int)u.position, p.size), page = p.table[b * p.table_row + column];
  if (page < 0 || page >= p.num_pages) return u;
  u.page = page;
  u.slot = (int)u.position - column * p.page_size;
  u.block = divided(u.slot, sc.by_block);
  u.old = u.slot - u.block * sc.block;
  return u;
}

// kv_grid workgroups take a unit and a share of its heads each, q_grid the queries, as head_rows_kernel does; eights of both kinds by turns
// (workgroup ids go round robin to the 8 XCDs), so that neither waits for the other: prompts of 8100 tokens 46.6 us, one kind behind the other
// 56. LPR lanes take a row, eight columns each (HALVES, PIECES: head_rows.h). A wave holds kHeld times the rows that it has at once, so that rows of a block are read and
// turned once; larger blocks are gone through twice. 2 / 4 / 8 times, us: prompts of 8100 tokens 56.2 / 47.6 / 57.2 (more registers, fewer waves), blocks of
// 64 81.4 / 77.1 / 84.6, 600 tokens 12.9 / 10.2 / 12.0, 32 x 100 26.6 / 22.1 / 28.4, heads of 64 57.9 / 58.9 / 83.6; but heads of 256 74.9 / 73.7 / 66.5.
template <typename T, int LPR, bool HALVES, bool PIECES>
__global__ __launch_bounds__(256, 4)
void scaled_rows_kernel(HeadArgs a, Pages p, Scales sc, unsigned kv_grid, unsigned q_grid, int shares, int q_waves) {
  constexpr int kRowsAtOnce = kWave / LPR, kHeld = 4;
  __shared__ __attribute__((aligned(16))) HeadRowsLds<T, LPR, HALVES> lds;
  extern __shared__ __attribute__((aligned(16))) f32x2 angle[];    // [tokens of the block][columns / 2]
  const uint32_t eight = blockIdx.x / 8, kv_eights = (kv_grid + 7) / 8, eights = gridDim.x / 8;
  const uint32_t before = (uint32_t)((uint64_t)eight * kv_eights / eights);      // eights of keys and values before this one
  const bool is_q = (uint32_t)((uint64_t)(eight + 1) * kv_eights / eights) == before;
  const uint32_t id = (is_q ? eight - before : before) * 8 + blockIdx.x % 8;
  if (is_q) {
    HeadArgs q = a;
    q.heads[1] = q.heads[2] = 0;
    if (id < q_grid) head_rows_of<T, LPR, HALVES, PIECES, true>(q, p, q_waves, id, q_grid, lds);
    return;
  }
  if (id >= kv_grid) return;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c0 = lane % LPR * 8, group = lane / LPR, half = a.columns / 2;
  const bool live = c0 < a.dim, turns = c0 < a.columns;
  const int share = id % shares;
  const Unit u = unit_at(p, sc, id / shares, lane);
  if (u.n <= 0 || u.page < 0) return;
  for (int i = threadIdx.x; i < u.n * half; i += 256) {
    const int t = i / half;
    float sn, cs;
    sincos_turns((double)(u.position + t) * a.inv_freq[i - t * half] * 0.15915494309189533577, sn, cs);       // 1 / (2 pi)
    angle[i] = f32x2{cs, sn};
  }
  __syncthreads();

  // row x of keys, token t of the unit, normed and turned
  auto turned = [&](int t, const Eight<T>& x, float* y) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = column(x, e);
    const T* w = static_cast<const T*>(a.kind[1].weight);
    float scale = 1.0f;
    if (w) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(y[e], y[e], sum);
      scale = rms_scale(fmaf(row_sum<LPR>(sum), 1.0f / (float)a.dim, a.eps));
      Eight<T> wt = {};
      if (live) wt = load_eight(w + c0);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * scale * column(wt, e);
    }
    const f32x2* at = angle + t * half;
    if constexpr (HALVES) {
      *reinterpret_cast<Eight<T>*>(&lds.beside[wave][lane * 8]) = x;
      asm volatile("" ::: "memory");                                // a wave's LDS accesses are in order
      const T* row = &lds.beside[wave][group * LPR * 8];
      if (turns) {
        if constexpr (PIECES) {
          const bool second = c0 >= half;
          const int other = second ? c0 - half : c0 + half, i = second ? c0 - half : c0;
          const Eight<T> o = *reinterpret_cast<const Eight<T>*>(row + other);
          Eight<T> ow = {};
          if (w) ow = load_eight(w + other);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float v = column(o, e);
            if (w) v = v * scale * column(ow, e);
            const f32x2 cs = at[i + e];
            y[e] = fmaf(y[e], cs[0], second ? v * cs[1] : -(v * cs[1]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int c = c0 + e;
            if (c >= a.columns) continue;
            const bool second = c >= half;
            const int other = second ? c - half : c + half;
            float v = to_f32<T>(row[other]);
            if (w) v = v * scale * to_f32<T>(w[other]);
            const f32x2 cs = at[second ? c - half : c];
            y[e] = fmaf(y[e], cs[0], second ? v * cs[1] : -(v * cs[1]));
          }
        }
      }
      asm volatile("" ::: "memory");
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c0 + 2 * e >= a.columns) continue;
        const f32x2 cs = at[c0 / 2 + e];
        const float x0 = y[2 * e], x1 = y[2 * e + 1];
        y[2 * e] = fmaf(x0, cs[0], -(x1 * cs[1]));
        y[2 * e + 1] = fmaf(x1, cs[0], x0 * cs[1]);
      }
    }
  };

  // ---- jobs: keys, then values, a head at a time (of one token kRowsAtOnce heads)
  const bool one = u.n == 1;
  const int each = one ? (p.kv_heads + kRowsAtOnce - 1) / kRowsAtOnce : p.kv_heads;
  const int passes = one ? 1 : (u.n + kRowsAtOnce - 1) / kRowsAtOnce;
  for (int job = share * 4 + wave; job < 2 * each; job += shares * 4) {
    const bool v = job >= each;
    const Kind& kind = v ? a.kind[2] : a.kind[1];
    const int in_kind = v ? job - each : job;
    const int at_head = one ? in_kind * kRowsAtOnce + group : in_kind, head = at_head < p.kv_heads ? at_head : p.kv_heads - 1;
    const bool is_head = live && at_head < p.kv_heads;
    const T* rows = static_cast<const T*>(kind.x) + u.token0 * kind.token + head * kind.head + (live ? c0 : 0);
    auto token_of = [&](int pass) __attribute__((always_inline)) {  // past the last: the last again
      const int t = one ? 0 : pass * kRowsAtOnce + group;
      return t < u.n ? t : u.n - 1;
    };
    float y[kHeld][8];
    float largest = 0.0f;
    auto hold = [&](int first) __attribute__((always_inline)) {     // passes first .. first + kHeld - 1, those that there are
      Eight<T> x[kHeld];
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (first + i < passes) x[i] = load_eight(rows + token_of(first + i) * kind.token);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (first + i >= passes) continue;
        if (!live) x[i] = {};
        if (v) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[i][e] = column(x[i], e);
        } else {
          turned(token_of(first + i), x[i], y[i]);
        }
      }
    };
    for (int first = 0; first < passes; first += kHeld) {
      hold(first);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        if (first + i >= passes) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(y[i][e]) < INFINITY ? fabsf(y[i][e]) : 0.0f);
      }
    }
    largest = one ? row_max<LPR>(largest) : wave_max(largest);
    uint8_t* scale = v ? sc.v + u.page * sc.v_page + head * sc.v_head + u.block * sc.v_block
                       : sc.k + u.page * sc.k_page + head * sc.k_head + u.block * sc.k_block;
    const int64_t slot_stride = v ? p.v_slot : p.k_slot;
    uint8_t* codes = static_cast<uint8_t*>(kind.out) + u.slot * slot_stride + c0 + (v ? u.page * p.v_page + head * p.v_head : u.page * p.k_page + head * p.k_head);
    int e = exponent_of(largest);
    e = e < kLeastExponent<T> ? kLeastExponent<T> : e < kMostExponent<T> ? e : kMostExponent<T>;
    if (u.old > 0) {
      // An exponent above T's range (a cache that was filled as another type) stays, so that its numbers keep their values. 255 is none: what
      // it scales is NaN, and becomes e4m3's.
      const int held = *scale, before = held - 127;
      if (before > e && held != 255) e = before;
      if (e != before && is_head) {                                 // older tokens' numbers again
        const float f = held == 255 ? NAN : __builtin_amdgcn_ldexpf(1.0f, before - e);
        for (int s = one ? 0 : group; s < u.old; s += one ? 1 : kRowsAtOnce) {
          u32x2* c = reinterpret_cast<u32x2*>(codes + (s - u.old) * slot_stride);
          *c = codes_again(*c, f);
        }
      }
    }
    for (int first = 0; first < passes; first += kHeld) {
      if (passes > kHeld) hold(first);
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int t = one ? 0 : (first + i) * kRowsAtOnce + group;
        if (first + i < passes && is_head && t < u.n) *reinterpret_cast<u32x2*>(codes + t * slot_stride) = to_codes<T>(y[i], e);
      }
    }
    if (c0 == 0 && is_head && (one || group == 0)) *scale = (uint8_t)(e + 127);
  }
}

template <typename T, int LPR>
int launch_rows(const HeadArgs& a, const Pages& p, const Scales& sc, hipStream_t s) {
  constexpr int64_t rows_at_once = kWave / LPR;
  const int64_t units = p.starts ? (int64_t)p.tokens / sc.block + 2 * ((int64_t)p.sequences + 2) : p.sequences;
  const int64_t jobs = 2 * (p.starts ? p.kv_heads : (p.kv_heads + rows_at_once - 1) / rows_at_once), most = (jobs + 3) / 4;
  int64_t shares = kUnitGroups / (units > 0 ? units : 1);
  shares = shares < 1 ? 1 : shares < most ? shares : most;
  HeadArgs q = a;
  q.heads[1] = q.heads[2] = 0;
  const int64_t q_waves = a.heads[0] > 0 ? waves_per_token<LPR>(q) : 0;
  const int64_t q_blocks = (a.tokens * q_waves + 3) / 4, q_grid = q_blocks < (1 << 22) ? q_blocks : 1 << 22;
  if (!grid_fits(units * shares + q_grid + 16, 256)) return HEXMI_ENOTSUP;
  const unsigned lds = (unsigned)((p.starts ? sc.block : 1) * (a.columns / 2) * sizeof(f32x2)), kv_grid = (unsigned)(units * shares);
  const dim3 grid((kv_grid + 7) / 8 * 8 + (unsigned)(q_grid + 7) / 8 * 8);
  if (grid.x == 0) return HEXMI_OK;
  if (!a.halves || a.columns == 0)
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, false, false>), grid, dim3(256), lds, s, a, p, sc, kv_grid, (unsigned)q_grid, (int)shares, (int)q_waves);
  else if (a.columns % 16 == 0)
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, true, true>), grid, dim3(256), lds, s, a, p, sc, kv_grid, (unsigned)q_grid, (int)shares, (int)q_waves);
  else
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, true, false>), grid, dim3(256), lds, s, a, p, sc, kv_grid, (unsigned)q_grid, (int)shares, (int)q_waves);
  return launch_status();
}
template <typename T>
int launch(const HeadArgs& a, const Pages& p, const Scales& sc, hipStream_t s) {
  return a.dim <= 64 ? launch_rows<T, 8>(a, p, sc, s) : a.dim <= 128 ? launch_rows<T, 16>(a, p, sc, s) : launch_rows<T, 32>(a, p, sc, s);
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

extern "C" int hexmi_paged_append_ex(const hexmi_head_rows* k, const hexmi_head_rows* v, const hexmi_head_rows* q, const hexmi_rotation* rotation,
                                     const hexmi_paged_batch* batch, const hexmi_paged_scales* scales, int dtype, hexmi_stream_t stream) {
  if (!scales) return hexmi_paged_append(k, v, q, rotation, batch, dtype, stream);
  if (!k || !v || !batch) return HEXMI_EINVAL;
  int rc = check_batch(*batch);
  HeadArgs a = {};
  if (rc != HEXMI_OK || (rc = turn(a, rotation, batch->dim)) != HEXMI_OK || (rc = check_scales(*batch, *scales)) != HEXMI_OK) return rc;
  if (k->heads != batch->kv_heads || v->heads != batch->kv_heads) return HEXMI_EINVAL;
  if ((dtype != HEXMI_F16 && dtype != HEXMI_BF16) || batch->dim % 8 != 0 || batch->dim > 256) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))) return HEXMI_EINVAL;
  if (!batch->k_pages || !batch->v_pages || scales->k_scales == scales->v_scales) return HEXMI_EINVAL;
  if ((rc = take(a, 0, q, true)) != HEXMI_OK || (rc = take(a, 1, k, false)) != HEXMI_OK || (rc = take(a, 2, v, false)) != HEXMI_OK) return rc;
  for (int i = 0; i < 3; ++i) {
    const Kind& r = a.kind[i];
    if (!aligned_to(r.x, 16) || !aligned_to(r.weight, 16) || r.token % 8 != 0 || r.head % 8 != 0) return HEXMI_ENOTSUP;
  }
  if (!aligned_to(a.kind[0].out, 16) || a.kind[0].out_token % 8 != 0 || a.kind[0].out_head % 8 != 0) return HEXMI_ENOTSUP;
  for (int64_t s : {batch->k_page, batch->k_head, batch->k_slot, batch->v_page, batch->v_head, batch->v_slot})
    if (s % 8 != 0) return HEXMI_ENOTSUP;
  if (!aligned_to(batch->k_pages, 8) || !aligned_to(batch->v_pages, 8)) return HEXMI_ENOTSUP;
  a.kind[1].out = batch->k_pages;
  a.kind[2].out = batch->v_pages;
  a.kind[2].weight = nullptr;
  a.tokens = (int)batch->tokens;
  begin_call();
  const Pages p = pages_of(*batch);
  const Scales sc = scales_of(*scales);
  return dtype == HEXMI_F16 ? launch<f16>(a, p, sc, as_stream(stream)) : launch<bf16>(a, p, sc, as_stream(stream));
}
