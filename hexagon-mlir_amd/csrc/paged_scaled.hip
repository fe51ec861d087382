// Keys and values of new tokens into a paged cache in 8 bits: rows normed and turned as head_rows.hip has them, rounded to e4m3 with one
// power-of-two scale for each block of slots and head; the queries' rows beside them.
//
// A block's scale is known when all of the call's rows in it are, so a workgroup takes the new tokens of one block of one sequence and a share
// of the heads: the angles of its tokens are worked out once, into LDS, and a wave takes a head's keys or values of the block, first for the
// largest value, then to write them (the rows come out of the caches the second time).
#include "head_rows.h"

namespace hexmi {
namespace {

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

// the least e with most <= 448 * 2^e = 1.75 * 2^(e + 8)
__device__ __forceinline__ int exponent_of(float most) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, most);
  return (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
}
// eight values (finite, or NaN for what is not) times `by`, rounded to e4m3, at most `limit`
__device__ __forceinline__ u32x2 to_codes(const float* y, float by, float limit) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = y[e] * by;
    v[e] = fabsf(y[e]) < INFINITY ? fminf(fmaxf(x, -limit), limit) : NAN;
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
  return u32x2{(uint32_t)lo, (uint32_t)hi};
}
// eight numbers of e4m3 times 2^by (by <= 0), rounded again
__device__ __forceinline__ u32x2 codes_again(u32x2 c, int by) {
  const float f = by < -126 ? 0.0f : power_of_two(by);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
    c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, lo, true);
  }
  return c;
}

// LPR lanes take a row, eight columns each. HALVES, PIECES: head_rows.hip.
template <typename T, int LPR, bool HALVES, bool PIECES>
__global__ __launch_bounds__(256)
void scaled_rows_kernel(HeadArgs a, Pages p, Scales sc, int shares, Divider by_heads) {
  extern __shared__ __attribute__((aligned(16))) f32x2 angle[];    // [tokens of the block][columns / 2]
  __shared__ __attribute__((aligned(16))) T beside[HALVES ? 4 : 1][HALVES ? kWave * 8 : 8];
  constexpr int kRowsAtOnce = kWave / LPR;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c0 = lane % LPR * 8, group = lane / LPR, half = a.columns / 2;
  const bool live = c0 < a.dim, turns = c0 < a.columns;
  const int unit = blockIdx.x / shares, share = blockIdx.x - unit * shares;

  // ---- the tokens: rows token0 .. token0 + m - 1 at positions from `position` on, in one block, or none of them has a page
  int b, token0, n;
  if (!p.starts) {
    b = unit;
    token0 = b;
    n = 1;
  } else {
    b = __builtin_amdgcn_readfirstlane(sequence_of_unit(p, sc, unit, lane));
    token0 = first_row(p, b);
    n = first_row(p, b + 1) - token0;
  }
  const bool none = b < 0 || b >= p.sequences;
  int64_t position = none ? 0 : (int64_t)p.lengths[b] - n;
  const int64_t most = (int64_t)p.table_cols * p.page_size;
  int first = 0;                                                    // tokens before the unit's own
  const int nth = p.starts ? unit - first_unit(p, sc, b) : 0;
  {
    const int r = position >= 0 && position < 0x7fffffff ? (int)position - divided((int)position, sc.by_block) * sc.block
                                                         : (int)((position % sc.block + sc.block) % sc.block);
    if (nth > 0) first = sc.block - r + (nth - 1) * sc.block;
    if (first >= n) return;
    const int next = sc.block - r + nth * sc.block;
    n = (next < n ? next : n) - first;
  }
  token0 += first;
  position += first;
  int page = -1, slot = 0, block = 0, old = 0;                      // old: slots of the block that older tokens of the sequence have
  if (!none && position >= 0 && position < most) {
    const int column = divided((int)position, p.size);
    page = p.table[b * p.table_row + column];
    if (page < 0 || page >= p.num_pages) page = -1;
    slot = (int)position - column * p.page_size;
    block = divided(slot, sc.by_block);
    old = slot - block * sc.block;
  }
  for (int i = threadIdx.x; i < n * half; i += 256) {
    const int t = i / half;
    float sn, cs;
    sincos_turns((double)(position + t) * a.inv_freq[i - t * half] * 0.15915494309189533577, sn, cs);       // 1 / (2 pi)
    angle[i] = f32x2{cs, sn};
  }
  __syncthreads();

  // ---- row (token t, head h) of a kind, normed and turned
  auto fetch = [&](const Kind& kind, int t, int h) __attribute__((always_inline)) {
    Eight<T> x = load_eight(static_cast<const T*>(kind.x) + (token0 + t) * kind.token + h * kind.head + (live ? c0 : 0));
    if (!live) x = {};
    return x;
  };
  auto turned = [&](const Kind& kind, int columns, int t, const Eight<T>& x, float* y) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = column(x, e);
    const T* w = static_cast<const T*>(kind.weight);
    Eight<T> wt = {};
    float scale = 1.0f;
    if (w) {
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(y[e], y[e], sum);
      scale = rms_scale(fmaf(row_sum<LPR>(sum), 1.0f / (float)a.dim, a.eps));
      if (live) wt = load_eight(w + c0);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * scale * column(wt, e);
    }
    if (columns == 0) return;
    const f32x2* at = angle + t * half;
    if constexpr (HALVES) {
      *reinterpret_cast<Eight<T>*>(&beside[wave][lane * 8]) = x;
      asm volatile("" ::: "memory");                                // a wave's LDS accesses are in order
      const T* row = &beside[wave][group * LPR * 8];
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
            if (c >= columns) continue;
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
        if (c0 + 2 * e >= columns) continue;
        const f32x2 cs = at[c0 / 2 + e];
        const float u = y[2 * e], v = y[2 * e + 1];
        y[2 * e] = fmaf(u, cs[0], -(v * cs[1]));
        y[2 * e + 1] = fmaf(v, cs[0], u * cs[1]);
      }
    }
  };
  auto most_of = [&](const float* y) __attribute__((always_inline)) {
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(y[e]) < INFINITY ? fabsf(y[e]) : 0.0f);
    return m;
  };

  // ---- jobs: rows of queries kRowsAtOnce at a time; keys, then values, a head at a time (of one token kRowsAtOnce heads)
  const int q_jobs = (n * a.heads[0] + kRowsAtOnce - 1) / kRowsAtOnce;
  const int each = n == 1 ? (p.kv_heads + kRowsAtOnce - 1) / kRowsAtOnce : p.kv_heads, jobs = q_jobs + (page < 0 ? 0 : 2 * each);
  for (int job = share * 4 + wave; job < jobs; job += shares * 4) {
    if (job < q_jobs) {
      const Kind& kind = a.kind[0];
      const int at = job * kRowsAtOnce + group, rows = n * a.heads[0], r = at < rows ? at : rows - 1;
      const int t = divided(r, by_heads), h = r - t * a.heads[0];
      float y[8];
      turned(kind, a.columns, t, fetch(kind, t, h), y);
      if (!live || at >= rows) continue;
      Eight<T> out;
#pragma unroll
      for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(out.w)[e] = from_f32<T>(none ? 0.0f : y[e]);
      store_eight(static_cast<T*>(kind.out) + (token0 + t) * kind.out_token + h * kind.out_head + c0, out);
      continue;
    }
    const bool v = job - q_jobs >= each;
    const Kind& kind = v ? a.kind[2] : a.kind[1];
    const int in_kind = job - q_jobs - (v ? each : 0), columns = v ? 0 : a.columns;
    const bool one = n == 1;
    const int at_head = one ? in_kind * kRowsAtOnce + group : in_kind, head = at_head < p.kv_heads ? at_head : p.kv_heads - 1;
    float largest = 0.0f;
    for (int t0 = 0; t0 < n; t0 += kRowsAtOnce) {
      const int t = one ? 0 : t0 + group < n ? t0 + group : n - 1;
      float y[8];
      turned(kind, columns, t, fetch(kind, t, head), y);
      largest = fmaxf(largest, most_of(y));
    }
    largest = one ? row_max<LPR>(largest) : wave_max(largest);
    uint8_t* scale = v ? sc.v + page * sc.v_page + head * sc.v_head + block * sc.v_block : sc.k + page * sc.k_page + head * sc.k_head + block * sc.k_block;
    uint8_t* codes = v ? static_cast<uint8_t*>(a.kind[2].out) + page * p.v_page + head * p.v_head
                       : static_cast<uint8_t*>(a.kind[1].out) + page * p.k_page + head * p.k_head;
    const int64_t slot_stride = v ? p.v_slot : p.k_slot;
    int e = exponent_of(largest);
    e = e < kLeastExponent<T> ? kLeastExponent<T> : e < kMostExponent<T> ? e : kMostExponent<T>;
    if (old > 0) {
      const int before = (int)*scale - 127;
      if (before > e) e = before < kMostExponent<T> ? before : kMostExponent<T>;
      if (e > before && live && at_head < p.kv_heads)               // older tokens' numbers again
        for (int s = one ? 0 : group; s < old; s += one ? 1 : kRowsAtOnce) {
          u32x2* c = reinterpret_cast<u32x2*>(codes + (slot - old + s) * slot_stride + c0);
          *c = codes_again(*c, before - e);
        }
    }
    const float by = power_of_two(-e), limit = e == kMostExponent<T> ? 240.0f : 448.0f;
    for (int t0 = 0; t0 < n; t0 += kRowsAtOnce) {
      const int t = one ? 0 : t0 + group < n ? t0 + group : n - 1;
      float y[8];
      turned(kind, columns, t, fetch(kind, t, head), y);
      if (live && at_head < p.kv_heads && (one || t0 + group < n))
        *reinterpret_cast<u32x2*>(codes + (slot + t) * slot_stride + c0) = to_codes(y, by, limit);
    }
    if (c0 == 0 && at_head < p.kv_heads && (one || group == 0)) *scale = (uint8_t)(e + 127);
  }
}

template <typename T, int LPR>
int launch_rows(const HeadArgs& a, const Pages& p, const Scales& sc, hipStream_t s) {
  const int64_t units = p.starts ? (int64_t)p.tokens / sc.block + 2 * ((int64_t)p.sequences + 2) : p.sequences;
  const int64_t rows_at_once = kWave / LPR, jobs = (a.heads[0] + rows_at_once - 1) / rows_at_once + 2 * (a.heads[1] + rows_at_once - 1) / rows_at_once;
  int64_t shares = 1024 / units, most = (jobs + 3) / 4;
  shares = shares < 1 ? 1 : shares < most ? shares : most;
  if (!grid_fits(units * shares, 256)) return HEXMI_ENOTSUP;
  const unsigned lds = (unsigned)((p.starts ? sc.block : 1) * (a.columns / 2) * sizeof(f32x2));
  const dim3 grid((unsigned)(units * shares));
  const Divider by_heads = divider(a.heads[0] > 0 ? a.heads[0] : 1);
  if (!a.halves || a.columns == 0)
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, false, false>), grid, dim3(256), lds, s, a, p, sc, (int)shares, by_heads);
  else if (a.columns % 16 == 0)
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, true, true>), grid, dim3(256), lds, s, a, p, sc, (int)shares, by_heads);
  else
    hipLaunchKernelGGL((scaled_rows_kernel<T, LPR, true, false>), grid, dim3(256), lds, s, a, p, sc, (int)shares, by_heads);
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
  if (!batch->k_pages || !batch->v_pages) return HEXMI_EINVAL;
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
