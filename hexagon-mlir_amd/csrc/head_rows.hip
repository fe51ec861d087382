// Rows of heads by position: the RMS norm of every query and key head and its rotation in one pass, and the same on the way into a
// paged cache, with the values beside them.
//
// A row x of dim columns becomes y = x / sqrt(mean(x^2) + eps) * w (where there is a weight), and pairs (a, b) of its leading columns
// become (a cos - b sin, b cos + a sin) at the angle position * inv_freq[i], all in fp32 but for the angle, which is a double until
// it is down to a quarter turn; one rounding at the end. Bound by HBM: every row is read once and written once.
#include "paged.h"

namespace hexmi {
namespace {

constexpr int kMaxDim = 512;
// A token's rows are shared by several waves up to so many in all: what the card holds at once, four a SIMD. 2048 / 4096 / 8192, 40 heads of 128
// bf16, us: 256 tokens 6.1 / 5.7 / 5.7, 1000 10.7 / 10.5 / 13.1, 2000 15.4 / 13.7 / 16.4, 1500 into a cache 19.0 / 14.7 / 17.8.
constexpr int kWavesWanted = 4096;

// the three kinds of rows, in the order in which they are numbered: queries, keys, values
struct Kind {
  const void* x;
  void* out;
  const void* weight;
  int64_t token, head, out_token, out_head;
};
struct HeadArgs {
  Kind kind[3];
  int heads[3], rows;                          // rows of a token, all kinds
  const double* inv_freq;
  int columns, halves, dim;
  float eps;
  const void* positions;
  int positions_64, tokens;
};

// where row h of a token belongs: its kind and the head of that kind
__device__ __forceinline__ int kind_of(const HeadArgs& a, int& h) {
  if (h < a.heads[0]) return 0;
  h -= a.heads[0];
  if (h < a.heads[1]) return 1;
  h -= a.heads[1];
  return 2;
}

// The position of a token, and its page where it has one (page -1: none). PAGED: the batch says so (none: no sequence).
struct Place {
  int64_t position;
  int page, slot;
  bool none;
};
template <bool PAGED>
__device__ __forceinline__ Place place_of(const HeadArgs& a, const Pages& p, int t, int lane) {
  Place at = {0, -1, 0, false};
  if constexpr (!PAGED) {
    if (a.positions) at.position = a.positions_64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
  } else {
    int b = t, behind = 1;                     // the token stands `behind` places before the end of sequence b
    if (p.starts) {
      b = sequence_of(p, t, lane);
      at.none = b < 0;
      if (at.none) return at;
      behind = first_row(p, b + 1) - t;
    }
    const int64_t position = (int64_t)p.lengths[b] - behind;
    at.position = position;
    if (position < 0 || position >= (int64_t)p.table_cols * p.page_size) return at;
    const int column = divided((int)position, p.size), page = p.table[b * p.table_row + column];
    if (page < 0 || page >= p.num_pages) return at;
    at.page = page;
    at.slot = (int)position - column * p.page_size;
  }
  return at;
}

// Any even number of rotated columns, any dim up to kMaxDim, any alignment: a wave takes a row, a lane every 64th column and the
// column that it is paired with.
template <typename T, bool PAGED>
__global__ __launch_bounds__(256)
void head_rows_any_kernel(HeadArgs a, Pages p) {
  constexpr int N = kMaxDim / kWave;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t rows = (int64_t)a.tokens * a.rows;
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < rows; row += (int64_t)gridDim.x * 4) {
    const int t = (int)(row / a.rows);
    int h = (int)(row - (int64_t)t * a.rows);
    const int k = kind_of(a, h);
    const Kind& kind = a.kind[k];
    const Place at = place_of<PAGED>(a, p, t, lane);
    T* out = static_cast<T*>(kind.out);
    if (PAGED && k != 0) {
      if (at.page < 0) continue;
      out += k == 1 ? at.page * p.k_page + h * p.k_head + at.slot * p.k_slot : at.page * p.v_page + h * p.v_head + at.slot * p.v_slot;
    } else {
      out += t * kind.out_token + h * kind.out_head;
    }
    const T* x = static_cast<const T*>(kind.x) + t * kind.token + h * kind.head;
    const T* w = static_cast<const T*>(kind.weight);
    const int columns = k == 2 ? 0 : a.columns;
    T y[N];
    float scale = 1.0f;
    if (w) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = i * kWave + lane;
        const float v = c < a.dim ? to_f32<T>(x[c]) : 0.0f;
        sum = fmaf(v, v, sum);
      }
      scale = 1.0f / sqrtf(wave_sum(sum) / (float)a.dim + a.eps);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * kWave + lane;
      if (c >= a.dim) continue;
      float v = to_f32<T>(x[c]);
      if (w) v = v * scale * to_f32<T>(w[c]);
      if (c < columns) {
        const int half = columns / 2;
        const bool second = a.halves ? c >= half : c & 1;
        const int other = a.halves ? (second ? c - half : c + half) : c ^ 1, pair = a.halves ? (second ? other : c) : c / 2;
        float o = to_f32<T>(x[other]);
        if (w) o = o * scale * to_f32<T>(w[other]);
        float sn, cs;
        sincos_turns((double)at.position * a.inv_freq[pair] * 0.15915494309189533577, sn, cs);       // 1 / (2 pi)
        v = second ? fmaf(v, cs, o * sn) : fmaf(v, cs, -(o * sn));
      }
      if (PAGED && at.none) v = 0.0f;
      y[i] = from_f32<T>(v);
    }
    // all of a row is read before any of it is written: out may be x itself
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = i * kWave + lane;
      if (c < a.dim) out[c] = y[i];
    }
  }
}

// Eight columns of a row as they stand in memory.
template <typename T> struct alignas(16) Eight {
  static constexpr int kWords = 8 * (int)sizeof(T) / 4;
  uint32_t w[kWords];
};
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p) {
  Eight<T> r;
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords / 4; ++i)
    *reinterpret_cast<u32x4*>(r.w + 4 * i) = *(reinterpret_cast<const u32x4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_eight(T* p, const Eight<T>& r) {
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords / 4; ++i)
    reinterpret_cast<u32x4*>(p)[i] = *reinterpret_cast<const u32x4*>(r.w + 4 * i);
}
template <typename T>
__device__ __forceinline__ float column(const Eight<T>& r, int e) {
  return to_f32<T>(reinterpret_cast<const T*>(r.w)[e]);
}
// the sum over the LPR lanes of a row, in all of them
template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  float a, b;
  if constexpr (LPR >= 16) v += dpp_move<0x140>(v);
  if constexpr (LPR >= 32) {
    swap16(v, a, b);
    v = a + b;
  }
  if constexpr (LPR == 64) {
    swap32(v, a, b);
    v = a + b;
  }
  return v;
}

// Rows on 16-byte boundaries, dim a multiple of 8. LPR lanes take a row, eight columns each, and the 64 / LPR rows of a wave are of one
// token: its angles are worked out once and serve every head. The pair of a column is in the same lane (adjacent) or comes out of LDS
// (halves), in one piece where columns / 2 is a multiple of 8 (PIECES: a lane's columns are all of one half, or none turns). The next rows
// are asked for before these are worked on.
// What a launch is bound by: its latency up to a few hundred tokens (4 tokens x 40 heads of 128 4.9 us, 64 tokens into a cache 4.6), then the
// rows in flight: 8192 tokens x 40 heads of 128 bf16, normed and turned, 40 us (4.2 TB/s; a copy of that size 33). Measured there: an
// angle worked out by every lane that needs it 50 us, pointers and strides chosen by the lane 62, no row asked for ahead 49, two ahead 42,
// 16384 waves 46, five waves a SIMD with what spills 44, nontemporal stores 41, and loads 43 (into a cache, prompts of 8700 tokens: 51 plain, 49
// and 53).
template <typename T, int LPR, bool HALVES, bool PIECES, bool PAGED>
__global__ __launch_bounds__(256, 4)
void head_rows_kernel(HeadArgs a, Pages p, int waves_per_token) {
  constexpr int kRowsAtOnce = kWave / LPR, kAngles = HALVES ? 8 : 4;
  __shared__ __attribute__((aligned(16))) f32x2 angle[4][LPR * 4 + 4];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c0 = lane % LPR * 8, group = lane / LPR, half = a.columns / 2;
  const bool live = c0 < a.dim, turns = c0 < a.columns;
  __shared__ __attribute__((aligned(16))) T beside[HALVES ? 4 : 1][HALVES ? kWave * 8 : 8];
  auto other = [&](int c) __attribute__((always_inline)) { return c >= a.columns ? c : c < half ? c + half : c - half; };
  Eight<T> weight[2], other_weight[2];                              // of queries and keys, at these columns and at their pairs'
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (a.kind[k].weight) {
      weight[k] = {};
      if (live) weight[k] = load_eight(static_cast<const T*>(a.kind[k].weight) + c0);
      if (HALVES) {
        const T* w = static_cast<const T*>(a.kind[k].weight);
        other_weight[k] = {};
        if (PIECES && turns) other_weight[k] = load_eight(w + other(c0));
        if (!PIECES && turns) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c0 + e < a.dim) reinterpret_cast<T*>(other_weight[k].w)[e] = w[other(c0 + e)];
        }
      }
    }
  const int q_chunks = (a.heads[0] + kRowsAtOnce - 1) / kRowsAtOnce, k_chunks = (a.heads[1] + kRowsAtOnce - 1) / kRowsAtOnce;
  const int chunks = q_chunks + k_chunks + (a.heads[2] + kRowsAtOnce - 1) / kRowsAtOnce;
  const int64_t all = (int64_t)a.tokens * waves_per_token;
  for (int64_t at_wave = (int64_t)blockIdx.x * 4 + wave; at_wave < all; at_wave += (int64_t)gridDim.x * 4) {
    const int t = (int)(at_wave / waves_per_token), share = (int)(at_wave - (int64_t)t * waves_per_token);
    const Place at = place_of<PAGED>(a, p, t, lane);
    // every angle of the token once, a lane each, and from LDS to the lanes whose columns turn by it
    const int pairs = a.columns / 2;
    for (int i = lane; i < pairs; i += kWave) {
      float sn, cs;
      sincos_turns((double)at.position * a.inv_freq[i] * 0.15915494309189533577, sn, cs);      // 1 / (2 pi)
      angle[wave][i] = f32x2{cs, sn};
    }
    asm volatile("" ::: "memory");                                  // a wave's LDS accesses are in order
    float cs[kAngles], sn[kAngles];                                 // halves: the sign of the sine says which one of a pair
    if (turns) {
#pragma unroll
      for (int e = 0; e < kAngles; ++e) {
        const int c = PIECES ? c0 : c0 + e;
        const bool second = HALVES && c >= half;
        const int i = !HALVES ? c0 / 2 + e : PIECES ? (second ? c0 - half : c0) + e : c >= a.columns ? 0 : second ? c - half : c;
        const f32x2 v = angle[wave][i];                             // past the last pair: not used
        cs[e] = v[0];
        sn[e] = HALVES && !second ? -v[1] : v[1];
      }
    }
    asm volatile("" ::: "memory");
    // the chunk's kind is the wave's, so its pointers and strides are scalars
    auto kind_at = [&](int chunk, int& h) __attribute__((always_inline)) {
      const int k = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;
      h = (chunk - (k == 0 ? 0 : k == 1 ? q_chunks : q_chunks + k_chunks)) * kRowsAtOnce + group;
      return k;
    };
    auto fetch = [&](int chunk) __attribute__((always_inline)) {    // lanes without a row of it: the kind's last row
      int h;
      const int k = kind_at(chunk < chunks ? chunk : chunks - 1, h);
      const Kind& kind = a.kind[k];
      h = h < a.heads[k] ? h : a.heads[k] - 1;
      return load_eight(static_cast<const T*>(kind.x) + t * kind.token + h * kind.head + (live ? c0 : 0));
    };
    Eight<T> next = fetch(share);
    for (int chunk = share; chunk < chunks; chunk += waves_per_token) {
      int h;
      const int k = kind_at(chunk, h);
      const Kind& kind = a.kind[k];
      const bool is_row = live && h < a.heads[k];
      Eight<T> x = next;
      if (!live) x = {};
      next = fetch(chunk + waves_per_token);
      T* out = static_cast<T*>(kind.out);
      if (PAGED && k != 0) {
        if (at.page < 0) continue;
        out += k == 1 ? at.page * p.k_page + at.slot * p.k_slot + h * p.k_head : at.page * p.v_page + at.slot * p.v_slot + h * p.v_head;
      } else {
        out += t * kind.out_token + h * kind.out_head;
      }
      if (k == 2) {                                                 // values as they are
        if (is_row) store_eight(out + c0, x);
        continue;
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = column(x, e);
      Eight<T> pair_x = {};
      if constexpr (HALVES) {
        *reinterpret_cast<Eight<T>*>(&beside[wave][lane * 8]) = x;
        asm volatile("" ::: "memory");
        const T* row = &beside[wave][group * LPR * 8];
        if constexpr (PIECES) {
          if (turns) pair_x = *reinterpret_cast<const Eight<T>*>(row + other(c0));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(pair_x.w)[e] = row[turns ? other(c0 + e) : 0];
        }
        asm volatile("" ::: "memory");
      }
      float scale = 1.0f;
      const bool norm = kind.weight != nullptr;
      const Eight<T> wt = k == 0 ? weight[0] : weight[1], other_wt = k == 0 ? other_weight[0] : other_weight[1];
      if (norm) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(y[e], y[e], sum);
        float mean = fmaf(row_sum<LPR>(sum), 1.0f / (float)a.dim, a.eps);
        const bool tiny = mean < 0x1p-100f;                         // the root's instruction takes no subnormal numbers
        mean = tiny ? mean * 0x1p60f : mean;
        const float r = __builtin_amdgcn_rsqf(mean);
        scale = r == 0.0f ? 0.0f : r * fmaf(-0.5f * mean * r, r, 1.5f);          // one Newton step; an infinite mean stays 0
        scale = tiny ? scale * 0x1p30f : scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = y[e] * scale * column(wt, e);
      }
      if (turns) {
        if constexpr (HALVES) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float o = column(pair_x, e);
            if (norm) o = o * scale * column(other_wt, e);
            const float turned = fmaf(y[e], cs[e], o * sn[e]);
            y[e] = PIECES || c0 + e < a.columns ? turned : y[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (c0 + 2 * e >= a.columns) continue;
            const float u = y[2 * e], v = y[2 * e + 1];
            y[2 * e] = fmaf(u, cs[e], -(v * sn[e]));
            y[2 * e + 1] = fmaf(v, cs[e], u * sn[e]);
          }
        }
      }
      if (!is_row) continue;
      Eight<T> r;
#pragma unroll
      for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(r.w)[e] = from_f32<T>(PAGED && at.none ? 0.0f : y[e]);
      store_eight(out + c0, r);
    }
  }
}

// whether head_rows_kernel takes the rows
template <typename T, bool PAGED>
bool takes(const HeadArgs& a, const Pages& p) {
  constexpr int n = 16 / (int)sizeof(T);
  if (a.dim % 8 != 0) return false;
  for (int k = 0; k < 3; ++k) {
    if (a.heads[k] == 0) continue;
    const Kind& r = a.kind[k];
    if (!aligned_to(r.x, 16) || !aligned_to(r.out, 16) || !aligned_to(r.weight, 16) || r.token % n != 0 || r.head % n != 0) return false;
    if (PAGED && k != 0) continue;
    if (r.out_token % n != 0 || r.out_head % n != 0) return false;
  }
  if (PAGED)
    for (int64_t s : {p.k_page, p.k_head, p.k_slot, p.v_page, p.v_head, p.v_slot})
      if (s % n != 0) return false;
  return true;
}

template <typename T, int LPR, bool PAGED>
int launch_rows(const HeadArgs& a, const Pages& p, hipStream_t s) {
  constexpr int at_once = kWave / LPR;
  int64_t most = 0;                            // chunks of a token's rows
  for (int k = 0; k < 3; ++k) most += (a.heads[k] + at_once - 1) / at_once;
  const int64_t wanted = kWavesWanted / a.tokens, per_token = wanted < 1 ? 1 : wanted < most ? wanted : most;
  const int64_t blocks = (a.tokens * per_token + 3) / 4;
  const dim3 grid((unsigned)(blocks < (1 << 22) ? blocks : 1 << 22));
  if (!a.halves || a.columns == 0) hipLaunchKernelGGL((head_rows_kernel<T, LPR, false, false, PAGED>), grid, dim3(256), 0, s, a, p, (int)per_token);
  else if (a.columns % 16 == 0) hipLaunchKernelGGL((head_rows_kernel<T, LPR, true, true, PAGED>), grid, dim3(256), 0, s, a, p, (int)per_token);
  else hipLaunchKernelGGL((head_rows_kernel<T, LPR, true, false, PAGED>), grid, dim3(256), 0, s, a, p, (int)per_token);
  return launch_status();
}

template <typename T, bool PAGED>
int launch(const HeadArgs& a, const Pages& p, hipStream_t s) {
  if (takes<T, PAGED>(a, p))
    return a.dim <= 64 ? launch_rows<T, 8, PAGED>(a, p, s) : a.dim <= 128 ? launch_rows<T, 16, PAGED>(a, p, s)
         : a.dim <= 256 ? launch_rows<T, 32, PAGED>(a, p, s) : launch_rows<T, 64, PAGED>(a, p, s);
  const int64_t rows = (int64_t)a.tokens * a.rows, blocks = (rows + 3) / 4;
  hipLaunchKernelGGL((head_rows_any_kernel<T, PAGED>), dim3((unsigned)(blocks < (1 << 22) ? blocks : 1 << 22)), dim3(256), 0, s, a, p);
  return launch_status();
}

int take(HeadArgs& a, int k, const hexmi_head_rows* r, bool needs_out) {
  if (!r) return HEXMI_OK;
  if (r->heads < 1 || !r->x || (needs_out && !r->out)) return HEXMI_EINVAL;
  if (r->heads > 65535) return HEXMI_ENOTSUP;
  a.kind[k] = {r->x, r->out, r->weight, r->token, r->head, r->out_token, r->out_head};
  a.heads[k] = (int)r->heads;
  a.rows += (int)r->heads;
  return HEXMI_OK;
}

int turn(HeadArgs& a, const hexmi_rotation* r, int64_t dim) {
  if (!r || dim < 1 || r->columns < 0 || r->columns % 2 != 0 || r->columns > dim || (r->columns > 0 && !r->inv_freq) ||
      (r->pairs != HEXMI_PAIRS_ADJACENT && r->pairs != HEXMI_PAIRS_HALVES))
    return HEXMI_EINVAL;
  if (dim > kMaxDim) return HEXMI_ENOTSUP;
  a.inv_freq = r->inv_freq;
  a.columns = (int)r->columns;
  a.halves = r->pairs == HEXMI_PAIRS_HALVES;
  a.dim = (int)dim;
  a.eps = r->eps;
  return HEXMI_OK;
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

extern "C" int hexmi_qk_norm_rope(const hexmi_head_rows* q, const hexmi_head_rows* k, const hexmi_rotation* rotation,
                                  const void* positions, int positions_64, int64_t tokens, int64_t dim, int dtype,
                                  hexmi_stream_t stream) {
  if (!q || tokens < 0) return HEXMI_EINVAL;
  HeadArgs a = {};
  int rc = turn(a, rotation, dim);
  if (rc != HEXMI_OK) return rc;
  if (tokens == 0) return HEXMI_OK;
  if (tokens > 0x3fffffff) return HEXMI_ENOTSUP;
  if ((rc = take(a, 0, q, true)) != HEXMI_OK || (rc = take(a, 1, k, true)) != HEXMI_OK) return rc;
  if (a.columns > 0 && !positions) return HEXMI_EINVAL;
  a.positions = positions;
  a.positions_64 = positions_64;
  a.tokens = (int)tokens;
  begin_call();
  switch (dtype) {
    case HEXMI_F32: return launch<float, false>(a, Pages{}, as_stream(stream));
    case HEXMI_F16: return launch<f16, false>(a, Pages{}, as_stream(stream));
    case HEXMI_BF16: return launch<bf16, false>(a, Pages{}, as_stream(stream));
    default: return HEXMI_ENOTSUP;
  }
}

extern "C" int hexmi_paged_append(const hexmi_head_rows* k, const hexmi_head_rows* v, const hexmi_head_rows* q,
                                  const hexmi_rotation* rotation, const hexmi_paged_batch* batch, int dtype, hexmi_stream_t stream) {
  if (!k || !v || !batch) return HEXMI_EINVAL;
  int rc = check_batch(*batch);
  HeadArgs a = {};
  if (rc != HEXMI_OK || (rc = turn(a, rotation, batch->dim)) != HEXMI_OK) return rc;
  if (k->heads != batch->kv_heads || v->heads != batch->kv_heads) return HEXMI_EINVAL;
  if (dtype != HEXMI_F16 && dtype != HEXMI_BF16) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))) return HEXMI_EINVAL;
  if (!batch->k_pages || !batch->v_pages) return HEXMI_EINVAL;
  if ((rc = take(a, 0, q, true)) != HEXMI_OK || (rc = take(a, 1, k, false)) != HEXMI_OK || (rc = take(a, 2, v, false)) != HEXMI_OK) return rc;
  a.kind[1].out = batch->k_pages;
  a.kind[2].out = batch->v_pages;
  a.kind[2].weight = nullptr;
  a.tokens = (int)batch->tokens;
  begin_call();
  const Pages p = pages_of(*batch);
  return dtype == HEXMI_F16 ? launch<f16, true>(a, p, as_stream(stream)) : launch<bf16, true>(a, p, as_stream(stream));
}
