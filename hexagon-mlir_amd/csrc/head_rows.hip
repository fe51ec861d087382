// Rows of heads by position: the RMS norm of every query and key head and its rotation in one pass, and the same on the way into a
// paged cache, with the values beside them.
//
// A row x of dim columns becomes y = x / sqrt(mean(x^2) + eps) * w (where there is a weight), and pairs (a, b) of its leading columns
// become (a cos - b sin, b cos + a sin) at the angle position * inv_freq[i], all in fp32 but for the angle, which is a double until
// it is down to a quarter turn; one rounding at the end. Bound by HBM: every row is read once and written once.
#include "head_rows.h"

namespace hexmi {
namespace {

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

template <typename T, int LPR, bool HALVES, bool PIECES, bool PAGED>
__global__ __launch_bounds__(256, 4)
void head_rows_kernel(HeadArgs a, Pages p, int waves_per_token) {
  __shared__ __attribute__((aligned(16))) HeadRowsLds<T, LPR, HALVES> lds;
  head_rows_of<T, LPR, HALVES, PIECES, PAGED>(a, p, waves_per_token, blockIdx.x, gridDim.x, lds);
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
  const int64_t per_token = waves_per_token<LPR>(a), blocks = (a.tokens * per_token + 3) / 4;
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
