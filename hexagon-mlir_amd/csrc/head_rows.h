// What the kernels that norm and turn rows of heads share (head_rows.hip, paged_scaled.hip): their arguments and what they refuse, eight columns
// of a row, the norm's factor.
#pragma once
#include "paged.h"

namespace hexmi {
namespace {

constexpr int kMaxDim = 512;

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
// 1 / sqrt(mean)
__device__ __forceinline__ float rms_scale(float mean) {
  const bool tiny = mean < 0x1p-100f;                               // the root's instruction takes no subnormal numbers
  mean = tiny ? mean * 0x1p60f : mean;
  const float r = __builtin_amdgcn_rsqf(mean);
  const float scale = r == 0.0f ? 0.0f : r * fmaf(-0.5f * mean * r, r, 1.5f);    // one Newton step; an infinite mean stays 0
  return tiny ? scale * 0x1p30f : scale;
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
