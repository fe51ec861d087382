// Attention over a paged cache in 8 bits, or within a window: a wave takes a row (token, head) and goes through its keys one by one, four
// columns a lane, with the running maximum and sum of a softmax in fp32.
#include "paged.h"

namespace hexmi {
namespace {

struct RowArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_token, q_head, out_token, out_head;
  const int32_t* shared;
  int prefix, heads, group, dim, window, sinks, scaled;
  float scale;
};

template <typename T>
__device__ __forceinline__ f32x4 four(const void* base, int64_t at, int scaled, const uint8_t* exponent) {
  if (scaled) {
    const uint32_t c = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + at);
    const float f = __builtin_bit_cast(float, (uint32_t)*exponent << 23);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    return f32x4{lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f};
  }
  const T* x = static_cast<const T*>(base) + at;
  return f32x4{to_f32<T>(x[0]), to_f32<T>(x[1]), to_f32<T>(x[2]), to_f32<T>(x[3])};
}

template <typename T>
__global__ __launch_bounds__(256)
void row_attention_kernel(RowArgs a, Pages p, Scales sc) {
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)p.tokens * a.heads) return;
  const int token = (int)(row / a.heads), head = (int)(row - (int64_t)token * a.heads), kvh = head / a.group, c = lane * 4;
  const bool live = c < a.dim;
  const int b = p.starts ? sequence_of(p, token, lane) : token;
  int keys = 0;
  if (b >= 0) {
    const int64_t position = (int64_t)p.lengths[b] - (p.starts ? first_row(p, b + 1) - token : 1), most = (int64_t)p.table_cols * p.page_size;
    keys = position < 0 ? 0 : position + 1 < most ? (int)position + 1 : (int)most;
  }
  const T* q = static_cast<const T*>(a.q) + token * a.q_token + head * a.q_head + (live ? c : 0);
  f32x4 x = {to_f32<T>(q[0]), to_f32<T>(q[1]), to_f32<T>(q[2]), to_f32<T>(q[3])}, o = {};
  if (!live) x = f32x4{};
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < keys; ++j) {
    if (a.window > 0 && j >= a.sinks && j < keys - a.window) j = keys - a.window;
    const int column = divided(j, p.size), slot = j - column * p.page_size;
    const int page = j < a.prefix ? a.shared[column] : p.table[b * p.table_row + column];
    if (page < 0 || page >= p.num_pages) continue;
    const int block = a.scaled ? divided(slot, sc.by_block) : 0;
    const f32x4 k = four<T>(a.k, page * p.k_page + kvh * p.k_head + slot * p.k_slot + (live ? c : 0), a.scaled,
                            sc.k + page * sc.k_page + kvh * sc.k_head + block * sc.k_block);
    const float s = wave_sum(x[0] * k[0] + x[1] * k[1] + x[2] * k[2] + x[3] * k[3]) * a.scale;
    const f32x4 v = four<T>(a.v, page * p.v_page + kvh * p.v_head + slot * p.v_slot + (live ? c : 0), a.scaled,
                            sc.v + page * sc.v_page + kvh * sc.v_head + block * sc.v_block);
    const float top = fmaxf(m, s), f = __builtin_amdgcn_exp2f(m - top), w = __builtin_amdgcn_exp2f(s - top);
    l = fmaf(l, f, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], f, w * v[e]);
    m = top;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (live) store4<T>(static_cast<T*>(a.out) + token * a.out_token + head * a.out_head + c, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

extern "C" int64_t hexmi_paged_attention_ex_workspace(const hexmi_paged_batch* batch, int64_t heads, int64_t shared,
                                                      const hexmi_paged_scales* scales, int64_t window, int64_t sinks) {
  if (!batch || scales || window_of(window, sinks, batch->table_cols * batch->page_size)) return 0;
  return hexmi_paged_attention_workspace(batch, heads, shared);
}

extern "C" int hexmi_paged_attention_ex(const hexmi_head_rows* q, const hexmi_paged_batch* batch, const hexmi_paged_scales* scales,
                                        const int32_t* shared_pages, int64_t shared, int64_t window, int64_t sinks, float sm_scale, int dtype,
                                        void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  if (!q || !batch || window < 0 || sinks < 0 || (shared > 0 && !shared_pages)) return HEXMI_EINVAL;
  int rc = check_batch(*batch);
  if (rc != HEXMI_OK || (scales && (rc = check_scales(*batch, *scales)) != HEXMI_OK)) return rc;
  if (window > 0 && shared > 0) return HEXMI_ENOTSUP;
  const int seen = window_of(window, sinks, batch->table_cols * batch->page_size);
  if (!scales && !seen) return hexmi_paged_attention(q, batch, shared_pages, shared, sm_scale, dtype, workspace, workspace_bytes, stream);
  if (q->heads < 1 || q->heads % batch->kv_heads != 0 || shared < 0 || shared > batch->table_cols) return HEXMI_EINVAL;
  if (!(sm_scale > 0.0f) || sm_scale > 2e38f) return HEXMI_EINVAL;
  if ((dtype != HEXMI_F16 && dtype != HEXMI_BF16) || batch->dim % 8 != 0 || batch->dim > 256 || q->heads > 65535) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (!q->x || !q->out || !batch->k_pages || !batch->v_pages ||
      (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))))
    return HEXMI_EINVAL;
  const int64_t step = scales && batch->dim % 16 == 0 ? 16 : 8;
  for (int64_t s : {q->token, q->head, q->out_token, q->out_head})
    if (s % 8 != 0) return HEXMI_ENOTSUP;
  for (int64_t s : {batch->k_page, batch->k_head, batch->k_slot, batch->v_page, batch->v_head, batch->v_slot})
    if (s % step != 0) return HEXMI_ENOTSUP;
  if (batch->k_slot < 0 || batch->k_slot > 1 << 26 || batch->v_slot < 0 || batch->v_slot > 1 << 26) return HEXMI_ENOTSUP;
  const size_t boundary = scales ? step : 16;
  if (!aligned_to(q->x, 16) || !aligned_to(q->out, 16) || !aligned_to(batch->k_pages, boundary) || !aligned_to(batch->v_pages, boundary))
    return HEXMI_ENOTSUP;
  const RowArgs a = {q->x, batch->k_pages, batch->v_pages, q->out, q->token, q->head, q->out_token, q->out_head, shared_pages,
                     (int)(shared * batch->page_size), (int)q->heads, (int)(q->heads / batch->kv_heads), (int)batch->dim, seen,
                     (int)(seen ? sinks : 0), scales != nullptr, sm_scale * 1.44269504088896340736f};
  const int64_t blocks = (batch->tokens * q->heads + 3) / 4;
  if (!grid_fits(blocks, 256)) return HEXMI_ENOTSUP;
  const Pages p = pages_of(*batch);
  const Scales sc = scales ? scales_of(*scales) : Scales{};
  begin_call();
  if (dtype == HEXMI_F16) hipLaunchKernelGGL((row_attention_kernel<f16>), dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), a, p, sc);
  else hipLaunchKernelGGL((row_attention_kernel<bf16>), dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), a, p, sc);
  return launch_status();
}
