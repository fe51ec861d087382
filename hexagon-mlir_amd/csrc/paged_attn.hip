// Attention over a paged cache of keys and values (fp16 / bf16): new tokens of many sequences over the positions before them.
#include "flash_attn_tiles.h"
#include "paged.h"

namespace hexmi {
namespace {

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_token, q_head, out_token, out_head;
  const int32_t* shared;                       // the pages of the positions below `prefix`
  int prefix, heads, group, dim;               // group: query heads of a key head
  float scale;                                 // sm_scale * log2 e
};

// A wave takes a row (token, query head): its lanes are eight columns each of as many keys as fit side by side, every lane group with
// its own running maximum and sum, which meet at the end.
template <typename T>
__global__ __launch_bounds__(256)
void paged_rows_kernel(AttnArgs a, Pages p) {
  typedef T Piece __attribute__((ext_vector_type(8)));
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)p.tokens * a.heads) return;
  const int t = (int)(row / a.heads), h = (int)(row - (int64_t)t * a.heads), kvh = h / a.group;
  int b = t, keys;
  if (p.starts) b = sequence_of(p, t, lane);
  if (b < 0) keys = 0;
  else {
    const int behind = p.starts ? p.starts[b + 1] - t - 1 : 0;            // tokens of the sequence after this one
    const int64_t n = (int64_t)p.lengths[b] - behind;
    const int most = p.table_cols * p.page_size;
    keys = n < 0 ? 0 : n < most ? (int)n : most;
  }
  const int lpr = a.dim <= 64 ? 8 : a.dim <= 128 ? 16 : 32, groups = kWave / lpr, g = lane / lpr, d0 = lane % lpr * 8;
  const bool live = d0 < a.dim;
  const T* q_row = static_cast<const T*>(a.q) + t * a.q_token + h * a.q_head + d0;
  float q[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = live ? to_f32<T>(q_row[e]) * a.scale : 0.0f;
    o[e] = 0.0f;
  }
  for (int k0 = 0; k0 < keys; k0 += groups) {
    const int key = k0 + g;
    bool there = key < keys;
    int page = -1, column = 0;
    if (there) {
      column = divided(key, p.size);
      page = key < a.prefix ? a.shared[column] : p.table[b * p.table_row + column];
      there = page >= 0 && page < p.num_pages;
    }
    const int slot = key - column * p.page_size;
    Piece kp = {}, vp = {};
    if (there && live) {
      kp = *reinterpret_cast<const Piece*>(static_cast<const T*>(a.k) + page * p.k_page + kvh * p.k_head + slot * p.k_slot + d0);
      vp = *reinterpret_cast<const Piece*>(static_cast<const T*>(a.v) + page * p.v_page + kvh * p.v_head + slot * p.v_slot + d0);
    }
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(to_f32<T>(kp[e]), q[e], s);
    for (int x = 1; x < lpr; x *= 2) s += __shfl_xor(s, x);
    if (!there) continue;
    const float m_new = fmaxf(m, s), alpha = __builtin_amdgcn_exp2f(m - m_new), w = __builtin_amdgcn_exp2f(s - m_new);
    m = m_new;
    l = fmaf(l, alpha, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmaf(o[e], alpha, w * to_f32<T>(vp[e]));
  }
  float top = m;
  for (int x = lpr; x < kWave; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
  l *= f;
  for (int x = lpr; x < kWave; x *= 2) l += __shfl_xor(l, x);
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  T* out = static_cast<T*>(a.out) + t * a.out_token + h * a.out_head + d0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = o[e] * f;
    for (int x = lpr; x < kWave; x *= 2) v += __shfl_xor(v, x);
    if (g == 0 && live) out[e] = from_f32<T>(v * inv);
  }
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

extern "C" int64_t hexmi_paged_attention_workspace(const hexmi_paged_batch* batch, int64_t heads, int64_t shared) {
  (void)batch, (void)heads, (void)shared;
  return 0;
}

extern "C" int hexmi_paged_attention(const hexmi_head_rows* q, const hexmi_paged_batch* batch, const int32_t* shared_pages, int64_t shared,
                                     float sm_scale, int dtype, void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  if (!q || !batch || shared < 0 || (shared > 0 && !shared_pages) || workspace_bytes < 0) return HEXMI_EINVAL;
  int rc = check_batch(*batch);
  if (rc != HEXMI_OK) return rc;
  if (q->heads < 1 || q->heads % batch->kv_heads != 0 || !(sm_scale > 0.0f) || sm_scale > 3e38f || shared > batch->table_cols) return HEXMI_EINVAL;
  if ((dtype != HEXMI_F16 && dtype != HEXMI_BF16) || batch->dim % 8 != 0 || batch->dim > 256 || q->heads > 65535) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (batch->tokens * q->heads > 0x7fffffff) return HEXMI_ENOTSUP;
  if (!q->x || !q->out || !batch->k_pages || !batch->v_pages ||
      (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))))
    return HEXMI_EINVAL;
  const int64_t strides[] = {q->token, q->head, q->out_token, q->out_head, batch->k_page, batch->k_head, batch->k_slot, batch->v_page,
                             batch->v_head, batch->v_slot};
  for (int64_t s : strides)
    if (s % 8 != 0) return HEXMI_ENOTSUP;
  if (!aligned_to(q->x, 16) || !aligned_to(q->out, 16) || !aligned_to(batch->k_pages, 16) || !aligned_to(batch->v_pages, 16)) return HEXMI_ENOTSUP;
  const int64_t need = hexmi_paged_attention_workspace(batch, q->heads, shared);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return HEXMI_EINVAL;
  AttnArgs a = {q->x, batch->k_pages, batch->v_pages, q->out, q->token, q->head, q->out_token, q->out_head, shared_pages,
                (int)(shared * batch->page_size), (int)q->heads, (int)(q->heads / batch->kv_heads), (int)batch->dim, sm_scale * kLog2e};
  const Pages p = pages_of(*batch);
  hipStream_t s = as_stream(stream);
  begin_call();
  const unsigned blocks = (unsigned)((batch->tokens * q->heads + 3) / 4);
  if (dtype == HEXMI_F16) hipLaunchKernelGGL((paged_rows_kernel<f16>), dim3(blocks), dim3(256), 0, s, a, p);
  else hipLaunchKernelGGL((paged_rows_kernel<bf16>), dim3(blocks), dim3(256), 0, s, a, p);
  return launch_status();
}
