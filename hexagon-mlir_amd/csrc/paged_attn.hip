// Attention over a paged cache of keys and values (fp16 / bf16): runs of new tokens of many sequences over the positions before them, and
// the prefix that all sequences share: what a call launches, the tiles of ragged batches (paged_tile.h) and the join of their sums.
#include "hexmi_calibrate.h"
#include "paged_tile.h"

namespace hexmi {
namespace {

template <typename T, int D, int COLS, bool PADDED, typename Shape>
__global__ __launch_bounds__(Shape::kThreads, D == 256 ? 1 : D == 64 ? 3 : 2)
void paged_tile_kernel(PagedAttnArgs a, Pages p, TileArgs w) {
  __shared__ __attribute__((aligned(16))) T lds[Shape::lds_elements(D)];
  __shared__ float m_lds[Shape::kGroups][Shape::kRows], l_lds[Shape::kGroups][Shape::kRows];
  paged_tile<T, D, COLS, PADDED, Shape>(a, p, w, blockIdx.x, gridDim.x, lds, m_lds, l_lds);
}

// A row's sums of all slots (at most 32) joined: 32 threads a row, a thread the columns d and, past 128, d + 128.
template <typename T>
__global__ __launch_bounds__(256)
void paged_join_kernel(PagedAttnArgs a, RowSums sums) {
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= sums.rows) return;
  const int d = threadIdx.x % 32 * 4;
  // lane x of the 32 has slot x's maximum and sum, and all four slots' columns are asked for at once
  constexpr int kSlots = 4;
  const int lane = threadIdx.x % kWave, own = lane % 32;
  const float2 ml = own < sums.slots ? sums.ml[own * sums.rows + row] : float2{-INFINITY, 0.0f};
  float top = ml.y != 0.0f ? ml.x : -INFINITY;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  const float f = ml.y != 0.0f ? __builtin_amdgcn_exp2f(ml.x - top) : 0.0f;      // NaN in a part makes it NaN
  float sum = ml.y * f;
#pragma unroll
  for (int x = 1; x < 32; x *= 2) sum += __shfl_xor(sum, x);
  f32x4 out[2] = {};
  for (int x0 = 0; x0 < sums.slots; x0 += kSlots) {
    f32x4 o[kSlots][2];
    float fx[kSlots];
#pragma unroll
    for (int x = 0; x < kSlots; ++x) {
      fx[x] = __shfl(f, (lane & 32) + x0 + x);                      // 0: nothing there, and its columns are not read
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        o[x][h] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (fx[x] != 0.0f && d + h * 128 < a.dim)
          o[x][h] = *reinterpret_cast<const f32x4*>(sums.o + ((x0 + x) * sums.rows + row) * a.dim + d + h * 128);
      }
    }
#pragma unroll
    for (int x = 0; x < kSlots; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[h][e] = fmaf(o[x][h][e], fx[x], out[h][e]);
  }
  const int token = (int)(row / a.heads), head = (int)(row - (int64_t)token * a.heads);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T* to = static_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (d + h * 128 < a.dim) store4o<T>(to + d + h * 128, out[h][0] * inv, out[h][1] * inv, out[h][2] * inv, out[h][3] * inv);
}

template <typename T>
int launch_tiles(const PagedAttnArgs& a, const Pages& p, const TileArgs& w, hipStream_t s) {
  const unsigned grid = (unsigned)(((int64_t)w.tiles * w.splits + (int64_t)w.shared_tiles * w.shared_splits) * p.kv_heads);
  auto launch = [&](auto width, auto shape) {
    typedef decltype(width) W;
    typedef decltype(shape) Shape;
    hipLaunchKernelGGL((paged_tile_kernel<T, W::D, W::COLS, W::PADDED, Shape>), dim3(grid), dim3(Shape::kThreads), 0, s, a, p, w);
    return launch_status();
  };
  return w.deep ? with_width<128>(a.dim, [&](auto width) { return launch(width, DeepTile{}); })
                : with_width<256>(a.dim, [&](auto width) { return launch(width, WideTile{}); });
}

// What a call launches: the prefix's tiles (prefix_splits 0: none), then one token a sequence (decode) or tiles of the sequences' own keys
// (splits), then the join of the tiles' sums.
struct Plan {
  bool decode, deep, workers;                  // one token a sequence; DeepTile; sequences of one new token apart
  int prefix_tiles, prefix_splits, splits;
  int64_t tiles;
  PagedDecodePlan one;
  int64_t rows, sum_bytes, decode_bytes;
  int slots() const { return prefix_splits == 0 && (decode || splits == 1) ? 0 : prefix_splits + (decode ? 1 : splits); }
};
// Parts of the keys for `units` tiles: `wanted` workgroups, no part below `least` keys. A row has 32 slots for the sums of its parts, of the
// prefix and its own together.
int parts_of(int64_t units, int64_t keys, int64_t wanted, int64_t least, int64_t limit) {
  const int64_t most = keys / least < limit ? keys / least : limit, parts = wanted / units < most ? wanted / units : most;
  return parts > 1 ? (int)parts : 1;
}
// Lengths are on the GPU, so a plan takes the table's width for them, and its rules were measured with tables no wider than the longest
// sequence. As wide / 8192 columns of 16, 32 heads of 128 over 8, us: one prompt of 40 tokens 7.6 / 14.1, of 400 14.6 / 22.6, of 1000 26.9 / 37.2 (parts
// that nothing fills, and their join), of 2000 54.9 / 54.8; 64 decoding behind 99 10.5 / 12.7; one behind 999, 64 behind 99 .. 16383, 509
// tokens beside 15 single ones and 4 x 4096 are level.
Plan plan_of(const hexmi_paged_batch& b, int64_t heads, int64_t shared) {
  Plan plan = {};
  const int64_t group = heads / b.kv_heads, prefix = shared * b.page_size, rows = b.tokens * group, cus = hexmi_num_cus();
  const int64_t own = b.table_cols * b.page_size - prefix;
  plan.decode = b.starts == nullptr;
  plan.rows = b.tokens * heads;
  const int64_t wide = (rows + WideTile::kRows - 1) / WideTile::kRows * b.kv_heads;
  // Tiles of 64 rows, two groups on the keys, where those of 128 would be fewer than the compute units, and up to half as many again over few
  // keys: 64 / 128 rows, 32 heads of 128 over 8, us: 100 tokens 9.4 / 10.4, 400 14.9 / 17.4, 8 x 4 behind 1000 .. 3000 24.7 / 27.2, 509 behind
  // 2046 beside 15 single ones 31 / 49 (alone 46 / 43.5), 1000 26 / 31, 1400 37 / 39.5; but 1800 53 / 50, 32 x 1 .. 300 behind up to 4000
  // 159 / 144: there what a block's keys are worth in rows counts.
  plan.deep = !plan.decode && b.dim <= 128 && (wide < cus || (wide < cus * 3 / 2 && own <= 2048));
  // Sequences of one new token to workers, where some may be: 509 tokens beside 15 single ones 31 us, as tiles 41; the launch with both costs a
  // batch without any 1.5 (8 x 4 tokens).
  plan.workers = plan.decode || b.sequences > 1 || b.tokens == 1;
  const int64_t tile_rows = plan.deep ? DeepTile::kRows : WideTile::kRows, full = (rows + tile_rows - 1) / tile_rows;
  // As many workgroups as the card holds at once (heads of 256, one and two a compute unit: 500 behind 3000 101 / 116 us; heads of 64, two and
  // three: 2 x 700 behind 3000 60 / 51), and no part below 512 keys, which a join costs: 256 / 512 / 1024, us: 1000 tokens of 128 columns
  // 37 / 31 / 31, of 256 67 / 60 / 60, 100 behind 1500 - / 22 / 33.
  const int64_t wanted = (b.dim <= 64 ? 3 : b.dim <= 128 ? 2 : 1) * cus, least = 512;
  if (shared > 0) {
    // Behind a prefix there is a join in any case. Its parts may be of 256 keys in ragged batches (256 / 512: 4 x 20 tokens behind 992
    // 19 / 28 us, 16 x 1 .. 40 behind 3008 of 64 columns 32 / 30); of 128 in a decode step (128 / 256 / 512, us: 16 sequences behind 1008
    // 18.6 / 21 / 34, 32 behind 4000 20.3 / 21.1 / 25.7, of 256 columns 28 / 32 / 43), as long as all rows have 16384 sets of sums to
    // join at most: 32 x 32 heads behind 8192 in 16 parts 27, in 31 29; 64 x 32 heads behind 2000 in 8 28, in 15 30.
    const int64_t rows_there = plan.rows > 0 ? plan.rows : 1, sets = 16384 / rows_there;
    plan.prefix_tiles = (int)full;
    plan.prefix_splits = parts_of(full * b.kv_heads, prefix, wanted, plan.decode ? 128 : 256, plan.decode ? (sets < 31 ? sets : 31) : 16);
  }
  if (plan.workers) {
    plan.one = plan_paged_decode(b, heads, prefix);
    plan.decode_bytes = (paged_decode_workspace(plan.one, b.dim) + 15) / 16 * 16;
  }
  if (!plan.decode) {
    plan.tiles = rows / tile_rows + b.sequences + 2;
    plan.splits = parts_of(full * b.kv_heads, own, wanted, least, 16);
  }
  plan.sum_bytes = plan.slots() * plan.rows * (b.dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2));
  return plan;
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

namespace {
int check(const hexmi_paged_batch& b, int64_t heads, int64_t shared) {
  const int rc = check_batch(b);
  if (rc != HEXMI_OK) return rc;
  if (heads < 1 || heads % b.kv_heads != 0 || shared < 0 || shared > b.table_cols) return HEXMI_EINVAL;
  if (b.dim % 8 != 0 || b.dim > 256 || heads > 65535) return HEXMI_ENOTSUP;
  // rows, the blocks of all sequences and heads, and a launch's threads stay below 2^31
  const int64_t group = heads / b.kv_heads, limit = 0x7fffffff, units = b.kv_heads * ((group + 15) / 16);
  const int64_t blocks = (b.table_cols * b.page_size + 127) / 128 + 1;
  if (b.tokens > limit / heads || b.sequences > limit / units / blocks) return HEXMI_ENOTSUP;
  if (!b.starts) return b.sequences <= limit / 256 / units ? HEXMI_OK : HEXMI_ENOTSUP;
  if (b.tokens == 0) return HEXMI_OK;          // nothing to launch: there is no plan of it (plan_of divides by the tiles)
  const Plan plan = plan_of(b, heads, shared);
  if (plan.slots() > 0 && plan.rows > limit / 32) return HEXMI_ENOTSUP;         // 32 threads a row join them
  const int64_t workers = b.sequences > limit / 1024 / units ? limit : b.sequences * units;
  return (plan.tiles * plan.splits + (int64_t)plan.prefix_tiles * plan.prefix_splits) * b.kv_heads + workers <= limit / 512 ? HEXMI_OK : HEXMI_ENOTSUP;
}
}  // namespace

extern "C" int64_t hexmi_paged_attention_workspace(const hexmi_paged_batch* batch, int64_t heads, int64_t shared) {
  if (!batch || check(*batch, heads, shared) != HEXMI_OK || batch->tokens == 0) return 0;
  const Plan plan = plan_of(*batch, heads, shared);
  return plan.decode_bytes + plan.sum_bytes;
}

extern "C" int hexmi_paged_attention(const hexmi_head_rows* q, const hexmi_paged_batch* batch, const int32_t* shared_pages, int64_t shared,
                                     float sm_scale, int dtype, void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  if (!q || !batch || (shared > 0 && !shared_pages) || workspace_bytes < 0) return HEXMI_EINVAL;
  int rc = check(*batch, q->heads, shared);
  if (rc != HEXMI_OK) return rc;
  if (!(sm_scale > 0.0f) || sm_scale > 2e38f) return HEXMI_EINVAL;
  if (dtype != HEXMI_F16 && dtype != HEXMI_BF16) return HEXMI_ENOTSUP;
  if (batch->tokens == 0) return HEXMI_OK;
  if (!q->x || !q->out || !batch->k_pages || !batch->v_pages ||
      (batch->sequences > 0 && (!batch->lengths || (batch->table_cols > 0 && !batch->page_table))))
    return HEXMI_EINVAL;
  const int64_t strides[] = {q->token, q->head, q->out_token, q->out_head, batch->k_page, batch->k_head, batch->k_slot, batch->v_page,
                             batch->v_head, batch->v_slot};
  for (int64_t s : strides)
    if (s % 8 != 0) return HEXMI_ENOTSUP;
  if (batch->k_slot < 0 || batch->k_slot > 1 << 26 || batch->v_slot < 0 || batch->v_slot > 1 << 26) return HEXMI_ENOTSUP;      // 32-bit offsets within a page
  if (!aligned_to(q->x, 16) || !aligned_to(q->out, 16) || !aligned_to(batch->k_pages, 16) || !aligned_to(batch->v_pages, 16)) return HEXMI_ENOTSUP;
  const Plan plan = plan_of(*batch, q->heads, shared);
  const int64_t need = plan.decode_bytes + plan.sum_bytes;
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16))) return HEXMI_EINVAL;
  const int64_t group = q->heads / batch->kv_heads;
  const PagedAttnArgs a = {q->x, batch->k_pages, batch->v_pages, q->out, q->token, q->head, q->out_token, q->out_head, shared_pages,
                           (int)(shared * batch->page_size), (int)q->heads, (int)group, (int)batch->dim, sm_scale * kLog2e, divider(group)};
  const Pages p = pages_of(*batch);
  float* o = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.decode_bytes);
  const RowSums sums = {o, reinterpret_cast<float2*>(o + plan.slots() * plan.rows * batch->dim), plan.rows, plan.slots()};
  hipStream_t s = as_stream(stream);
  begin_call();
  const TileArgs tiles = {plan.deep, plan.workers, plan.prefix_tiles, plan.prefix_splits, (int)plan.tiles, plan.splits, sums};
  rc = plan.workers ? paged_decode(plan.one, a, p, dtype, workspace, tiles, s)
       : dtype == HEXMI_F16 ? launch_tiles<f16>(a, p, tiles, s) : launch_tiles<bf16>(a, p, tiles, s);
  if (rc != HEXMI_OK || plan.decode || sums.slots == 0) return rc;
  const unsigned blocks = (unsigned)((plan.rows + 7) / 8);
  if (dtype == HEXMI_F16) hipLaunchKernelGGL((paged_join_kernel<f16>), dim3(blocks), dim3(256), 0, s, a, sums);
  else hipLaunchKernelGGL((paged_join_kernel<bf16>), dim3(blocks), dim3(256), 0, s, a, sums);
  return launch_status();
}

extern "C" int hexmi_paged_tile_column(int64_t dim, int64_t chunk) {
  if (dim < 8 || dim > 256 || dim % 8 != 0 || chunk < 0) return -1;
  return with_width<256>(dim, [&](auto width) {
    typedef decltype(width) W;
    return chunk < W::D / 8 ? copied_column<W::D, W::COLS, W::PADDED>((int)chunk * 8, (int)dim) : -1;
  });
}
