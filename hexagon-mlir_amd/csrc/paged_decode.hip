// Attention of one new token a sequence over the pages of its sequence (fp16 / bf16): a decode step of a batch.
// The workers are in paged_decode.h; here is what is launched, and the join of the units that several share.
#include "paged_decode.h"

namespace hexmi {
namespace {

// The units that several workers share: block (w, row) takes the one that worker w began. With join_all every unit is joined with the
// prefix's sums: block (unit, row).
template <typename T>
__global__ __launch_bounds__(256)
void paged_decode_join_kernel(PagedAttnArgs a, Pages p, DecodeArgs w) {
  __shared__ float o_lds[8][256 + 4];
  __shared__ float m_lds[8], l_lds[8];
  const int units = p.kv_heads * w.row_tiles, r = blockIdx.y;
  int b, u, w0 = 0, w1 = 0;
  if (w.join_all) {
    b = blockIdx.x / units;
    u = blockIdx.x - b * units;
    if (w.workers) {
      const int lane = threadIdx.x % kWave;
      const Dealt dealt = {a.view, a.scales.k ? kExtraBlocks : 0};
      const BlockList list = block_list<kWaves>(p, a.prefix, dealt, lane);
      int before = 0;
      for (int x = lane; x < b; x += kWave) before += x < kWave ? list.blocks : blocks_of<kWaves>(p, x, a.prefix, dealt);
      const int blocks = blocks_at<kWaves>(list, p, a.prefix, dealt, b), total = list.all * units;
      const int first = of_last_lane(sum_up_to(before)) * units + u * blocks;
      w0 = worker_of(total, w.workers, first);
      w1 = worker_of(total, w.workers, first + blocks - 1);
    }
  } else {
    const BegunUnit begun = w.begun[blockIdx.x];
    if (begun.last < 0) return;
    b = begun.sequence;
    u = begun.unit;
    w0 = blockIdx.x;
    w1 = begun.last;
  }
  const int kvh = u / w.row_tiles, row0 = (u - kvh * w.row_tiles) * 16;
  if (r >= a.group - row0) return;
  const int head = kvh * a.group + row0 + r;
  const int token = first_row(p, b);
  const int64_t row = (int64_t)token * a.heads + head;
  // eight groups of 32 threads take every eighth set of sums, a thread the columns d and, past 128, d + 128
  const int group = threadIdx.x / 32, d = threadIdx.x % 32 * 4;
  float top = -INFINITY, sum = 0.0f;
  f32x4 out[2] = {};
  // n sets of sums, this group's four at a time on their way: place(x, ml, o) says where set x stands
  auto take = [&](int n, auto place) __attribute__((always_inline)) {
    for (int x0 = group; x0 < n; x0 += 32) {
      float2 ml[4];
      f32x4 ox[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2* at_ml;
        const float* at_o;
        place(x0 + 8 * i < n ? x0 + 8 * i : x0, at_ml, at_o);
        ml[i] = *at_ml;
#pragma unroll
        for (int h = 0; h < 2; ++h) ox[i][h] = d + h * 128 < a.dim ? *reinterpret_cast<const f32x4*>(at_o + d + h * 128) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (x0 + 8 * i >= n || ml[i].y == 0.0f) continue;            // nothing there: its columns may be anything
        const float new_top = fmaxf(top, ml[i].x), f = __builtin_amdgcn_exp2f(ml[i].x - new_top), old = __builtin_amdgcn_exp2f(top - new_top);
        sum = fmaf(ml[i].y, f, sum * old);
        top = new_top;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[h][e] = fmaf(ox[i][h][e], f, out[h][e] * old);
      }
    }
  };
  if (w0 < w1)
    take(w1 - w0 + 1, [&](int x, const float2*& ml, const float*& o) {
      const int64_t slot = (int64_t)(w0 + x) * 2 + (x == 0 ? 1 : 0);
      ml = w.part_ml + slot * 16 + r;
      o = w.part_o + (slot * 16 + r) * a.dim;
    });
  if (w.join_all)
    take(w0 < w1 ? w.own : w.own + 1, [&](int x, const float2*& ml, const float*& o) {
      ml = w.sums.ml + x * w.sums.rows + row;
      o = w.sums.o + (x * w.sums.rows + row) * a.dim;
    });
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
  const float base = top == -INFINITY ? 0.0f : top;                 // no key: sums of 0; a NaN among the scores stays one
  for (int x = 0; x < 8; ++x) {
    const float f = __builtin_amdgcn_exp2f(m_lds[x] - base);
    l = fmaf(l_lds[x], f, l);
    o = fmaf(o_lds[x][c], f, o);
  }
  if (w.sums.slots && !w.join_all) {                                // a set of sums like a tile's
    const int64_t at = w.own * w.sums.rows + row;
    w.sums.o[at * a.dim + c] = o;
    if (c == 0) {
      w.sums.ml[at] = float2{top, l};
      for (int x = w.own + 1; x < w.sums.slots; ++x) w.sums.ml[x * w.sums.rows + row] = float2{-INFINITY, 0.0f};
    }
    return;
  }
  static_cast<T*>(a.out)[token * a.out_token + head * a.out_head + c] = from_f32<T>(l == 0.0f ? 0.0f : o / l);
}

template <typename T>
int launch(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, const DecodeArgs& w, const TileArgs& tiles, int dtype,
           hipStream_t s) {
  const unsigned grid = plan.workers ? plan.workers : (unsigned)((int64_t)p.sequences * p.kv_heads * plan.row_tiles);
  if (tiles.shared_splits || tiles.splits) {
    const int rc = with_kind(a, [&](auto kind) { return launch_paged_shared<decltype(kind)>(a, p, tiles, w, grid, dtype, s); });
    if (rc != HEXMI_OK || (!w.join_all && plan.workers < 2)) return rc;
    const dim3 joins(w.join_all ? (unsigned)((int64_t)p.sequences * p.kv_heads * plan.row_tiles) : plan.workers - 1, plan.rows);
    hipLaunchKernelGGL((paged_decode_join_kernel<T>), joins, dim3(256), 0, s, a, p, w);
    return launch_status();
  }
  const int rc = with_kind(a, [&](auto kind) { return launch_paged_workers<decltype(kind)>(a, p, w, grid, dtype, s); });
  if (rc != HEXMI_OK || plan.workers < 2) return rc;
  hipLaunchKernelGGL((paged_decode_join_kernel<T>), dim3(plan.workers - 1, plan.rows), dim3(256), 0, s, a, p, w);
  return launch_status();
}

}  // namespace

template int launch_paged_workers<Whole>(const PagedAttnArgs&, const Pages&, const DecodeArgs&, unsigned, int, hipStream_t);

PagedDecodePlan plan_paged_decode(const hexmi_paged_batch& b, int64_t heads, int64_t prefix, int64_t view) {
  const int64_t group = heads / b.kv_heads, tiles = (group + 15) / 16, units = b.sequences * b.kv_heads * tiles;
  const int64_t there = b.table_cols * b.page_size, most = (there < view ? there : view) - prefix, blocks = most > kBlockKeys ? (most + kBlockKeys - 1) / kBlockKeys : 1;
  const int rows = (int)(group < 16 ? group : 16);
  if (blocks <= 1) return {0, (int)tiles, rows};
  // A block each while they are fewer than the compute units; then four and more, so that a worker's sums are few beside its keys, on as
  // many workgroups as a compute unit holds. One and two a compute unit, heads of 128: 1 sequence x 16000 keys x 8 heads 21.9 / 24.5 us,
  // 3 x 5000 15.2 / 17.0; 128 x 500 58 / 52, 16 x 2048 x 32 97.7 / 93.5. Heads of 256, of which it holds one: 16 x 2048 x 8 56 / 60.
  // Beside tiles one: 16 sequences behind 4096 31.0 / 32.8, 15 beside 509 new tokens 30.8 / 31.4.
  const int64_t cus = hexmi_num_cus(), all = units * blocks, held = cus * (prefix > 0 || b.starts ? 1 : b.dim <= 96 ? 3 : b.dim <= 128 ? 2 : 1);
  const int64_t fours = all / 4 < cus ? cus : all / 4, workers = all < cus ? all : fours < held ? fours : held;
  return {(int)(workers < 1 ? 1 : workers), (int)tiles, rows};
}

int64_t paged_decode_workspace(const PagedDecodePlan& plan, int64_t dim) {
  return (int64_t)plan.workers * (2 * 16 * (dim * (int64_t)sizeof(float) + (int64_t)sizeof(float2)) + (int64_t)sizeof(BegunUnit));
}

int paged_decode(const PagedDecodePlan& plan, const PagedAttnArgs& a, const Pages& p, int dtype, void* workspace, const TileArgs& tiles,
                 hipStream_t s) {
  float* o = static_cast<float*>(workspace);
  float2* ml = reinterpret_cast<float2*>(o + (int64_t)plan.workers * 2 * 16 * a.dim);
  const DecodeArgs w = {o, ml, reinterpret_cast<BegunUnit*>(ml + (int64_t)plan.workers * 2 * 16), plan.workers,
                        plan.row_tiles, tiles.sums, tiles.shared_splits, p.starts == nullptr && tiles.shared_splits > 0};
  return dtype == HEXMI_F16 ? launch<f16>(plan, a, p, w, tiles, dtype, s) : launch<bf16>(plan, a, p, w, tiles, dtype, s);
}

}  // namespace hexmi
