// Tiles (paged_tile.h), which the matrix cores bind, and workers on sequences of one new token (paged_decode.h), which wait for memory, in one
// launch side by side: a decode step behind a prefix that all sequences share, whose sums paged_decode_join_kernel joins, and a batch of
// prompts and decode steps. 32 sequences x 200 keys behind 8192 (32 heads over 8, of 128): one launch after the other 37 us, this way 22, and
// 6 to join. 509 new tokens beside 15 sequences of one: 31 us with the join, all of them as tiles 41. Tiles come first in the grid: by turns
// with the workers one kind lands on half of the compute units (4 x 509 tokens 104 us, by turns in eights 141).
#include "paged_decode.h"
#include "paged_tile.h"

namespace hexmi {
namespace {

template <typename T, int D, int COLS, bool PADDED, typename Shape>
__global__ __launch_bounds__(Shape::kThreads, D == 256 ? 1 : D == 64 ? 3 : 2)
void paged_shared_decode_kernel(PagedAttnArgs a, Pages p, TileArgs tiles, DecodeArgs w, unsigned tile_grid) {
  constexpr int W = Shape::kThreads / kWave, kTileBytes = Shape::lds_elements(D) * 2, kDecodeBytes = W * decode_wave_bytes(D, COLS);
  __shared__ __attribute__((aligned(16))) char lds[kTileBytes > kDecodeBytes ? kTileBytes : kDecodeBytes];
  __shared__ union Statistics {
    float tile[2][Shape::kGroups][Shape::kRows];
    float worker[2][W][16];
  } ml;
  if (blockIdx.x < tile_grid)
    paged_tile<T, D, COLS, PADDED, Shape>(a, p, tiles, blockIdx.x, tile_grid, reinterpret_cast<T*>(lds), ml.tile[0], ml.tile[1]);
  else
    paged_decode_worker<T, D, COLS, PADDED, W>(a, p, w, blockIdx.x - tile_grid, lds, ml.worker[0], ml.worker[1]);
}

template <typename T>
int launch(const PagedAttnArgs& a, const Pages& p, const TileArgs& tiles, const DecodeArgs& w, unsigned workers, hipStream_t s) {
  const unsigned tile_grid = (unsigned)(((int64_t)tiles.shared_tiles * tiles.shared_splits + (int64_t)tiles.tiles * tiles.splits) * p.kv_heads);
  const unsigned grid = tile_grid + workers;
  auto launch = [&](auto width, auto shape) {
    typedef decltype(width) W;
    typedef decltype(shape) Shape;
    hipLaunchKernelGGL((paged_shared_decode_kernel<T, W::D, W::COLS, W::PADDED, Shape>), dim3(grid), dim3(Shape::kThreads), 0, s, a, p, tiles,
                       w, tile_grid);
    return launch_status();
  };
  return tiles.deep ? with_width<128>(a.dim, [&](auto width) { return launch(width, DeepTile{}); })
                    : with_width<256>(a.dim, [&](auto width) { return launch(width, WideTile{}); });
}

}  // namespace

int paged_shared_decode(const PagedAttnArgs& a, const Pages& p, const TileArgs& tiles, const DecodeArgs& w, unsigned grid, int dtype,
                        hipStream_t s) {
  return dtype == HEXMI_F16 ? launch<f16>(a, p, tiles, w, grid, s) : launch<bf16>(a, p, tiles, w, grid, s);
}

}  // namespace hexmi
