// The pages of a cache: rows that go on from others' with their last page copied (fork), and the pages in use moved to the front (compact).
// Copies, bound by HBM; what is in use is found from the table, so nothing is counted beside it.
// 256 rows from 64 parents, pages of 256 x 8 heads of 128 in 8 bits, 22 us (135 MB); 21880 pages of 16 x 8 heads of 128 of which 40 % are free 159 us
// (688 MB, 4.9 TB/s but for the launches that number them); four rows or 486 small pages are bound by one and two launches (5.6, 9.4 us).
#include "paged.h"

namespace hexmi {
namespace {

// Keys (or values) as bytes: strides in bytes, `row` bytes of a head at a slot, copied in pieces of `piece` bytes (16, or what divides all)
struct Side {
  char* pages;
  int64_t page, head, slot;
};
struct CopyArgs {
  Side side[2];
  uint8_t* scales[2];
  int64_t scale_page[2], scale_head[2], scale_block[2];
  int block;                                   // 0: none
  Divider by_block;
  int pieces;                                  // of a row
};

// pieces first, first + step, .. of all of the first `slots` slots of page `from` to page `to`, in the order of memory: heads within slots or slots
// within heads, what stands side by side as one run. Four are on their way at a time.
template <typename Piece>
__device__ __forceinline__ void copy_rows(const Side& side, int from, int to, int heads, int slots, int pieces, int first, int step) {
  const bool slots_inside = side.slot < side.head;
  const int64_t row = pieces * (int64_t)sizeof(Piece), inner_stride = slots_inside ? side.slot : side.head, outer_stride = slots_inside ? side.head : side.slot;
  const int inner = slots_inside ? slots : heads, all = heads * slots * pieces;
  const bool runs = inner_stride == row;
  const int run = runs ? inner * pieces : pieces;
  const char* src = side.pages + from * side.page;
  char* dst = side.pages + to * side.page;
  constexpr int kAtOnce = 4;
  for (int i0 = first; i0 < all; i0 += kAtOnce * step) {
    Piece x[kAtOnce];
    int64_t at[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * step, o = i / run;
      at[u] = (runs ? o * outer_stride : o / inner * outer_stride + o % inner * inner_stride) + (i - o * run) * (int64_t)sizeof(Piece);
      if (i < all) x[u] = *reinterpret_cast<const Piece*>(src + at[u]);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
      if (i0 + u * step < all) *reinterpret_cast<Piece*>(dst + at[u]) = x[u];
  }
}
__device__ __forceinline__ void copy_scales(const CopyArgs& c, int side, int from, int to, int heads, int blocks, int first, int step) {
  uint8_t* s = c.scales[side];
  for (int i = first; i < heads * blocks; i += step) {
    const int h = i / blocks, j = i - h * blocks;
    const int64_t at = h * c.scale_head[side] + j * c.scale_block[side];
    s[to * c.scale_page[side] + at] = s[from * c.scale_page[side] + at];
  }
}

// Workgroup (row, share): a share of the row's copies, keys and values, and of its entries of the table.
template <typename Piece>
__global__ __launch_bounds__(256)
void fork_kernel(CopyArgs c, Pages p, const int32_t* parents, const int32_t* pages, int32_t* table_out, int64_t table_out_row, int32_t* lengths_out,
                 int shares) {
  const int row = blockIdx.x / shares, share = blockIdx.x - row * shares;
  const int parent = parents[row], page = pages[row];
  const bool is = parent >= 0 && parent < p.sequences;
  const int length = is ? p.lengths[parent] : 0, there = is ? length_of(p, parent) : 0;
  const int column = divided(there, p.size), filled = there - column * p.page_size;
  const int32_t* table = p.table + (is ? parent : 0) * p.table_row;
  int last = -1;
  if (is && column < p.table_cols && filled > 0) last = table[column];
  const bool last_is = last >= 0 && last < p.num_pages;
  const bool takes = is && page >= 0 && page < p.num_pages && column < p.table_cols && (filled == 0 || last_is);
  for (int i = share * 256 + threadIdx.x; i < p.table_cols; i += shares * 256)
    table_out[row * table_out_row + i] = takes && i == column ? page : is ? table[i] : -1;
  if (share == 0 && threadIdx.x == 0) lengths_out[row] = length;
  if (!takes || filled == 0 || page == last) return;
  const int first = share * 256 + threadIdx.x, step = shares * 256;
  for (int side = 0; side < 2; ++side) {
    copy_rows<Piece>(c.side[side], last, page, p.kv_heads, filled, c.pieces, first, step);
    if (c.block) copy_scales(c, side, last, page, p.kv_heads, divided(filled + c.block - 1, c.by_block), first, step);
  }
}

// ---- compact: mark (a bit a page), number what is to go and where to, move and rename. Few entries and pages go to one workgroup, and two
// launches do.
constexpr int kFewEntries = 8192, kFewWords = 8192;
constexpr int kMovePieces = 1024;              // of a page, a workgroup at a time
struct CompactSpace {
  uint32_t* marks;                             // [words]
  int32_t *renamed, *sources, *targets;        // [pages]
  int32_t* moves;                              // [1]
};
__host__ __device__ inline int64_t words_of(int64_t pages) { return (pages + 31) / 32; }

__global__ __launch_bounds__(256)
void clear_kernel(uint32_t* marks, int64_t words) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < words) marks[i] = 0;
}

struct View {
  int window, sinks;                           // window 0: all
  int ahead;                                   // positions past a length that count too
  const int32_t* shared_pages;                 // the first `shared` pages of every sequence, whatever the table says there
  int shared;
};
// the page that entry (b, column) of the table names, -1: none in use
__device__ __forceinline__ int used_page(const Pages& p, const View& w, int b, int column) {
  const int length = length_of(p, b);
  const int first = column * p.page_size;
  if (first - w.ahead >= length) return -1;
  if (w.window > 0 && first >= w.sinks && first + p.page_size <= length - w.window) return -1;
  const int page = column < w.shared ? w.shared_pages[column] : p.table[b * p.table_row + column];
  return page >= 0 && page < p.num_pages ? page : -1;
}
// entry i of the table, row by row
__device__ __forceinline__ int used_page(const Pages& p, const View& w, int64_t i) {
  const int b = (int)(i / p.table_cols);
  return used_page(p, w, b, (int)(i - (int64_t)b * p.table_cols));
}
// shared page i, in use in any case
__device__ __forceinline__ int shared_page(const Pages& p, const View& w, int i) {
  const int page = w.shared_pages[i];
  return page >= 0 && page < p.num_pages ? page : -1;
}
__global__ __launch_bounds__(256)
void mark_kernel(Pages p, View w, uint32_t* marks, int64_t entries) {
  auto mark = [&](int page) __attribute__((always_inline)) {
    if (page < 0) return;
    const uint32_t bit = 1u << page % 32;
    if (!(__hip_atomic_load(marks + page / 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) & bit)) atomicOr(marks + page / 32, bit);
  };
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t i = first; i < entries; i += step) mark(used_page(p, w, i));
  for (int64_t i = first; i < w.shared; i += step) mark(shared_page(p, w, (int)i));
}

// By a workgroup of 1024: how many pages are marked, which of them go where, and their new names. A thread takes a run of words, twice.
__device__ __forceinline__ void number_pages(const uint32_t* marks, const CompactSpace& s, int num_pages, int32_t* count) {
  __shared__ int sums[16], used_below, total;
  const int words = (int)words_of(num_pages), each = (words + 1023) / 1024;
  const int w0 = (int)threadIdx.x * each < words ? (int)threadIdx.x * each : words, w1 = w0 + each < words ? w0 + each : words;
  int n = 0;
  for (int w = w0; w < w1; ++w) n += __popc(marks[w]);
  // the sum over the threads before this one
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int up_to = n;
  for (int d = 1; d < kWave; d *= 2) {
    const int v = __shfl_up(up_to, d);
    if (lane >= d) up_to += v;
  }
  if (lane == kWave - 1) sums[wave] = up_to;
  __syncthreads();
  int before = up_to - n;
  for (int x = 0; x < wave; ++x) before += sums[x];
  if (threadIdx.x == 1023) total = before + n;
  if (threadIdx.x == 0) used_below = 0;
  __syncthreads();
  const int front = total;
  // used pages below `front`: the thread whose run holds it says
  if (front / 32 >= w0 && front / 32 < w1) {
    int below = before;
    for (int w = w0; w < front / 32; ++w) below += __popc(marks[w]);
    used_below = below + __popc(marks[front / 32] & ((1u << front % 32) - 1));
  } else if (threadIdx.x == 0 && front / 32 >= words) {
    used_below = total;                                             // all pages are in use
  }
  __syncthreads();
  const int moved = used_below, moves = front - moved;
  int used = before;
  for (int w = w0; w < w1; ++w) {
    const uint32_t word = marks[w];
    const int page0 = w * 32;
    // of a word's pages those below `front` that are free, and those from it on that are in use
    const uint32_t below = front >= page0 + 32 ? ~0u : front <= page0 ? 0u : (1u << (front - page0)) - 1;
    for (uint32_t free = ~word & below; free; free &= free - 1) {
      const int i = __ffs(free) - 1;
      s.targets[page0 + i - used - __popc(word & ((1u << i) - 1))] = page0 + i;
    }
    for (uint32_t go = word & ~below; go; go &= go - 1) {
      const int i = __ffs(go) - 1;
      s.sources[used + __popc(word & ((1u << i) - 1)) - moved] = page0 + i;
    }
    used += __popc(word);
  }
  if (threadIdx.x == 0) {
    *s.moves = moves;
    *count = front;
  }
  __syncthreads();                                                  // sources and targets are the workgroup's own
  for (int i = threadIdx.x; i < moves; i += 1024) s.renamed[s.sources[i]] = s.targets[i];
}
__global__ __launch_bounds__(1024)
void number_kernel(CompactSpace s, int num_pages, int32_t* count) { number_pages(s.marks, s, num_pages, count); }

// All of it by one workgroup, the marks in LDS.
__global__ __launch_bounds__(1024)
void mark_and_number_kernel(Pages p, View w, CompactSpace s, int32_t* count, int entries) {
  __shared__ uint32_t marks[kFewWords];
  const int words = (int)words_of(p.num_pages);
  for (int i = threadIdx.x; i < words; i += 1024) marks[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int i = threadIdx.x; i < entries; i += 1024) {
    const int page = used_page(p, w, i);
    if (page >= 0) atomicOr(marks + page / 32, 1u << page % 32);
  }
  for (int i = threadIdx.x; i < w.shared; i += 1024) {
    const int page = shared_page(p, w, i);
    if (page >= 0) atomicOr(marks + page / 32, 1u << page % 32);
  }
  __syncthreads();
  number_pages(marks, s, p.num_pages, count);
}

template <typename Piece>
__global__ __launch_bounds__(256)
void move_kernel(CopyArgs c, Pages p, View w, CompactSpace s, const int32_t* count, int32_t* table_out, int64_t table_out_row, int32_t* shared_out,
                 int64_t entries, int parts) {
  const int front = *count, moves = *s.moves;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)gridDim.x * 256) {
    const int b = (int)(i / p.table_cols), column = (int)(i - (int64_t)b * p.table_cols), page = used_page(p, w, b, column);
    table_out[b * table_out_row + column] = page >= front ? s.renamed[page] : page;
  }
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < w.shared; i += (int64_t)gridDim.x * 256) {
    const int page = shared_page(p, w, (int)i);
    shared_out[i] = page >= front ? s.renamed[page] : page;
  }
  for (int64_t i = blockIdx.x; i < 2 * (int64_t)moves * parts; i += gridDim.x) {
    const int64_t unit = i / parts;
    const int part = (int)(i - unit * parts), move = (int)(unit / 2), side = (int)(unit - 2 * (int64_t)move), from = s.sources[move], to = s.targets[move];
    copy_rows<Piece>(c.side[side], from, to, p.kv_heads, p.page_size, c.pieces, part * 256 + threadIdx.x, parts * 256);
    if (c.block) copy_scales(c, side, from, to, p.kv_heads, divided(p.page_size, c.by_block), part * 256 + threadIdx.x, parts * 256);
  }
}

// HEXMI_OK, or why a cache is refused; the copies' arguments and the bytes of their pieces. One row of a result is as good with any stride.
int check_cache(const hexmi_paged_batch* batch, const hexmi_paged_scales* scales, int dtype, int64_t rows_out, int64_t table_out_row, CopyArgs& c, int& piece) {
  if (!batch) return HEXMI_EINVAL;
  hexmi_paged_batch b = *batch;
  b.starts = nullptr;
  b.tokens = b.sequences;
  int rc = check_batch(b);
  if (rc == HEXMI_OK && scales) rc = check_scales(b, *scales);
  if (rc != HEXMI_OK) return rc;
  if (dtype != HEXMI_F16 && dtype != HEXMI_BF16) return HEXMI_ENOTSUP;
  if (!b.k_pages || !b.v_pages || (b.sequences > 0 && (!b.lengths || (b.table_cols > 0 && !b.page_table)))) return HEXMI_EINVAL;
  const int size = scales ? 1 : 2;
  if (b.dim > (1 << 20)) return HEXMI_ENOTSUP;
  if (rows_out > 1 && table_out_row < b.table_cols) return HEXMI_EINVAL;
  c = {};
  c.side[0] = {static_cast<char*>(b.k_pages), b.k_page * size, b.k_head * size, b.k_slot * size};
  c.side[1] = {static_cast<char*>(b.v_pages), b.v_page * size, b.v_head * size, b.v_slot * size};
  piece = 16;
  for (const Side& s : c.side)
    for (int64_t x : {(int64_t)reinterpret_cast<uintptr_t>(s.pages), s.page, s.head, s.slot, b.dim * size})
      while (x % piece != 0) piece /= 2;
  c.pieces = (int)(b.dim * size / piece);
  if (b.kv_heads * b.page_size > 0x3fffffff / c.pieces) return HEXMI_ENOTSUP;     // pieces of a page are counted in 32 bits
  if (scales) {
    c.scales[0] = scales->k_scales;
    c.scales[1] = scales->v_scales;
    c.scale_page[0] = scales->k_page, c.scale_head[0] = scales->k_head, c.scale_block[0] = scales->k_block;
    c.scale_page[1] = scales->v_page, c.scale_head[1] = scales->v_head, c.scale_block[1] = scales->v_block;
    c.block = (int)scales->block;
    c.by_block = divider(scales->block);
  }
  return HEXMI_OK;
}
// f of a piece's type
template <typename F> int with_piece(int piece, F&& f) {
  switch (piece) {
    case 16: return f(u32x4{});
    case 8: return f(u32x2{});
    case 4: return f(uint32_t{});
    case 2: return f(uint16_t{});
    default: return f(uint8_t{});
  }
}
CompactSpace space_of(void* workspace, int64_t pages) {
  CompactSpace s;
  s.marks = static_cast<uint32_t*>(workspace);
  s.renamed = reinterpret_cast<int32_t*>(s.marks + words_of(pages));
  s.sources = s.renamed + pages;
  s.targets = s.sources + pages;
  s.moves = s.targets + pages;
  return s;
}

}  // namespace
}  // namespace hexmi

using namespace hexmi;

extern "C" int hexmi_paged_fork(const hexmi_paged_batch* batch, const hexmi_paged_scales* scales, const int32_t* parents, const int32_t* pages,
                                int64_t rows, int32_t* table_out, int64_t table_out_row, int32_t* lengths_out, int dtype, hexmi_stream_t stream) {
  CopyArgs c;
  int piece;
  const int rc = check_cache(batch, scales, dtype, rows, table_out_row, c, piece);
  if (rc != HEXMI_OK) return rc;
  if (rows < 0) return HEXMI_EINVAL;
  if (rows == 0) return HEXMI_OK;
  if (!parents || !pages || !lengths_out || (batch->table_cols > 0 && !table_out)) return HEXMI_EINVAL;
  // a workgroup for some KiB of a full page, as many as the card holds at once
  const int64_t page_bytes = 2 * batch->kv_heads * batch->page_size * c.pieces * piece, most = (page_bytes + 8191) / 8192;
  int64_t shares = 2048 / rows;
  shares = shares < 1 ? 1 : shares < most ? shares : most;
  if (!grid_fits(rows * shares, 256)) return HEXMI_ENOTSUP;
  const Pages p = pages_of(*batch);
  begin_call();
  return with_piece(piece, [&](auto x) {
    hipLaunchKernelGGL((fork_kernel<decltype(x)>), dim3((unsigned)(rows * shares)), dim3(256), 0, as_stream(stream), c, p, parents, pages, table_out,
                       table_out_row, lengths_out, (int)shares);
    return launch_status();
  });
}

extern "C" int64_t hexmi_paged_compact_workspace(const hexmi_paged_batch* batch) {
  if (!batch || batch->num_pages < 1 || batch->num_pages > 0x7fffffff) return 0;
  return (words_of(batch->num_pages) + 3 * batch->num_pages + 1) * 4;
}

extern "C" int hexmi_paged_compact(const hexmi_paged_batch* batch, const hexmi_paged_scales* scales, int64_t window, int64_t sinks, int32_t* table_out,
                                   int64_t table_out_row, int32_t* count, int dtype, void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  return hexmi_paged_compact_ex(batch, scales, nullptr, 0, window, sinks, 0, table_out, table_out_row, nullptr, count, dtype, workspace, workspace_bytes,
                                stream);
}

extern "C" int hexmi_paged_compact_ex(const hexmi_paged_batch* batch, const hexmi_paged_scales* scales, const int32_t* shared_pages, int64_t shared,
                                      int64_t window, int64_t sinks, int64_t ahead, int32_t* table_out, int64_t table_out_row, int32_t* shared_out,
                                      int32_t* count, int dtype, void* workspace, int64_t workspace_bytes, hexmi_stream_t stream) {
  CopyArgs c;
  int piece;
  const int rc = check_cache(batch, scales, dtype, batch ? batch->sequences : 0, table_out_row, c, piece);
  if (rc != HEXMI_OK) return rc;
  if (window < 0 || sinks < 0 || ahead < 0 || !count || (batch->sequences * batch->table_cols > 0 && !table_out)) return HEXMI_EINVAL;
  if (shared < 0 || shared > batch->table_cols || (shared > 0 && (!shared_pages || !shared_out))) return HEXMI_EINVAL;
  if (window > 0 && shared > 0) return HEXMI_ENOTSUP;
  const int64_t entries = batch->sequences * batch->table_cols, all = entries + shared;
  if (!workspace || !aligned_to(workspace, 16) || workspace_bytes < hexmi_paged_compact_workspace(batch)) return HEXMI_EINVAL;
  const Pages p = pages_of(*batch);
  const CompactSpace space = space_of(workspace, batch->num_pages);
  const int64_t positions = batch->table_cols * batch->page_size;
  const View view = {window_of(window, sinks, positions), (int)(sinks < 0x7fffffff ? sinks : 0x7fffffff), (int)(ahead < positions ? ahead : positions),
                     shared_pages, (int)shared};
  const hipStream_t s = as_stream(stream);
  const int64_t words = words_of(batch->num_pages);
  auto blocks = [](int64_t n, int64_t most) { return dim3((unsigned)((n + 255) / 256 < most ? (n + 255) / 256 : most)); };
  begin_call();
  if (all <= kFewEntries && words <= kFewWords) {
    hipLaunchKernelGGL(mark_and_number_kernel, dim3(1), dim3(1024), 0, s, p, view, space, count, (int)entries);
  } else {
    hipLaunchKernelGGL(clear_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, space.marks, words);
    if (all > 0) hipLaunchKernelGGL(mark_kernel, blocks(all, 4096), dim3(256), 0, s, p, view, space.marks, entries);
    hipLaunchKernelGGL(number_kernel, dim3(1), dim3(1024), 0, s, space, (int)batch->num_pages, count);
  }
  // a workgroup for some KiB of a page; no more than half of the pages move
  const int64_t page_pieces = batch->kv_heads * batch->page_size * c.pieces, parts = (page_pieces + kMovePieces - 1) / kMovePieces;
  const int64_t units = batch->num_pages * parts > (all + 255) / 256 ? batch->num_pages * parts : (all + 255) / 256;
  return with_piece(piece, [&](auto x) {
    hipLaunchKernelGGL((move_kernel<decltype(x)>), dim3((unsigned)(units < 2048 ? units : 2048)), dim3(256), 0, s, c, p, view, space, count, table_out,
                       table_out_row, shared_out, entries, (int)parts);
    return launch_status();
  });
}
