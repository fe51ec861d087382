// Attention over a cache in 8 bits, within a window or not: tiles, decode workers and both in one launch.
#include "paged_shared.h"

namespace hexmi {
template int launch_paged_tiles<Scaled>(const PagedAttnArgs&, const Pages&, const TileArgs&, int, hipStream_t);
template int launch_paged_workers<Scaled>(const PagedAttnArgs&, const Pages&, const DecodeArgs&, unsigned, int, hipStream_t);
template int launch_paged_shared<Scaled>(const PagedAttnArgs&, const Pages&, const TileArgs&, const DecodeArgs&, unsigned, int, hipStream_t);
}  // namespace hexmi
