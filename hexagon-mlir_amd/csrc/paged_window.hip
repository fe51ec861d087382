// Attention over a cache in 16 bits within a window: tiles, decode workers and both in one launch.
#include "paged_shared.h"

namespace hexmi {
template int launch_paged_tiles<Windowed>(const PagedAttnArgs&, const Pages&, const TileArgs&, int, hipStream_t);
template int launch_paged_workers<Windowed>(const PagedAttnArgs&, const Pages&, const DecodeArgs&, unsigned, int, hipStream_t);
template int launch_paged_shared<Windowed>(const PagedAttnArgs&, const Pages&, const TileArgs&, const DecodeArgs&, unsigned, int, hipStream_t);
}  // namespace hexmi
