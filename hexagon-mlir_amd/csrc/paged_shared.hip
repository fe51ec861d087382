// Tiles and decode workers in one launch (paged_shared.h) over a cache in 16 bits.
#include "paged_shared.h"

namespace hexmi {
template int launch_paged_shared<Whole>(const PagedAttnArgs&, const Pages&, const TileArgs&, const DecodeArgs&, unsigned, int, hipStream_t);
}  // namespace hexmi
