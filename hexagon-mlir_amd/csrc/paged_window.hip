// Attention over a cache in 16 bits within a window: tiles, decode workers and both in one launch.
#include "paged_shared.h"

namespace hexmi {
HEXMI_PAGED_KIND(, Windowed)
}  // namespace hexmi
