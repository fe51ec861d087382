// Attention over a cache in 8 bits, within a window or not: tiles, decode workers and both in one launch.
#include "paged_shared.h"

namespace hexmi {
HEXMI_PAGED_KIND(, Scaled)
}  // namespace hexmi
