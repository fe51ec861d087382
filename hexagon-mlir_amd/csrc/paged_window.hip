// Attention over a cache in 16 bits within a window: tiles, decode workers and both in one launch.
// What is seen is walked as if it stood side by side, the rest is as without a window: decode of 32 sequences within 4096 + 4 keys, 32 heads over 8 of
// 128, 104 us (HBM, 5.2 TB/s); a prompt of 16001 tokens within 1024 + 4 336 us (instruction issue, a quarter of the blocks masked).
#include "paged_shared.h"

namespace hexmi {
HEXMI_PAGED_KIND(, Windowed)
}  // namespace hexmi
