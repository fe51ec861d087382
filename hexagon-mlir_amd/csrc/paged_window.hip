// Attention over a cache in 16 bits within a window: tiles, decode workers and both in one launch.
// What is seen is walked as if it stood side by side, the rest is as without a window: decode of 32 sequences within 4096 + 4 keys, 32 heads over 8 of
// 128, 104 us (HBM, 5.2 TB/s); a prompt of 16001 tokens within 500, 1024 and 4096 (+ 4) 211, 340 and 1001 us: 13.8 for every block of 64 keys that
// all tiles walk (its products take 11 at the rate of a large matrix product), and 85 to 100 that are a tile's once: look-up, first copies, masked blocks, stores.
#include "paged_shared.h"

namespace hexmi {
HEXMI_PAGED_KIND(, Windowed)
}  // namespace hexmi
