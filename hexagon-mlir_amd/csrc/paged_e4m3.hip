// Attention over a cache in 8 bits, within a window or not: tiles, decode workers and both in one launch.
// A number of e4m3 times its block's power of two is one of T, so keys and values are widened exactly (v_cvt_scalef32_pk_*_fp8, two numbers an
// instruction, the scale its operand) and the rest is as in 16 bits. Decode is bound by HBM (16 x 2048 x 32 heads of 128 54.3 us, 4.9 TB/s; 64
// sequences of 100 to 16384 over 8 heads 94), tiles by instruction issue (prompts of 4 x 4096, 32 heads over 8 of 128, bf16 612 us, fp16 656; in 16
// bits 589).
#include "paged_shared.h"

namespace hexmi {
HEXMI_PAGED_KIND(, Scaled)
}  // namespace hexmi
