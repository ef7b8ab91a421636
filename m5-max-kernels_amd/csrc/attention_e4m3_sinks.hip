// Attention over pages of a multiple of 16 keys that hold E4M3 codes, window and first keys (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(PAGES16, true, E4M3)
