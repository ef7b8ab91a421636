// Attention over pages of a multiple of 16 keys (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(PAGES16, false, NO_CODES)
