// Attention over pages of any size, window and first keys (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(PAGES, true, NO_CODES)
