// Attention over pages of any size (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(PAGES, false, NO_CODES)
