// Attention over dense keys and values, window and first keys (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(DENSE, true, NO_CODES)
