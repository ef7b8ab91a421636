// Attention over dense keys and values (attention_core.h).
#include "attention_core.h"

M5K_ATTENTION_UNIT(DENSE, false, NO_CODES)
