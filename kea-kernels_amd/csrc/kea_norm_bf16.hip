// kea_block_norm on streams of __bf16 elements.
#define KEA_NORM_STREAM __bf16
#include "kea_norm_inst.h"
