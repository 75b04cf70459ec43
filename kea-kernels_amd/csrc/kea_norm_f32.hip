// kea_block_norm on streams of float elements.
#define KEA_NORM_STREAM float
#include "kea_norm_inst.h"
