// kea_block_norm on streams of _Float16 elements.
#define KEA_NORM_STREAM _Float16
#include "kea_norm_inst.h"
