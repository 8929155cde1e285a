// Attention kernels for f32 tensors.
#include "dptm_attn_short.h"

DPTM_ATTN_DEFINE(f32, float)
