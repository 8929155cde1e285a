// Attention kernels for f16 tensors.
#include "dptm_attn_short.h"

DPTM_ATTN_DEFINE(f16, _Float16)
