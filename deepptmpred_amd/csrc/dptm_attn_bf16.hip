// Attention kernels for bf16 tensors.
#include "dptm_attn_short.h"

DPTM_ATTN_DEFINE(bf16, __bf16)
