// Attention kernels for f16 tensors.
#include "dptm_attn_grad.h"

DPTM_ATTN_DEFINE(f16, _Float16)
