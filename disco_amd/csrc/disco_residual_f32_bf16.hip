// disco_residual_f32_bf16.hip -- join kernels for a float stream and __bf16 blocks (disco_residual.h).
#define DISCO_RESIDUAL_KERNELS
#include "disco_residual.h"

DISCO_RESIDUAL_PAIR(kPairF32BF16, float, __bf16)
