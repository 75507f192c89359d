// disco_residual_bf16.hip -- join kernels for a __bf16 stream and __bf16 blocks (disco_residual.h).
#define DISCO_RESIDUAL_KERNELS
#include "disco_residual.h"

DISCO_RESIDUAL_PAIR(kPairBF16, __bf16, __bf16)
