// disco_residual_f32_f16.hip -- join kernels for a float stream and _Float16 blocks (disco_residual.h).
#define DISCO_RESIDUAL_KERNELS
#include "disco_residual.h"

DISCO_RESIDUAL_PAIR(kPairF32F16, float, _Float16)
