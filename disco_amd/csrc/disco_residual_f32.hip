// disco_residual_f32.hip -- join kernels for a float stream and float blocks (disco_residual.h).
#define DISCO_RESIDUAL_KERNELS
#include "disco_residual.h"

DISCO_RESIDUAL_PAIR(kPairF32, float, float)
