// disco_residual_f16.hip -- join kernels for a _Float16 stream and _Float16 blocks (disco_residual.h).
#define DISCO_RESIDUAL_KERNELS
#include "disco_residual.h"

DISCO_RESIDUAL_PAIR(kPairF16, _Float16, _Float16)
