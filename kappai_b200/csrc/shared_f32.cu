// Attention behind a shared prefix with rows, keys and values in float32: shared.cu's kernels.
#define SH_F32
#include "shared.cu"
