// The layer norm's kernels of rows with a dropout in front of the residual sum.
#define HIPRESS_NORM_DROPOUT
#include "layer_norm.cu"
