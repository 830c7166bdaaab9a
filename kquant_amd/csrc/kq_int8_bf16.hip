// The int8 linear's tiles with bf16 results.
#include "kq_int8_dense.h"

hipError_t kq::int8::dense_bf16(const DenseArgs& g, int grid, hipStream_t st) { return dense<KQ_DT_BF16>(g, grid, st); }
