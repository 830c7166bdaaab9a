// The int8 linear's tiles with f16 results.
#include "kq_int8_dense.h"

hipError_t kq::int8::dense_f16(const DenseArgs& g, int grid, hipStream_t st) { return dense<KQ_DT_F16>(g, grid, st); }
