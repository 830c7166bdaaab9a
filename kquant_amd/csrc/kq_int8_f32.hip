// The int8 linear's tiles with f32 results.
#include "kq_int8_dense.h"

hipError_t kq::int8::dense_f32(const DenseArgs& g, int grid, hipStream_t st) { return dense<KQ_DT_F32>(g, grid, st); }
