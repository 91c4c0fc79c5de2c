// dgnn_gemm_f32.hip -- the matrix product of dgnn_gemm.h for one element type.
#include "dgnn_gemm.h"

int dgnn::gemm_f32(const dgnn::Gemm& g) { return gemm_typed<float>(g); }
