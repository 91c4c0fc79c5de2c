// dgnn_gemm_f16.hip -- the matrix product of dgnn_gemm.h for one element type.
#include "dgnn_gemm.h"

int dgnn::gemm_f16(const dgnn::Gemm& g) { return gemm_typed<_Float16>(g); }
