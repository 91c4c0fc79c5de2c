// dgnn_gemm_bf16.hip -- the matrix product of dgnn_gemm.h for one element type.
#include "dgnn_gemm.h"

int dgnn::gemm_bf16(const dgnn::Gemm& g) { return gemm_typed<__bf16>(g); }
