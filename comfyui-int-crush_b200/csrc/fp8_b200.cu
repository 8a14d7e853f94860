// Translation unit of the 8-bit floating point linear: block quantisation, the
// product, the group norm in front of it, and their entry points.
#include "ic_common.cuh"
#include "quant_fp8.cu"
#include "gemm_fp8.cu"
#include "group_norm.cu"
#include "abi_fp8.cu"
