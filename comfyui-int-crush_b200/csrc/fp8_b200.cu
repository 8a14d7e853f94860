// Translation unit of the 8-bit floating point linear: block quantisation, the
// product, the group norm in front of it, and their entry points.
// The product hands a buffer over every 850 to 950 clocks: its waits poll without a
// suspend hint, from which waking up took longer (40 clocks more a block).
#define IC_WAIT_NOHINT
#include "ic_common.cuh"
#include "quant_fp8.cu"
#include "gemm_fp8.cu"
#include "group_norm.cu"
#include "abi_fp8.cu"
