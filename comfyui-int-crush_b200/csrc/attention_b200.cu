// Translation unit of the attention-side operators: head norm + rotation,
// cross attention, many-request adapters, and their entry points.
#include "ic_common.cuh"
#include "qk_norm_rope.cu"
#include "lora_batched.cu"
#include "cross_attention_tc.cu"
#include "cross_attention.cu"
#include "abi_attention.cu"
