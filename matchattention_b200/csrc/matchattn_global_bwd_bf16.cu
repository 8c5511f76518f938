#include <cuda_bf16.h>
#include <cuda_fp16.h>
#define MATCHATTN_T __nv_bfloat16
#include "matchattn_global_bwd.inl"
