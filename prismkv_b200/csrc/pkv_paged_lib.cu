// pkv_paged_lib.cu -- the translation unit of the paged-cache kernels (they share one device error word).
#include "pkv_paged_attn.cu"
#include "pkv_paged_ops.cu"
#include "pkv_paged_api.cu"
