// pkv_lib.cu -- one translation unit for everything but the paged cache (its kernels share
// a device error word without relocatable device code).
#include "pkv_codec.cu"
#include "pkv_encode_tc.cu"
#include "pkv_attn.cu"
#include "pkv_scores.cu"
#include "pkv_api.cu"
#include "pkv_noalloc.cu"
