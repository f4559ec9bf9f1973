// attn_paged.cuh for bf16 queries.
#include "attn_paged.cuh"

B200_PAGED_TENSOR_CORE(__nv_bfloat16)
