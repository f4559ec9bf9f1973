// attn_paged.cuh for f16 queries.
#include "attn_paged.cuh"

B200_PAGED_TENSOR_CORE(__half)
