// The tile kernels of the paged attention with P as two bf16 halves, built beside the others.
#define PAGED_HALVES
#include "paged_attention.hip"
