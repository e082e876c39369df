// Attention over the 4-bit paged cache, head dim 256.
#include "int4_attn.cuh"

namespace akv {

int int4_attn_256(const Int4AttnParams& p, int nt, cudaStream_t st) { return attn_dispatch<256>(p, nt, st); }

}  // namespace akv
