// Attention over the 4-bit paged cache, head dim 64.
#include "int4_attn.cuh"

namespace akv {

int int4_attn_64(const Int4AttnParams& p, int nt, cudaStream_t st) { return attn_dispatch<64>(p, nt, st); }

}  // namespace akv
