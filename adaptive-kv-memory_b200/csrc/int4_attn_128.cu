// Attention over the 4-bit paged cache, head dim 128.
#include "int4_attn.cuh"

namespace akv {

int int4_attn_128(const Int4AttnParams& p, int nt, cudaStream_t st) { return attn_dispatch<128>(p, nt, st); }

}  // namespace akv
