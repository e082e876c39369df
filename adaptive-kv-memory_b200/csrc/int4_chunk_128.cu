// Chunk attention over the 4-bit paged cache, head dim 128.
#include "int4_chunk.cuh"

namespace akv {
int int4_chunk_128(const ChunkParams& P, cudaStream_t st) { return chunk_dispatch<128>(P, st); }
}  // namespace akv
