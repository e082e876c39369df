// Chunk attention over the 4-bit paged cache, head dim 256.
#include "int4_chunk.cuh"

namespace akv {
int int4_chunk_256(const ChunkParams& P, cudaStream_t st) { return chunk_dispatch<256>(P, st); }
}  // namespace akv
