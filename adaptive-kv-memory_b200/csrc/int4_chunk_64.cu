// Chunk attention over the 4-bit paged cache, head dim 64.
#include "int4_chunk.cuh"

namespace akv {
int int4_chunk_64(const ChunkParams& P, cudaStream_t st) { return chunk_dispatch<64>(P, st); }
}  // namespace akv
