// Chunk attention over the 4-bit paged cache: argument checks, workspace, launches.
#include "int4_chunk.cuh"

using namespace akv;

namespace {

int chunk_rows(int head_dim) { return head_dim == 256 ? 128 : 256; }  // query rows of a unit

// workspace: the units' meta records, sums, parts
struct ChunkWs {
  size_t ml, part, bytes;
};
ChunkWs chunk_ws(int head_dim) {
  ChunkWs w{};
  const size_t rows = 2 * static_cast<size_t>(kChunkSMs) * chunk_rows(head_dim);
  w.ml = kChunkSMs * sizeof(int4);
  w.part = w.ml + rows * sizeof(float2);
  w.bytes = w.part + rows * head_dim * sizeof(float);
  return w;
}

}  // namespace

extern "C" size_t akv_int4_chunk_workspace_bytes(int head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  return chunk_ws(head_dim).bytes;
}

extern "C" int akv_int4_chunk_attention(const akv_int4_attention_args* a, void* stream) {
  if (!a) return AKV_ERR_NULL;
  const akv_int4_cache* c = a->cache;
  const int rc = int4_check(c);
  if (rc) return rc;
  if (a->dtype != AKV_FP16 && a->dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (a->R < 0 || a->M < 0 || a->Hq <= 0 || a->Hq % c->kv_heads) return AKV_ERR_SHAPE;
  if (a->R == 0 || a->M == 0) return AKV_OK;
  if (!a->q || !a->out || !a->workspace) return AKV_ERR_NULL;
  if (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) & 1) ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 15))
    return AKV_ERR_ALIGN;
  const ChunkWs w = chunk_ws(c->head_dim);
  if (a->workspace_bytes < w.bytes) return AKV_ERR_WORKSPACE;
  if (a->Hq / c->kv_heads > kChunkRep) return AKV_ERR_UNSUPPORTED;
  const int64_t q_rows = static_cast<int64_t>(a->M) * (a->Hq / c->kv_heads);
  const int64_t tiles = (q_rows + chunk_rows(c->head_dim) - 1) / chunk_rows(c->head_dim);
  if (tiles > kChunkEntries) return AKV_ERR_UNSUPPORTED;  // more query rows than one launch lists
  // rows of a launch: its entries, their units and their token tiles are counted in 32 bits
  int64_t rows = kChunkEntries / tiles;
  if (rows > kChunkRowsMax) rows = kChunkRowsMax;
  const int64_t row_tiles = tiles * (static_cast<int64_t>(c->max_blocks) + kChunkSetup) * c->kv_heads;
  if (rows > INT32_MAX / 2 / row_tiles) rows = INT32_MAX / 2 / row_tiles;
  if (rows == 0) return AKV_ERR_UNSUPPORTED;
  ChunkParams p{};
  p.c = *c;
  p.rows = a->rows;
  p.n_new = a->n_new;
  p.M = a->M;
  p.Hq = a->Hq;
  p.tiles = static_cast<int>(tiles);
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_sr = a->q_sr; p.q_sh = a->q_sh; p.q_sm = a->q_sm;
  p.scale = a->sm_scale;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_sr = a->o_sr; p.o_sh = a->o_sh; p.o_sm = a->o_sm;
  p.lse = a->lse;
  p.bf16 = a->dtype == AKV_BF16;
  p.q16 = rows_aligned16(a->q, a->q_sr, a->q_sh, a->q_sm);
  p.o16 = rows_aligned16(a->out, a->o_sr, a->o_sh, a->o_sm);
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.meta = reinterpret_cast<int4*>(ws);
  p.ml = reinterpret_cast<float2*>(ws + w.ml);
  p.part = reinterpret_cast<float*>(ws + w.part);
  p.rep_inv = 0xFFFFFFFFu / static_cast<uint32_t>(a->Hq / c->kv_heads) + 1;
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int64_t r = 0; r < a->R; r += rows) {
    p.row0 = static_cast<int>(r);
    p.R = static_cast<int>(a->R - r < rows ? a->R - r : rows);
    const int e = c->head_dim == 64 ? int4_chunk_64(p, st)
                  : c->head_dim == 128 ? int4_chunk_128(p, st) : int4_chunk_256(p, st);
    if (e) return e;
  }
  return AKV_OK;
}
