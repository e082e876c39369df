// Attention over the 4-bit paged cache: argument checks, workspace, launches.
#include "int4_attn.cuh"

using namespace akv;

namespace {

// call rows of one launch, and their units (row, row tile, KV head)
struct Plan {
  int nt, tiles, rows;
  bool fused;  // each unit's last CTA merges its parts: no second launch
  size_t meta, part;
};

Plan attn_plan(int R, int M, int Hq, int kv_heads, int D, int max_blocks) {
  Plan p{};
  const int q_rows = M * (Hq / kv_heads);
  p.nt = attn_nt(q_rows);
  p.tiles = (q_rows + 8 * p.nt - 1) / (8 * p.nt);
  p.rows = kAttnEntries / p.tiles;
  const int64_t row_pages = static_cast<int64_t>(p.tiles) * kv_heads * max_blocks;
  if (p.rows > INT32_MAX / row_pages) p.rows = static_cast<int>(INT32_MAX / row_pages);  // 0: too many
  // a counter for every unit, in a region of its own at the workspace's start
  const int64_t row_units = static_cast<int64_t>(p.tiles) * kv_heads;
  if (p.rows > kAttnUnits / row_units) p.rows = static_cast<int>(kAttnUnits / row_units);
  if (p.rows > R) p.rows = R;
  const size_t units = static_cast<size_t>(p.rows) * p.tiles * kv_heads;
  // the most CTAs that can share a unit, and the query rows each leaves there
  const int segs = max_blocks / kAttnMinPages + 2;
  const int q_rows_tile = q_rows < 8 * p.nt ? q_rows : 8 * p.nt;
  p.fused = static_cast<int64_t>(segs) * q_rows_tile <= kAttnFused;
  p.meta = (units * sizeof(int2) + 15) / 16 * 16;
  // a CTA and a unit meet at most once, and along the list of pages their
  // numbers' sum only grows: it is the slot of the partial result
  p.part = (units + kSMs * attn_occ(D, p.nt)) * 8 * p.nt * (D + 2) * sizeof(float);
  return p;
}

}  // namespace

extern "C" size_t akv_int4_attention_workspace_bytes(int R, int M, int Hq, int kv_heads, int head_dim, int max_blocks) {
  if (R < 0 || M < 0 || Hq <= 0 || kv_heads <= 0 || Hq % kv_heads || max_blocks <= 0) return 0;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
  if (R == 0 || M == 0) return 16;
  if (static_cast<int64_t>(M) * (Hq / kv_heads) > 8 * kAttnEntries) return 0;
  const Plan p = attn_plan(R, M, Hq, kv_heads, head_dim, max_blocks);
  if (p.rows == 0 || static_cast<int64_t>(R) * Hq * M > INT32_MAX) return 0;
  return kAttnUnits * sizeof(unsigned) + p.meta + p.part;
}

extern "C" int akv_int4_attention(const akv_int4_attention_args* a, void* stream) {
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
  const size_t need =
      akv_int4_attention_workspace_bytes(a->R, a->M, a->Hq, c->kv_heads, c->head_dim, c->max_blocks);
  if (need == 0) return AKV_ERR_UNSUPPORTED;  // more query rows than one launch lists
  if (a->workspace_bytes < need) return AKV_ERR_WORKSPACE;
  const Plan plan = attn_plan(a->R, a->M, a->Hq, c->kv_heads, c->head_dim, c->max_blocks);
  Int4AttnParams p{};
  p.c = *c;
  p.rows = a->rows;
  p.n_new = a->n_new;
  p.M = a->M;
  p.Hq = a->Hq;
  p.tiles = plan.tiles;
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_sr = a->q_sr; p.q_sh = a->q_sh; p.q_sm = a->q_sm;
  p.scale = a->sm_scale;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_sr = a->o_sr; p.o_sh = a->o_sh; p.o_sm = a->o_sm;
  p.out4 = ((reinterpret_cast<uintptr_t>(a->out) & 3) | ((a->o_sr | a->o_sh | a->o_sm) & 1)) == 0;
  p.lse = a->lse;
  p.bf16 = a->dtype == AKV_BF16;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.arrived = reinterpret_cast<unsigned*>(ws);
  ws += kAttnUnits * sizeof(unsigned);
  p.meta = plan.fused ? nullptr : reinterpret_cast<int2*>(ws);
  p.part = reinterpret_cast<float*>(ws + plan.meta);
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  for (int r = 0; r < a->R; r += plan.rows) {
    p.row0 = r;
    p.R = a->R - r < plan.rows ? a->R - r : plan.rows;
    const int e = c->head_dim == 64 ? int4_attn_64(p, plan.nt, st)
                  : c->head_dim == 128 ? int4_attn_128(p, plan.nt, st) : int4_attn_256(p, plan.nt, st);
    if (e) return e;
  }
  return AKV_OK;
}
