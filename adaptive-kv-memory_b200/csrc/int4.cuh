// Shared pieces of the 4-bit paged cache: record layout, argument checks,
// row and page lookup, element conversion.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"

namespace akv {

// Byte offsets of one (page, KV head) record; akv_int4_layout_init and the
// kernels' compile-time offsets both come from here.
struct Int4Layout {
  int kc, vc, kp, vp, bytes;
};

__host__ __device__ constexpr Int4Layout int4_layout(int D, int G) {
  Int4Layout r{};
  r.kc = 0;
  r.vc = kBlockTokens * D / 2;
  r.kp = 2 * r.vc;
  r.vp = r.kp + kBlockTokens * G * 4;
  r.bytes = r.vp + kBlockTokens * G * 4;
  return r;
}

inline bool int4_shape_ok(int D, int group) {
  return (D == 64 || D == 128 || D == 256) && group > 0 && (group == D || group == D / 2 || group == D / 4);
}

inline int int4_check(const akv_int4_cache* c) {
  if (!c || !c->pool || !c->table || !c->lens) return AKV_ERR_NULL;
  if (!int4_shape_ok(c->head_dim, c->group)) return AKV_ERR_SHAPE;
  if (c->n_pages <= 0 || c->max_seqs <= 0 || c->max_blocks <= 0 || c->kv_heads <= 0 ||
      c->max_blocks > INT32_MAX / kBlockTokens || c->table_stride < c->max_blocks)
    return AKV_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(c->pool) | static_cast<uintptr_t>(c->page_stride) |
       static_cast<uintptr_t>(c->head_stride)) & 15)
    return AKV_ERR_ALIGN;
  return AKV_OK;
}

// One call row: its sequence, the tokens it holds and how many of them are new.
struct Int4Row {
  int seq, len, n_new;  // seq -1: a bad row number
};

AKV_DEV Int4Row int4_row(const akv_int4_cache& c, const int32_t* rows, const int32_t* n_new, int i, int M,
                         int* status) {
  Int4Row r;
  r.seq = rows ? __ldg(rows + i) : i;
  if (static_cast<unsigned>(r.seq) >= static_cast<unsigned>(c.max_seqs)) {
    set_status(status, AKV_ERR_SHAPE);
    return Int4Row{-1, 0, 0};
  }
  const int cap = c.max_blocks * kBlockTokens;
  r.len = __ldg(c.lens + r.seq);
  if (r.len < 0 || r.len > cap) {
    set_status(status, AKV_ERR_SHAPE);
    r.len = r.len < 0 ? 0 : cap;
  }
  const int n = n_new ? __ldg(n_new + i) : M;
  r.n_new = n < 0 ? 0 : (n > M ? M : n);
  return r;
}

// ---------------------------------------------------------------- elements
template <bool BF>
AKV_DEV float elem_to_float(uint16_t u) {
  if constexpr (BF) return __uint_as_float(static_cast<uint32_t>(u) << 16);
  return __half2float(__ushort_as_half(u));
}

template <bool BF>
AKV_DEV uint16_t float_to_elem(float x) {
  if constexpr (BF) return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  return __half_as_ushort(__float2half_rn(x));
}

template <bool BF>
AKV_DEV uint32_t pack_elems(float lo, float hi) {
  if constexpr (BF) {
    __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&p);
  }
  return pack_h2(lo, hi);
}

// element pointer, each stride and the row all on a 16-byte boundary
inline bool rows_aligned16(const void* p, int64_t a, int64_t b, int64_t c) {
  return ((reinterpret_cast<uintptr_t>(p) & 15) | ((a | b | c) & 7)) == 0;
}

}  // namespace akv
