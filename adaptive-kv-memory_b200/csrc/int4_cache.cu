// Writing and reading back the 4-bit paged cache.
//
// Per group x_0..x_{g-1} of one token's row, in fp32:
//   z = fp16(min x), s = fp16((max x - z) / 15),
//   c = clamp(rint((x - z) / s), 0, 15) (0 where s is 0), value = c*s + z.
// Scale and zero are rounded to fp16 because they are stored so; the codes are
// chosen against the rounded pair, so the stored pair is the one that counts.
// Bound by memory: 2*D*2 bytes in and D + 8*G bytes out per token and head.
// One thread holds 8 channels (one 16-byte load, one 4-byte store of codes),
// D/8 threads a row; a group's min and max meet in log2(g/8) shuffles.
#include "int4.cuh"

namespace akv {

struct Int4Io {
  akv_int4_cache c;
  const int32_t* rows;
  const int32_t* n_new;
  const int32_t* start;
  int M;
  uint16_t* k;
  int64_t k_sr, k_sh, k_sm;
  uint16_t* v;
  int64_t v_sr, v_sh, v_sm;
  int aligned;  // rows on 16-byte boundaries: vector accesses
  int* status;
};

constexpr int kIoThreads = 256;

// x / s to the nearest float, for s an fp16 value and r the float nearest
// 1/s: one Newton step on the quotient leaves the correctly rounded result
// (Markstein), so ties in rint() fall as they do for the true division.
AKV_DEV float div_by(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-s, q, x), r, q);
}

template <bool BF>
__global__ void __launch_bounds__(kIoThreads) int4_append_kernel(Int4Io a) {
  const int D = a.c.head_dim, L = D / 8;
  const int i = blockIdx.y;
  const int64_t unit = (blockIdx.x * static_cast<int64_t>(kIoThreads) + threadIdx.x) / L;
  const int part = threadIdx.x % L;  // L divides the block
  const Int4Row row = int4_row(a.c, a.rows, a.n_new, i, a.M, a.status);
  const int H = a.c.kv_heads;
  const int m = static_cast<int>(unit / (2 * H));
  const int hk = static_cast<int>(unit % (2 * H));
  const int h = hk >> 1, is_v = hk & 1;
  const int pos = row.len - row.n_new + m;
  bool on = row.seq >= 0 && m < row.n_new && pos >= 0;
  int page = -1;
  if (on) {
    page = a.c.table[row.seq * a.c.table_stride + pos / kBlockTokens];
    if (page < 0 || page >= a.c.n_pages) {
      set_status(a.status, AKV_ERR_SHAPE);
      on = false;
    }
  }
  float x[8];
  if (on) {
    const uint16_t* src = is_v ? a.v + i * a.v_sr + h * a.v_sh + m * a.v_sm : a.k + i * a.k_sr + h * a.k_sh + m * a.k_sm;
    src += part * 8;
    uint16_t e[8];
    if (a.aligned) {
      *reinterpret_cast<uint4*>(e) = ldg_nc_v4(src);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = src[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = elem_to_float<BF>(e[j]);
      x[j] = f == f ? fminf(fmaxf(f, -65504.f), 65504.f) : 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = 0.f;
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) {
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  const int gl = a.c.group / 8;  // threads of a group
  for (int o = 1; o < gl; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
  }
  if (!on) return;
  const __half zh = __float2half_rn(lo);
  const float z = __half2float(zh);
  const __half sh = __float2half_rn(__fdiv_rn(__fsub_rn(hi, z), 15.f));
  const float s = __half2float(sh);
  const float r = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float q = s > 0.f ? rintf(div_by(__fsub_rn(x[j], z), s, r)) : 0.f;
    const uint32_t code = static_cast<uint32_t>(fminf(fmaxf(q, 0.f), 15.f));
    word |= code << ((j & 1 ? 0 : 4) + 8 * (j >> 1));
  }
  const int G = D / a.c.group;
  const int vc = kBlockTokens * D / 2;
  const int slot = pos % kBlockTokens;
  uint8_t* rec = a.c.pool + page * a.c.page_stride + h * a.c.head_stride;
  *reinterpret_cast<uint32_t*>(rec + is_v * vc + slot * (D / 2) + part * 4) = word;
  if (part % gl == 0) {
    const __half2 p = __halves2half2(sh, zh);
    *reinterpret_cast<__half2*>(rec + 2 * vc + is_v * kBlockTokens * G * 4 + (slot * G + part / gl) * 4) = p;
  }
}

template <bool BF>
__global__ void __launch_bounds__(kIoThreads) int4_read_kernel(Int4Io a) {
  const int D = a.c.head_dim, L = D / 8;
  const int i = blockIdx.y;
  const int64_t unit = (blockIdx.x * static_cast<int64_t>(kIoThreads) + threadIdx.x) / L;
  const int part = threadIdx.x % L;
  const int H = a.c.kv_heads;
  const int m = static_cast<int>(unit / (2 * H));
  if (m >= a.M) return;
  const int hk = static_cast<int>(unit % (2 * H));
  const int h = hk >> 1, is_v = hk & 1;
  const Int4Row row = int4_row(a.c, a.rows, a.n_new, i, a.M, a.status);
  const int64_t pos = a.start ? static_cast<int64_t>(a.start[i]) + m : static_cast<int64_t>(row.len) - row.n_new + m;
  const bool on = row.seq >= 0 && pos >= 0 && pos < row.len;
  uint32_t out[4] = {0u, 0u, 0u, 0u};
  if (on) {
    int page = a.c.table[row.seq * a.c.table_stride + pos / kBlockTokens];
    if (page < 0 || page >= a.c.n_pages) {
      set_status(a.status, AKV_ERR_SHAPE);
      page = 0;
    }
    const int G = D / a.c.group, vc = kBlockTokens * D / 2, slot = static_cast<int>(pos % kBlockTokens);
    const uint8_t* rec = a.c.pool + page * a.c.page_stride + h * a.c.head_stride;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(rec + is_v * vc + slot * (D / 2) + part * 4);
    const __half2 p = *reinterpret_cast<const __half2*>(rec + 2 * vc + is_v * kBlockTokens * G * 4 +
                                                        (slot * G + part * 8 / a.c.group) * 4);
    const float s = __low2float(p), z = __high2float(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float e = fmaf(static_cast<float>((word >> (8 * j + 4)) & 15u), s, z);
      float o = fmaf(static_cast<float>((word >> (8 * j)) & 15u), s, z);
      if constexpr (!BF) {  // 15 steps of a rounded-up scale can pass the largest fp16
        e = fminf(fmaxf(e, -65504.f), 65504.f);
        o = fminf(fmaxf(o, -65504.f), 65504.f);
      }
      out[j] = pack_elems<BF>(e, o);
    }
  }
  uint16_t* dst = is_v ? a.v + i * a.v_sr + h * a.v_sh + m * a.v_sm : a.k + i * a.k_sr + h * a.k_sh + m * a.k_sm;
  dst += part * 8;
  if (a.aligned) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) dst[j] = static_cast<uint16_t>(out[j / 2] >> (16 * (j & 1)));
  }
}

}  // namespace akv

using namespace akv;

extern "C" int akv_int4_layout_init(int head_dim, int group, akv_int4_layout* out) {
  if (!out) return AKV_ERR_NULL;
  if (!int4_shape_ok(head_dim, group)) return AKV_ERR_SHAPE;
  const Int4Layout l = int4_layout(head_dim, head_dim / group);
  *out = akv_int4_layout{head_dim, group, head_dim / group, l.kc, l.vc, l.kp, l.vp, l.bytes};
  return AKV_OK;
}

// shared argument checks and launch of append and read
template <class Launch>
static int int4_io(const akv_int4_cache* c, int R, int M, const void* k, int64_t k_sr, int64_t k_sh, int64_t k_sm,
                   const void* v, int64_t v_sr, int64_t v_sh, int64_t v_sm, int dtype, Int4Io& a, Launch launch) {
  const int rc = int4_check(c);
  if (rc) return rc;
  if (dtype != AKV_FP16 && dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (R < 0 || M < 0) return AKV_ERR_SHAPE;
  if (R == 0 || M == 0) return AKV_OK;
  if (!k || !v) return AKV_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1) return AKV_ERR_ALIGN;
  const int64_t threads = static_cast<int64_t>(M) * c->kv_heads * 2 * (c->head_dim / 8);
  const int64_t blocks = (threads + kIoThreads - 1) / kIoThreads;
  if (R > 65535 || blocks > INT32_MAX) return AKV_ERR_UNSUPPORTED;
  a.c = *c;
  a.M = M;
  a.k = static_cast<uint16_t*>(const_cast<void*>(k));
  a.k_sr = k_sr; a.k_sh = k_sh; a.k_sm = k_sm;
  a.v = static_cast<uint16_t*>(const_cast<void*>(v));
  a.v_sr = v_sr; a.v_sh = v_sh; a.v_sm = v_sm;
  a.aligned = rows_aligned16(k, k_sr, k_sh, k_sm) && rows_aligned16(v, v_sr, v_sh, v_sm);
  launch(dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(R)), a);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

extern "C" int akv_int4_append(const akv_int4_cache* c, const int32_t* rows, const int32_t* n_new, int R, int M,
                               const void* k, int64_t k_sr, int64_t k_sh, int64_t k_sm,
                               const void* v, int64_t v_sr, int64_t v_sh, int64_t v_sm, int dtype, int* status,
                               void* stream) {
  Int4Io a{};
  a.rows = rows;
  a.n_new = n_new;
  a.status = status;
  return int4_io(c, R, M, k, k_sr, k_sh, k_sm, v, v_sr, v_sh, v_sm, dtype, a, [&](dim3 grid, const Int4Io& p) {
    if (dtype == AKV_BF16)
      int4_append_kernel<true><<<grid, kIoThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    else
      int4_append_kernel<false><<<grid, kIoThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  });
}

extern "C" int akv_int4_read(const akv_int4_cache* c, const int32_t* rows, const int32_t* start, const int32_t* n_new,
                             int R, int N, void* k, int64_t k_sr, int64_t k_sh, int64_t k_sm,
                             void* v, int64_t v_sr, int64_t v_sh, int64_t v_sm, int dtype, int* status, void* stream) {
  Int4Io a{};
  a.rows = rows;
  a.n_new = n_new;
  a.start = start;
  a.status = status;
  return int4_io(c, R, N, k, k_sr, k_sh, k_sm, v, v_sr, v_sh, v_sm, dtype, a, [&](dim3 grid, const Int4Io& p) {
    if (dtype == AKV_BF16)
      int4_read_kernel<true><<<grid, kIoThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    else
      int4_read_kernel<false><<<grid, kIoThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  });
}
