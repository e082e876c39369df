// Writing and reading back the 4-bit paged cache.
//
// Per group x_0..x_{g-1} of one token's row, in fp32:
//   z = fp16(min x), s = fp16((max x - z) / 15),
//   c = clamp(rint((x - z) / s), 0, 15) (0 where s is 0), value = c*s + z.
// Scale and zero are rounded to fp16 because they are stored so; the codes are
// chosen against the rounded pair, so the stored pair is the one that counts.
// Bound by memory: 2*D*2 bytes in and D + 8*G bytes out per token and head.
// One thread holds 8 channels (one 16-byte load, one 4-byte store of codes),
// D/8 threads a row, four rows in flight; a group's min and max meet as one
// 16-bit pair in log2(g/8) shuffles.  A CTA takes 64 tokens of one sequence,
// so the row and page lookups are paid once.
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
constexpr int kIoTokens = 64;  // tokens of a CTA: at most three pages
constexpr int kIoUnroll = 4;   // rows a thread has in flight

// The CTA's tokens [m0, m0 + count) of call row i: their first position and the
// pages they lie on (-1: none), read once.
struct IoTile {
  int seq, count, page0;
  int64_t pos0;
  int pages[3];
};

AKV_DEV bool io_tile(const Int4Io& a, int i, int m0, bool write, IoTile& t, int* s_pages) {
  const Int4Row row = int4_row(a.c, a.rows, a.n_new, i, a.M, threadIdx.x == 0 ? a.status : nullptr);
  t.seq = row.seq;
  int n = a.M - m0;  // tokens of the call here
  if (write && n > row.n_new - m0) n = row.n_new - m0;
  t.count = n < kIoTokens ? n : kIoTokens;
  const int64_t first = a.start ? static_cast<int64_t>(a.start[i]) : static_cast<int64_t>(row.len) - row.n_new;
  t.pos0 = first + m0;
  // a page is looked up where it holds one of these tokens
  const int64_t lo = t.pos0 > 0 ? t.pos0 : 0;
  t.page0 = lo < row.len ? static_cast<int>(lo / kBlockTokens) : 0;
  if (threadIdx.x < 3) {
    const int j = t.page0 + threadIdx.x;
    int p = -1;
    if (row.seq >= 0 && static_cast<int64_t>(j) * kBlockTokens < row.len &&
        static_cast<int64_t>(j) * kBlockTokens < t.pos0 + t.count) {
      p = a.c.table[row.seq * a.c.table_stride + j];
      if (p < 0 || p >= a.c.n_pages) {
        set_status(a.status, AKV_ERR_SHAPE);
        p = write ? -1 : 0;
      }
    }
    s_pages[threadIdx.x] = p;
  }
  __syncthreads();
  return t.count > 0;
}

// Walk of the (token, head, K / V) rows of a tile by groups of L threads,
// without a division per row.
struct IoWalk {
  int m, hk, dm, dhk, rows2;
  AKV_DEV void init(int first, int step, int h2) {
    rows2 = h2;
    m = first / h2, hk = first % h2;
    dm = step / h2, dhk = step % h2;
  }
  AKV_DEV void next() {
    m += dm;
    hk += dhk;
    if (hk >= rows2) hk -= rows2, ++m;
  }
};

// x / s to the nearest float, for r the float nearest 1/s: one Newton step on
// the quotient leaves the correctly rounded result (Markstein), so ties in
// rint() fall as they do for the true division.
AKV_DEV float div_by(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-s, q, x), r, q);
}

// the float nearest 1/s for an fp16 value s > 0
AKV_DEV float recip(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return __fmaf_rn(__fmaf_rn(-s, r, 1.f), r, r);
}

// minimum of both halves
template <bool BF>
AKV_DEV uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF) asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool BF>
__global__ void __launch_bounds__(kIoThreads) int4_append_kernel(const Int4Io a) {
  __shared__ int s_pages[3];
  IoTile tile;
  const int i = blockIdx.y, m0 = blockIdx.x * kIoTokens;
  if (!io_tile(a, i, m0, true, tile, s_pages)) return;
  const int D = a.c.head_dim, L = D / 8, group = a.c.group;
  const int part = threadIdx.x % L;  // 8 channels of a row
  const int gl = group / 8;          // threads of a group
  const int G = D / group, gi = part / gl;
  const int vc = kBlockTokens * D / 2, vp = kBlockTokens * G * 4;
  const uint16_t* k = a.k + i * a.k_sr + m0 * a.k_sm + part * 8;
  const uint16_t* v = a.v + i * a.v_sr + m0 * a.v_sm + part * 8;
  IoWalk w;
  w.init(threadIdx.x / L, kIoThreads / L, 2 * a.c.kv_heads);
  // all threads of a warp stay together (the shuffles): rows past the end idle
  const int rows = tile.count * w.rows2, rounds = (rows + kIoThreads / L - 1) / (kIoThreads / L);
  for (int it = 0; it < rounds; it += kIoUnroll) {
    uint4 raw[kIoUnroll];
    int m[kIoUnroll], hk[kIoUnroll];
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      m[u] = w.m, hk[u] = w.hk;
      w.next();
      raw[u] = make_uint4(0u, 0u, 0u, 0u);
      if (m[u] < tile.count) {
        const int h = hk[u] >> 1;
        const uint16_t* src = hk[u] & 1 ? v + h * a.v_sh + m[u] * a.v_sm : k + h * a.k_sh + m[u] * a.k_sm;
        if (a.aligned) {
          raw[u] = ldg_nc_v4(src);
        } else {
          uint16_t e[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) e[j] = src[j];
          raw[u] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      uint32_t e[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      // NaN counts as 0, anything past fp16's range as its end
      bool odd = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (BF) {
          odd |= !(fabsf(__uint_as_float(e[j] << 16)) <= 65504.f) | !(fabsf(__uint_as_float(e[j] & 0xFFFF0000u)) <= 65504.f);
        } else {
          odd |= (e[j] & 0x7C00u) == 0x7C00u || (e[j] & 0x7C000000u) == 0x7C000000u;
        }
      }
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = elem_to_float<BF>(static_cast<uint16_t>(e[j]));
        x[2 * j + 1] = elem_to_float<BF>(static_cast<uint16_t>(e[j] >> 16));
      }
      float lo, hi;
      if (__any_sync(~0u, odd)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -65504.f), 65504.f) : 0.f;
        lo = hi = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]);
        for (int o = 1; o < gl; o <<= 1) {
          lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
          hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
        }
      } else {
        // (minimum, minimum of the negated) of the group in one 16-bit pair
        uint32_t a2 = min2<BF>(min2<BF>(e[0], e[1]), min2<BF>(e[2], e[3]));
        uint32_t b2 = min2<BF>(min2<BF>(e[0] ^ 0x80008000u, e[1] ^ 0x80008000u),
                               min2<BF>(e[2] ^ 0x80008000u, e[3] ^ 0x80008000u));
        uint32_t p = min2<BF>(prmt(a2, b2, 0x5410), prmt(a2, b2, 0x7632));
        for (int o = 1; o < gl; o <<= 1) p = min2<BF>(p, __shfl_xor_sync(~0u, p, o));
        lo = elem_to_float<BF>(static_cast<uint16_t>(p));
        hi = -elem_to_float<BF>(static_cast<uint16_t>(p >> 16));
      }
      if (m[u] >= tile.count) continue;
      const __half zh = __float2half_rn(lo);
      const float z = __half2float(zh);
      const __half sh = __float2half_rn(div_by(__fsub_rn(hi, z), 15.f, 1.f / 15.f));
      const float s = __half2float(sh);
      const float r = s > 0.f ? recip(s) : 0.f;  // scale 0: every quotient 0
      // the float 1.5 * 2^23 + c holds the code in its low bits (rounded half to even by the addition)
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = div_by(__fsub_rn(x[j], z), s, r);
        const float c = fminf(fmaxf(__fadd_rn(q, 12582912.f), 12582912.f), 12582927.f);
        word += __float_as_uint(c) << ((j & 1 ? 0 : 4) + 8 * (j >> 1));
      }
      word -= 0x4B400000u * 0x11111111u;  // the eight exponents' share of the sum
      const int64_t pos = tile.pos0 + m[u];
      const int page = pos >= 0 ? s_pages[static_cast<int>(pos / kBlockTokens) - tile.page0] : -1;
      if (page < 0) continue;
      const int slot = static_cast<int>(pos) % kBlockTokens;
      uint8_t* rec = a.c.pool + page * a.c.page_stride + (hk[u] >> 1) * a.c.head_stride;
      *reinterpret_cast<uint32_t*>(rec + (hk[u] & 1) * vc + slot * (D / 2) + part * 4) = word;
      if (part % gl == 0)
        *reinterpret_cast<__half2*>(rec + 2 * vc + (hk[u] & 1) * vp + (slot * G + gi) * 4) = __halves2half2(sh, zh);
    }
  }
}

template <bool BF>
__global__ void __launch_bounds__(kIoThreads) int4_read_kernel(const Int4Io a) {
  __shared__ int s_pages[3];
  IoTile tile;
  const int i = blockIdx.y, m0 = blockIdx.x * kIoTokens;
  if (!io_tile(a, i, m0, false, tile, s_pages)) return;
  const int D = a.c.head_dim, L = D / 8, group = a.c.group;
  const int part = threadIdx.x % L;
  const int G = D / group, gi = part * 8 / group;
  const int vc = kBlockTokens * D / 2, vp = kBlockTokens * G * 4;
  const int len = tile.seq >= 0 ? a.c.lens[tile.seq] : 0;
  uint16_t* k = a.k + i * a.k_sr + m0 * a.k_sm + part * 8;
  uint16_t* v = a.v + i * a.v_sr + m0 * a.v_sm + part * 8;
  IoWalk w;
  w.init(threadIdx.x / L, kIoThreads / L, 2 * a.c.kv_heads);
  while (w.m < tile.count) {
    uint32_t word[kIoUnroll];
    __half2 sz[kIoUnroll];
    int m[kIoUnroll], hk[kIoUnroll];
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      m[u] = w.m, hk[u] = w.hk;
      w.next();
      word[u] = 0u;
      sz[u] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
      const int64_t pos = tile.pos0 + m[u];
      if (m[u] < tile.count && pos >= 0 && pos < len) {
        const int page = s_pages[static_cast<int>(pos / kBlockTokens) - tile.page0];
        const int slot = static_cast<int>(pos) % kBlockTokens;
        const uint8_t* rec = a.c.pool + page * a.c.page_stride + (hk[u] >> 1) * a.c.head_stride;
        word[u] = __ldg(reinterpret_cast<const uint32_t*>(rec + (hk[u] & 1) * vc + slot * (D / 2) + part * 4));
        sz[u] = __ldg(reinterpret_cast<const __half2*>(rec + 2 * vc + (hk[u] & 1) * vp + (slot * G + gi) * 4));
      }
    }
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      if (m[u] >= tile.count) continue;
      const float s = __low2float(sz[u]), z = __high2float(sz[u]);
      uint32_t out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float e = fmaf(static_cast<float>((word[u] >> (8 * j + 4)) & 15u), s, z);
        float o = fmaf(static_cast<float>((word[u] >> (8 * j)) & 15u), s, z);
        if constexpr (!BF) {  // 15 steps of a rounded-up scale can pass the largest fp16
          e = fminf(fmaxf(e, -65504.f), 65504.f);
          o = fminf(fmaxf(o, -65504.f), 65504.f);
        }
        out[j] = pack_elems<BF>(e, o);
      }
      const int h = hk[u] >> 1;
      uint16_t* dst = hk[u] & 1 ? v + h * a.v_sh + m[u] * a.v_sm : k + h * a.k_sh + m[u] * a.k_sm;
      if (a.aligned) {
        *reinterpret_cast<uint4*>(dst) = make_uint4(out[0], out[1], out[2], out[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j] = static_cast<uint16_t>(out[j / 2] >> (16 * (j & 1)));
      }
    }
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
  const int blocks = (M + kIoTokens - 1) / kIoTokens;
  if (R > 65535 || c->kv_heads > (1 << 20)) return AKV_ERR_UNSUPPORTED;
  a.c = *c;
  a.M = M;
  a.k = static_cast<uint16_t*>(const_cast<void*>(k));
  a.k_sr = k_sr; a.k_sh = k_sh; a.k_sm = k_sm;
  a.v = static_cast<uint16_t*>(const_cast<void*>(v));
  a.v_sr = v_sr; a.v_sh = v_sh; a.v_sm = v_sm;
  a.aligned = rows_aligned16(k, k_sr, k_sh, k_sm) && rows_aligned16(v, v_sr, v_sh, v_sm);
  launch(dim3(blocks, R), a);
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
