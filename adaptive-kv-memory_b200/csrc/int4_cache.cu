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
// 16-bit pair in log2(g/8) shuffles.  A CTA takes one page of one sequence, so
// the row and page lookups are paid once.
//
// Measured (4 x 32,767 tokens, 8 heads of 128, bf16, groups of 32; 705 MB moved
// by each direction's kernel): append 137 us (5.1 TB/s; 91 instructions per 8
// values, issue slots 64 %, the rest waits for loads), read 118 us (6.0 TB/s:
// memory).  Append with the unusual groups looked for in every row instead of
// once for four: 147; two rows in flight: 164; three CTAs an SM, no spills: 155;
// five: 159.
#include <type_traits>

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
  int* status;
};

constexpr int kIoThreads = 256;
constexpr int kIoWarps = kIoThreads / 32;
constexpr int kIoUnroll = 4;    // token steps in flight per warp: append,
constexpr int kReadUnroll = 8;  // read (a quarter of the bytes a step)

// The call tokens of row i that lie on one page: block `blk` of the pages that
// its tokens start on.  Token m of the call is at position pos0 + m.
struct IoPage {
  int page;
  int m0, m1;   // call tokens on it
  int end;      // those from here on do not exist (yet)
  int slot0;    // slot of token m0
};

AKV_DEV IoPage io_page(const Int4Io& a, int i, int blk, bool write) {
  int* status = threadIdx.x == 0 ? a.status : nullptr;
  const Int4Row row = int4_row(a.c, a.rows, a.n_new, i, a.M, status);
  IoPage t;
  t.page = -1;
  const int64_t pos0 = a.start ? static_cast<int64_t>(a.start[i]) : static_cast<int64_t>(row.len) - row.n_new;
  const int64_t b0 = pos0 >= 0 ? pos0 / kBlockTokens : -((kBlockTokens - 1 - pos0) / kBlockTokens);  // floor
  const int64_t first = (b0 + blk) * kBlockTokens - pos0;  // call token at the page's first slot
  const int n = write ? row.n_new : a.M;
  t.m0 = first > 0 ? static_cast<int>(first < n ? first : n) : 0;
  t.m1 = first + kBlockTokens < n ? static_cast<int>(first + kBlockTokens) : n;
  t.slot0 = first > 0 ? 0 : static_cast<int>(-first);
  const int64_t pos = (b0 + blk) * kBlockTokens;
  if (row.seq >= 0 && b0 + blk >= 0 && pos < row.len && t.m0 < t.m1) {
    t.page = a.c.table[row.seq * a.c.table_stride + b0 + blk];
    if (t.page < 0 || t.page >= a.c.n_pages) {
      set_status(status, AKV_ERR_SHAPE);
      t.page = write ? -1 : 0;
    }
  }
  const int64_t end = row.len - pos0;
  t.end = t.page < 0 || end < t.m0 ? t.m0 : (end < t.m1 ? static_cast<int>(end) : t.m1);
  if (write) t.m1 = t.end;
  return t;
}

// x / s to the nearest float, for r the float nearest 1/s: one Newton step on
// the quotient leaves the correctly rounded result (Markstein), so ties in
// rint() fall as they do for the true division.  Tested for every fp16 scale,
// at and around the half steps, against the division itself.
AKV_DEV float div_by(float x, float s, float r) {
  const float q = __fmul_rn(x, r);
  return __fmaf_rn(__fmaf_rn(-s, q, x), r, q);
}

// the float nearest 1/s for an fp16 value s > 0: Newton's step on an estimate
AKV_DEV float recip(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return __fmaf_rn(__fmaf_rn(-s, r, 1.f), r, r);
}

template <bool BF>
AKV_DEV uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF) asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF>
AKV_DEV uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF) asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// the same, but NaN where either is
template <bool BF>
AKV_DEV uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF>
AKV_DEV uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool BF>
AKV_DEV void floats_of(uint4 raw, float (&x)[8]) {
  const uint32_t e[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = elem_to_float<BF>(static_cast<uint16_t>(e[j]));
    x[2 * j + 1] = BF ? __uint_as_float(e[j] & 0xFFFF0000u) : elem_to_float<BF>(static_cast<uint16_t>(e[j] >> 16));
  }
}

// (minimum, negated maximum) of a group spread over gl threads as one 16-bit
// pair: NaN where an element is, for the caller to see
template <bool BF, int gl>
AKV_DEV uint32_t group_range(uint4 e) {
  const uint32_t a2 = min2_nan<BF>(min2_nan<BF>(e.x, e.y), min2_nan<BF>(e.z, e.w));
  const uint32_t b2 = max2_nan<BF>(max2_nan<BF>(e.x, e.y), max2_nan<BF>(e.z, e.w)) ^ 0x80008000u;
  uint32_t p = min2_nan<BF>(prmt(a2, b2, 0x5410), prmt(a2, b2, 0x7632));
#pragma unroll
  for (int o = 1; o < gl; o <<= 1) p = min2_nan<BF>(p, __shfl_xor_sync(~0u, p, o));
  return p;
}

// the scale of values from z to hi; the (scale, zero) of values from lo to hi
AKV_DEV __half scale_of(float z, float hi) { return __float2half_rn(div_by(__fsub_rn(hi, z), 15.f, 1.f / 15.f)); }

AKV_DEV __half2 scale_zero(float lo, float hi) {
  const __half z = __float2half_rn(lo);
  return __halves2half2(scale_of(__half2float(z), hi), z);
}

// Codes of eight channels (word in the record's byte order).
template <bool CLAMP>
AKV_DEV uint32_t codes8(const float (&x)[8], __half2 sz) {
  const float s = __low2float(sz), z = __high2float(sz);
  const float r = s > 0.f ? recip(s) : 0.f;  // scale 0: every quotient 0
  // 1.5 * 2^23 + quotient: the sum rounds half to even and holds the code in its low bits
  const uint64_t nz = f2_make(-z, -z), r2 = f2_make(r, r), ns = f2_make(-s, -s), magic = f2_make(12582912.f, 12582912.f);
  float c[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t d = f2_add(f2_make(x[2 * j], x[2 * j + 1]), nz);
    const uint64_t q0 = f2_mul(d, r2);
    const uint64_t q = f2_fma(f2_fma(ns, q0, d), r2, q0);
    const float2 v = f2_split(f2_add(q, magic));
    c[2 * j] = v.x, c[2 * j + 1] = v.y;
  }
  if constexpr (CLAMP) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = fminf(fmaxf(c[j], 12582912.f), 12582927.f);
  }
  // nibbles from the top: channels 6 7 4 5 2 3 0 1; the exponents' share of the sum taken off at the end
  uint32_t w = __float_as_uint(c[6]);
  w = w * 16u + __float_as_uint(c[7]);
  w = w * 16u + __float_as_uint(c[4]);
  w = w * 16u + __float_as_uint(c[5]);
  w = w * 16u + __float_as_uint(c[2]);
  w = w * 16u + __float_as_uint(c[3]);
  w = w * 16u + __float_as_uint(c[0]);
  w = w * 16u + __float_as_uint(c[1]);
  return w - 0x4B400000u * 0x11111111u;
}

// Steps with NaN, elements past fp16's range, or quotients past the codes: NaN
// counts as 0, anything out of range as its end.
template <bool BF, int gl>
AKV_DEV uint32_t quantise8_any(uint4 raw, __half2& sz) {
  float x[8];
  floats_of<BF>(raw, x);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -65504.f), 65504.f) : 0.f;
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]);
#pragma unroll
  for (int o = 1; o < gl; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
  }
  sz = scale_zero(lo, hi);
  return codes8<true>(x, sz);
}

// kIoUnroll steps of eight channels a thread, each group spread over gl
// threads; one vote sends the unusual ones to the general form.  All lanes of
// the warp take part.
template <bool BF, int gl, class Store>
AKV_DEV void quantise_steps(const uint4 (&raw)[kIoUnroll], Store store) {
  constexpr uint32_t PAST = BF ? 0x38803880u : 0x04000400u;  // carries into bits 15 / 31 past 65504, and for NaN
  __half2 sz[kIoUnroll];
  bool odd = false;
#pragma unroll
  for (int u = 0; u < kIoUnroll; ++u) {
    const uint32_t p = group_range<BF, gl>(raw[u]);
    const float lo = elem_to_float<BF>(static_cast<uint16_t>(p));
    const float hi = -elem_to_float<BF>(static_cast<uint16_t>(p >> 16));
    odd |= (((p & 0x7FFF7FFFu) + PAST) & 0x80008000u) != 0;
    // quotients leave [0, 15.5) only where the zero was rounded up (an fp16
    // minimum is its own zero) or the scale has lost bits (below the normal range)
    if constexpr (BF) {
      sz[u] = scale_zero(lo, hi);
      odd |= __high2float(sz[u]) > lo;
    } else {
      sz[u] = __halves2half2(scale_of(lo, hi), __ushort_as_half(static_cast<uint16_t>(p)));
    }
    odd |= __half_as_ushort(__low2half(sz[u])) - 1u < 0x3FFu;
  }
  if (__any_sync(~0u, odd)) {
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      const uint32_t w = quantise8_any<BF, gl>(raw[u], sz[u]);
      store(u, w, sz[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kIoUnroll; ++u) {
      float x[8];
      floats_of<BF>(raw[u], x);
      store(u, codes8<false>(x, sz[u]), sz[u]);
    }
  }
}

// A CTA takes one page of one call row, a warp one (head, K / V) of it at a
// time: D/8 threads a token, so 32 / (D/8) tokens a step.
template <bool BF, int D, int G, bool AL>
__global__ void __launch_bounds__(kIoThreads, 4) int4_append_kernel(const Int4Io a) {
  constexpr int L = D / 8, TW = 32 / L;
  const int i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const IoPage t = io_page(a, i, blockIdx.x, true);
  const int n = t.m1 - t.m0;
  if (n <= 0) return;
  const int part = lane % L, tw = lane / L;
  constexpr int gl = L / G;  // threads of a group
  for (int hk = warp; hk < 2 * a.c.kv_heads; hk += kIoWarps) {
    const int h = hk >> 1, is_v = hk & 1;
    const int64_t sm = is_v ? a.v_sm : a.k_sm;
    const uint16_t* src = (is_v ? a.v + i * a.v_sr + h * a.v_sh : a.k + i * a.k_sr + h * a.k_sh) +
                          (t.m0 + tw) * sm + part * 8;
    uint8_t* rec = a.c.pool + t.page * a.c.page_stride + h * a.c.head_stride;
    uint8_t* codes = rec + is_v * (kBlockTokens * D / 2) + (t.slot0 + tw) * (D / 2) + part * 4;
    uint8_t* pairs = rec + kBlockTokens * D + is_v * (kBlockTokens * G * 4) + ((t.slot0 + tw) * G + part / gl) * 4;
    const bool lead = part % gl == 0;
    // kIoUnroll steps; only the last round of a page has to look at its end
    auto round = [&](int m, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      uint4 raw[kIoUnroll];
#pragma unroll
      for (int u = 0; u < kIoUnroll; ++u) {
        if (!WHOLE) raw[u] = make_uint4(0u, 0u, 0u, 0u);
        if (WHOLE || m + u * TW + tw < n) {
          const uint16_t* p = src + u * (TW * sm);
          if constexpr (AL) {
            raw[u] = ldg_nc_v4(p);
          } else {
            raw[u].x = p[0] | static_cast<uint32_t>(p[1]) << 16;
            raw[u].y = p[2] | static_cast<uint32_t>(p[3]) << 16;
            raw[u].z = p[4] | static_cast<uint32_t>(p[5]) << 16;
            raw[u].w = p[6] | static_cast<uint32_t>(p[7]) << 16;
          }
        }
      }
      quantise_steps<BF, gl>(raw, [&](int u, uint32_t w, __half2 sz) {
        if (WHOLE || m + u * TW + tw < n) {
          *reinterpret_cast<uint32_t*>(codes + u * (TW * D / 2)) = w;
          if (lead) *reinterpret_cast<__half2*>(pairs + u * (TW * G * 4)) = sz;
        }
      });
      src += TW * kIoUnroll * sm;
      codes += TW * kIoUnroll * (D / 2);
      pairs += TW * kIoUnroll * G * 4;
    };
    int m = 0;
    for (; m + TW * kIoUnroll <= n; m += TW * kIoUnroll) round(m, std::true_type{});
    if (m < n) round(m, std::false_type{});
  }
}

// Values of eight channels: four output words.
template <bool BF>
AKV_DEV uint4 dequantise8(uint32_t word, __half2 sz) {
  // fp16 pairs of codes: channels (1, 5), (0, 4), (3, 7), (2, 6)
  uint32_t c[4];
  c[0] = h2_as_u32(__hadd2(u32_as_h2(lop_magic<0x000F000Fu>(word)), u32_as_h2(0xE400E400u)));  // 1024 + c - 1024
  c[1] = fix_magic<16>(lop_magic<0x00F000F0u>(word));
  c[2] = h2_as_u32(__hadd2(u32_as_h2(lop_magic<0x000F000Fu>(word >> 8)), u32_as_h2(0xE400E400u)));
  c[3] = fix_magic<16>(lop_magic<0x00F000F0u>(word >> 8));
  if constexpr (BF) {
    const float s = __low2float(sz), z = __high2float(sz);
    float2 f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = __half22float2(u32_as_h2(c[j]));
      f[j].x = fmaf(f[j].x, s, z);
      f[j].y = fmaf(f[j].y, s, z);
    }
    return make_uint4(pack_elems<true>(f[1].x, f[0].x), pack_elems<true>(f[3].x, f[2].x),
                      pack_elems<true>(f[1].y, f[0].y), pack_elems<true>(f[3].y, f[2].y));
  } else {
    // c*s + z in one rounding; 15 steps of a rounded-up scale can pass the largest fp16
    const __half2 s2 = __low2half2(sz), z2 = __high2half2(sz);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c[j] = max2<false>(min2<false>(h2_as_u32(__hfma2(u32_as_h2(c[j]), s2, z2)), 0x7BFF7BFFu), 0xFBFFFBFFu);
    return make_uint4(prmt(c[1], c[0], 0x5410), prmt(c[3], c[2], 0x5410), prmt(c[1], c[0], 0x7632),
                      prmt(c[3], c[2], 0x7632));
  }
}

template <bool BF, int D, int G, bool AL>
__global__ void __launch_bounds__(kIoThreads, 4) int4_read_kernel(const Int4Io a) {
  constexpr int L = D / 8, TW = 32 / L;
  const int i = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const IoPage t = io_page(a, i, blockIdx.x, false);
  const int n = t.m1 - t.m0;
  if (n <= 0) return;
  const int have = t.end - t.m0;  // the rest are zeros
  const int part = lane % L, tw = lane / L;
  constexpr int gl = L / G;
  for (int hk = warp; hk < 2 * a.c.kv_heads; hk += kIoWarps) {
    const int h = hk >> 1, is_v = hk & 1;
    const int64_t sm = is_v ? a.v_sm : a.k_sm;
    uint16_t* dst = (is_v ? a.v + i * a.v_sr + h * a.v_sh : a.k + i * a.k_sr + h * a.k_sh) + (t.m0 + tw) * sm + part * 8;
    const uint8_t* rec = a.c.pool + (t.page < 0 ? 0 : t.page) * a.c.page_stride + h * a.c.head_stride;
    const uint8_t* codes = rec + is_v * (kBlockTokens * D / 2) + (t.slot0 + tw) * (D / 2) + part * 4;
    const uint8_t* pairs = rec + kBlockTokens * D + is_v * (kBlockTokens * G * 4) + ((t.slot0 + tw) * G + part / gl) * 4;
    auto round = [&](int m, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      uint32_t word[kReadUnroll];
      __half2 sz[kReadUnroll];
#pragma unroll
      for (int u = 0; u < kReadUnroll; ++u) {
        if (!WHOLE) word[u] = 0u, sz[u] = u32_as_h2(0u);
        if (WHOLE || m + u * TW + tw < have) {
          word[u] = __ldg(reinterpret_cast<const uint32_t*>(codes + (m + u * TW) * (D / 2)));
          sz[u] = __ldg(reinterpret_cast<const __half2*>(pairs + (m + u * TW) * G * 4));
        }
      }
#pragma unroll
      for (int u = 0; u < kReadUnroll; ++u) {
        if (!WHOLE && m + u * TW + tw >= n) continue;
        const uint4 v = dequantise8<BF>(word[u], sz[u]);
        uint16_t* p = dst + (m + u * TW) * sm;
        if constexpr (AL) {
          *reinterpret_cast<uint4*>(p) = v;
        } else {
          const uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) p[j] = static_cast<uint16_t>(o[j / 2] >> (16 * (j & 1)));
        }
      }
    };
    int m = 0;
    for (; m + TW * kReadUnroll <= have; m += TW * kReadUnroll) round(m, std::true_type{});
    for (; m < n; m += TW * kReadUnroll) round(m, std::false_type{});
  }
}

template <bool WRITE, bool BF, bool AL>
void io_launch_dim(const Int4Io& p, dim3 grid, cudaStream_t st) {
  auto one = [&](auto dim, auto groups) {
    constexpr int D = decltype(dim)::value, G = decltype(groups)::value;
    if constexpr (WRITE) int4_append_kernel<BF, D, G, AL><<<grid, kIoThreads, 0, st>>>(p);
    else int4_read_kernel<BF, D, G, AL><<<grid, kIoThreads, 0, st>>>(p);
  };
  auto by_group = [&](auto dim) {
    const int G = p.c.head_dim / p.c.group;
    if (G == 1) one(dim, std::integral_constant<int, 1>{});
    else if (G == 2) one(dim, std::integral_constant<int, 2>{});
    else one(dim, std::integral_constant<int, 4>{});
  };
  if (p.c.head_dim == 64) by_group(std::integral_constant<int, 64>{});
  else if (p.c.head_dim == 128) by_group(std::integral_constant<int, 128>{});
  else by_group(std::integral_constant<int, 256>{});
}

template <bool WRITE>
void io_launch(const Int4Io& p, dim3 grid, bool bf16, bool aligned, cudaStream_t st) {
  if (aligned) bf16 ? io_launch_dim<WRITE, true, true>(p, grid, st) : io_launch_dim<WRITE, false, true>(p, grid, st);
  else bf16 ? io_launch_dim<WRITE, true, false>(p, grid, st) : io_launch_dim<WRITE, false, false>(p, grid, st);
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

// argument checks and launch of append and read
template <bool WRITE>
static int int4_io(const akv_int4_io_args* x, void* stream) {
  if (!x) return AKV_ERR_NULL;
  const int rc = int4_check(x->cache);
  if (rc) return rc;
  if (x->dtype != AKV_FP16 && x->dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (x->R < 0 || x->M < 0) return AKV_ERR_SHAPE;
  if (x->R == 0 || x->M == 0) return AKV_OK;
  if (!x->k || !x->v) return AKV_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(x->k) | reinterpret_cast<uintptr_t>(x->v)) & 1) return AKV_ERR_ALIGN;
  if (x->R > 65535 || x->cache->kv_heads > (1 << 20) || x->M > INT32_MAX - 64) return AKV_ERR_UNSUPPORTED;
  Int4Io a{};
  a.c = *x->cache;
  a.rows = x->rows;
  a.n_new = x->n_new;
  a.start = WRITE ? nullptr : x->start;
  a.M = x->M;
  a.k = static_cast<uint16_t*>(x->k);
  a.k_sr = x->k_sr; a.k_sh = x->k_sh; a.k_sm = x->k_sm;
  a.v = static_cast<uint16_t*>(x->v);
  a.v_sr = x->v_sr; a.v_sh = x->v_sh; a.v_sm = x->v_sm;
  a.status = x->status;
  // M tokens from any slot on touch at most this many pages
  const int blocks = (x->M + 2 * kBlockTokens - 2) / kBlockTokens;
  const bool aligned = rows_aligned16(x->k, x->k_sr, x->k_sh, x->k_sm) && rows_aligned16(x->v, x->v_sr, x->v_sh, x->v_sm);
  io_launch<WRITE>(a, dim3(blocks, x->R), x->dtype == AKV_BF16, aligned, static_cast<cudaStream_t>(stream));
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

extern "C" int akv_int4_append(const akv_int4_io_args* a, void* stream) { return int4_io<true>(a, stream); }

extern "C" int akv_int4_read(const akv_int4_io_args* a, void* stream) { return int4_io<false>(a, stream); }
