// Attention of a chunk of new tokens over the 4-bit paged cache, on the fifth-
// generation tensor cores (kernel templates; one translation unit per head dim
// instantiates them).
//
//   S = Q K^T   softmax over the tokens a query sees   O = P V
// with K, V values c*s + z unpacked from the pages, a tile of TK tokens at a
// time, into shared memory, where all query heads of the KV head read them.
//
// Work.  A unit is one (call row, KV head, tile of NQ x 128 query rows), a row
// being one (token, query head of the group), tokens outer.  The units' token
// tiles form one list that is cut into equal shares, one per CTA (one CTA an
// SM), from the lengths on the device; a unit's set-up counts kChunkSetup tiles
// more.  A unit cut in two or more leaves unnormalised parts that a second
// kernel joins in order.
//
// Roles of a CTA's warps, which meet at mbarriers only:
//   softmax  one warpgroup per 128 query rows, thread = row = TMEM lane: query
//            rows into shared memory, online softmax, P into tensor memory over
//            S, O out
//   values   one warpgroup: pages into registers a tile ahead, then the tile's
//            K and V into their rings
//   MMA      one thread: S = Q K^T from shared memory, O += P V with P from
//            tensor memory
// While one tile's softmax runs, the other's MMAs do.
//
// Roundings.  Queries are scaled per row by a power of two into fp16's middle
// range (bf16; exact unless 2^-24 of the row's largest) or taken as they are
// (fp16).  For a bf16 output K, V and the weights enter the MMAs as one fp16
// term each, every one an eighth of the output's own rounding.  For an fp16
// output (LO) K and the weights are two terms, the second the first's error,
// and V one: its rounding and the output's are alike.  The accumulators, the
// maximum (its weight stands at 2^9, so that small weights keep their bits) and
// the sums are fp32.
//
// Shared-memory operands are unswizzled core matrices of 8 rows x 16 bytes,
// rows 128 B apart by eights, column blocks of 8 channels TK * 16 (Q: 2048)
// bytes apart.  Within a block channels stand as the codes come out of a word,
// 0 4 1 5 2 6 3 7, in Q and K alike; V's order is undone when O is stored.
#pragma once

#include "int4.cuh"
#include "umma.cuh"

namespace akv {

constexpr int kChunkSMs = 148;      // CTAs: one an SM
constexpr int kChunkEntries = 4096; // (row, tile) pairs of one launch
constexpr int kChunkRowsMax = 1024; // call rows of one launch
constexpr int kChunkSetup = 2;      // token tiles that a unit's set-up counts for
constexpr float kChunkTop = 9.f, kChunkMost = 15.f;  // log2: see the header

struct ChunkParams {
  akv_int4_cache c;
  const int32_t* rows;
  const int32_t* n_new;
  int row0, R;  // call rows [row0, row0 + R) of this launch
  int M, Hq, tiles;
  const uint16_t* q;
  int64_t q_sr, q_sh, q_sm;
  float scale;
  uint16_t* out;
  int64_t o_sr, o_sh, o_sm;
  float* lse;
  int bf16;
  int q16, o16;   // query, output rows on 16-byte boundaries
  int4* meta;     // per CTA: (entry, head, last CTA, 1) of the unit whose first part it holds
  float* part;    // [2 * CTA + (first part ? 1 : 0)][D / 4][rows][4]
  float2* ml;     // [slot][rows]: log2 of the maximum's unit, sum
  int* status;
};

template <int D, int G, int LO>
struct ChunkShape {
  static constexpr int NQ = D == 256 ? 1 : 2;
  static constexpr int TK = D == 256 || (D == 128 && LO) ? 64 : 128;
  static constexpr int ROWS = 128 * NQ;
  static constexpr int QB = 128 * D * 2;            // a query tile
  static constexpr int VB = TK * D * 2;             // a tile of V
  static constexpr int KB = VB * (LO ? 2 : 1);      // of K: one or two terms
  static constexpr int KS = D == 256 && LO ? 1 : 2; // ring slots
  static constexpr int VS = 2;
  static constexpr int THREADS = 128 * NQ + 128 + 32;
  static constexpr int PARTS = 128 / TK;            // value threads of a token
  static constexpr int CH = D / PARTS;              // channels of a value thread
  static constexpr int NG = CH * G / D < 1 ? 1 : CH * G / D;  // groups among them
  static constexpr int OFF_K = NQ * QB;
  static constexpr int OFF_V = OFF_K + KS * KB;
  static constexpr int OFF_EX = OFF_V + VS * VB;    // per row: exponent, or a mark for a query that is not finite
  static constexpr int OFF_BAR = OFF_EX + ROWS * 4;
  static constexpr int OFF_ROWS = OFF_BAR + 144;    // lengths, new tokens, prefix sums
  static constexpr int smem(int rows, int entries) { return OFF_ROWS + (2 * rows + entries + 1) * 4; }
  // tensor memory: S (and P) of each tile, then O
  static constexpr int T_S = 0, T_O = NQ * TK;
  static_assert(NQ * (TK + D) <= 512, "tensor memory");
  static_assert(smem(kChunkRowsMax, kChunkEntries) <= 227 * 1024, "shared memory");
};

// The part of a unit that a CTA takes: tiles [t0, t1) of `tiles`.
struct ChunkPart {
  int e, h, i, seq, len, n_new, row;  // row: first query row of the tile
  int t0, t1, tiles, last;            // last: the CTA that takes the unit's end
};

// Walks the CTA's share of the list; every role keeps its own.
template <int TK, int ROWS>
struct ChunkWalk {
  const ChunkParams* P;
  const int *len, *n_new, *pref;
  int H, rep, entries;
  int64_t share, begin, end, pos;
  int e;

  AKV_DEV static int tiles_of(int len, int n_new, int rep, int tile) {
    const int first = tile * ROWS / rep;  // its first query token
    const int last = min((tile * ROWS + ROWS - 1) / rep, n_new - 1);
    const int see = len - n_new + last + 1;
    return first <= last && see > 0 ? (see + TK - 1) / TK : 0;
  }
  AKV_DEV int weight(int x) const { return pref[x + 1] - pref[x]; }

  AKV_DEV void start(const ChunkParams* p, const int* l, const int* n, const int* pr) {
    P = p, len = l, n_new = n, pref = pr;
    H = p->c.kv_heads;
    rep = p->Hq / H;
    entries = p->R * p->tiles;
    const int64_t total = static_cast<int64_t>(pref[entries]) * H;
    share = (total + gridDim.x - 1) / gridDim.x;
    if (share < 2 + kChunkSetup) share = 2 + kChunkSetup;
    begin = min(share * blockIdx.x, total);
    end = min(begin + share, total);
    pos = begin;
    int lo = 0, hi = entries;  // the last entry that starts at or before pos
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<int64_t>(pref[mid]) * H <= pos) lo = mid; else hi = mid;
    }
    e = lo;
  }
  AKV_DEV bool next(ChunkPart& u) {
    while (pos < end) {
      while (static_cast<int64_t>(pref[e + 1]) * H <= pos) ++e;
      const int w = weight(e);
      const int64_t at = pos - static_cast<int64_t>(pref[e]) * H;
      u.h = static_cast<int>(at / w);
      const int off = static_cast<int>(at - static_cast<int64_t>(u.h) * w);
      const int64_t unit = pos - off, stop = min(unit + w, end);
      u.tiles = w - kChunkSetup;
      u.t0 = max(0, off - kChunkSetup);
      u.t1 = static_cast<int>(stop - unit) - kChunkSetup;
      pos = stop;
      if (u.t1 <= u.t0) continue;
      const int r = e / P->tiles;
      u.e = e;
      u.i = P->row0 + r;
      u.seq = P->rows ? __ldg(P->rows + u.i) : u.i;  // in range: it has tiles
      u.len = len[r];
      u.n_new = n_new[r];
      u.row = e % P->tiles * ROWS;
      u.last = static_cast<int>((unit + w - 1) / share);
      return true;
    }
    return false;
  }
};

// ------------------------------------------------------------------ values
// c = the codes of a word, as fp16 pairs of channels (0, 4) (1, 5) (2, 6) (3, 7)
AKV_DEV void codes_of_word(uint32_t w, __half2 (&c)[4]) {
  const uint32_t v = w >> 8;
  const __half2 back = u32_as_h2(0xE400E400u), back16 = u32_as_h2(0xD400D400u), sixteenth = u32_as_h2(0x2C002C00u);
  c[0] = __hfma2(u32_as_h2(lop_magic<0x00F000F0u>(w)), sixteenth, back16);
  c[1] = __hadd2(u32_as_h2(lop_magic<0x000F000Fu>(w)), back);
  c[2] = __hfma2(u32_as_h2(lop_magic<0x00F000F0u>(v)), sixteenth, back16);
  c[3] = __hadd2(u32_as_h2(lop_magic<0x000F000Fu>(v)), back);
}

AKV_DEV __half2 hold(__half2 x) {  // past fp16's range: its ends
  const __half2 top = u32_as_h2(0x7BFF7BFFu);
  return __hmax2(__hmin2(x, top), __hneg2(top));
}

// Rows of one or two terms (c*s + z, and what its rounding left out) at `dst`:
// column blocks `step` bytes apart, the second term `second` bytes on.
template <int NW, int NG, bool TWO>
AKV_DEV void store_values(const uint32_t (&w)[NW], const uint32_t (&pair)[NG], unsigned char* dst, int step, int second) {
  constexpr int PER = NW / NG;  // words (of 8 channels) of a group
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint32_t sz = pair[i / PER];
    const __half2 s = u32_as_h2(prmt(sz, sz, 0x1010)), z = u32_as_h2(prmt(sz, sz, 0x3232));
    // halves, so that no step passes fp16's range (below 2^-13 they lose 2^-25)
    const __half2 half = u32_as_h2(0x38003800u), sh = __hmul2(s, half), zh = __hmul2(z, half);
    __half2 c[4], v[4], r[4];
    codes_of_word(w[i], c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[k] = hold(__hfma2(c[k], s, z));
      if constexpr (TWO) {
        // z - v = d + e exactly, both halved; c*s + d is what v left out, but for e
        const __half2 vh = __hmul2_rn(v[k], half), d = __hsub2(zh, vh), b = __hsub2(d, zh);
        const __half2 e = __hsub2(__hsub2(zh, __hsub2(d, b)), __hadd2(vh, b));
        const __half2 h = __hadd2(__hfma2(c[k], sh, d), e);
        r[k] = __hadd2(h, h);
      }
    }
    *reinterpret_cast<uint4*>(dst + i * step) = make_uint4(h2_as_u32(v[0]), h2_as_u32(v[1]), h2_as_u32(v[2]), h2_as_u32(v[3]));
    if constexpr (TWO)
      *reinterpret_cast<uint4*>(dst + second + i * step) =
          make_uint4(h2_as_u32(r[0]), h2_as_u32(r[1]), h2_as_u32(r[2]), h2_as_u32(r[3]));
  }
}

// ------------------------------------------------------------------ the kernel
template <int D, int G, int LO>
__global__ void __launch_bounds__(ChunkShape<D, G, LO>::THREADS, 1) int4_chunk_kernel(const ChunkParams P) {
  using S = ChunkShape<D, G, LO>;
  constexpr int NQ = S::NQ, TK = S::TK, ROWS = S::ROWS;
  extern __shared__ __align__(1024) unsigned char smem[];
  int* s_ex = reinterpret_cast<int*>(smem + S::OFF_EX);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint64_t *q_ready = bars, *s_full = bars + 2, *p_ready = bars + 4, *o_full = bars + 6;
  uint64_t *k_full = bars + 8, *k_free = bars + 10, *v_full = bars + 12, *v_free = bars + 14;
  uint64_t* drained = bars + 16;
  int* s_len = reinterpret_cast<int*>(smem + S::OFF_ROWS);
  int* s_new = s_len + P.R;
  int* s_pref = s_new + P.R;
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[S::THREADS / 32];

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int H = P.c.kv_heads, rep = P.Hq / H, entries = P.R * P.tiles;

  if (t == 0) {
    for (int k = 0; k < 2; ++k) {
      mbar_init(q_ready + k, 128);
      mbar_init(s_full + k, 1);
      mbar_init(p_ready + k, 128);
      mbar_init(o_full + k, 1);
      mbar_init(k_full + k, 128);
      mbar_init(k_free + k, 1);
      mbar_init(v_full + k, 128);
      mbar_init(v_free + k, 1);
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    P.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- lengths; prefix sums of the entries' weights (tiles and set-up)
  for (int r = t; r < P.R; r += S::THREADS) {
    const Int4Row row = int4_row(P.c, P.rows, P.n_new, P.row0 + r, P.M, P.status);
    s_len[r] = row.len;
    s_new[r] = row.n_new;
  }
  __syncthreads();
  {
    int base = 0;
    for (int e0 = 0; e0 < entries; e0 += S::THREADS) {
      const int e = e0 + t;
      int x = 0;
      if (e < entries) {
        x = ChunkWalk<TK, ROWS>::tiles_of(s_len[e / P.tiles], s_new[e / P.tiles], rep, e % P.tiles);
        if (x) x += kChunkSetup;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      int before = base;
#pragma unroll
      for (int w = 0; w < S::THREADS / 32; ++w) {
        if (w < warp) before += s_scan[w];
        base += s_scan[w];
      }
      if (e < entries) s_pref[e + 1] = before + x;
      __syncthreads();
    }
    if (t == 0) s_pref[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  // ---- entries without any visible token: zero output
  for (int u = blockIdx.x; u < entries * H; u += gridDim.x) {
    const int e = u / H, h = u % H, i = P.row0 + e / P.tiles;
    if (s_pref[e + 1] != s_pref[e]) continue;
    for (int n = warp; n < ROWS; n += S::THREADS / 32) {
      const int rr = e % P.tiles * ROWS + n, m = rr / rep, hq = h * rep + rr - m * rep;
      if (m >= P.M) break;
      uint16_t* o = P.out + i * P.o_sr + hq * P.o_sh + m * P.o_sm;
      for (int c = lane; c < D; c += 32) o[c] = 0;
      if (P.lse && lane == 0) P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = -INFINITY;
    }
  }

  ChunkWalk<TK, ROWS> walk;
  walk.start(&P, s_len, s_new, s_pref);
  ChunkPart u{};
  bool ok = true;  // no bounded wait of this warp has run out
  auto wait = [&](uint64_t* bar, uint32_t phase) {  // by whole warps
    if (ok) ok = __all_sync(~0u, mbar_wait(bar, phase, P.status));
    return ok;
  };

  if (warp < 4 * NQ) {
    // ================================================================ softmax
    const int qt = warp >> 2, r = t & 127;        // query tile, row = TMEM lane
    unsigned char* q_tile = smem + qt * S::QB;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + S::T_S + qt * TK, tO = tmem + lanes + S::T_O + qt * D;

    // this thread's query row into shared memory, as fp16; its exponent for later
    auto load_q = [&](const ChunkPart& x) {
      const int rr = x.row + qt * 128 + r, m = rr / rep, hq = x.h * rep + rr - m * rep;
      const bool on = m < x.n_new;
      const uint16_t* src = P.q + x.i * P.q_sr + hq * P.q_sh + m * P.q_sm;
      auto piece = [&](int c) -> uint4 {  // channels 8c .. 8c + 7
        if (!on) return make_uint4(0u, 0u, 0u, 0u);
        if (P.q16) return *reinterpret_cast<const uint4*>(src + 8 * c);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = src[8 * c + 2 * k] | static_cast<uint32_t>(src[8 * c + 2 * k + 1]) << 16;
        return make_uint4(w[0], w[1], w[2], w[3]);
      };
      uint32_t top = 0u;  // largest magnitude, as the 15 bits of the type
#pragma unroll 8
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = piece(c);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, w[k] >> 16 & 0x7FFFu));
      }
      const bool bad = top >= (P.bf16 ? 0x7F80u : 0x7C00u);  // no softmax: computed as zeros, NaN at the end
      int ex = 0;  // bf16: 2^ex brings the largest into [2^9, 2^10)
      if (P.bf16 && top && !bad) ex = 9 - (static_cast<int>(top >> 7) - 127);
      ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
      const float up = exp2f(static_cast<float>(ex)) * (P.scale < 0.f ? -1.f : 1.f);
      const uint32_t flip = P.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 8
      for (int c = 0; c < D / 8; ++c) {
        const uint4 v = piece(c);
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if (P.bf16) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = pack_h2(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xFFFF0000u) * up);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] ^= flip;
        }
        if (bad) w[0] = w[1] = w[2] = w[3] = 0u;
        *reinterpret_cast<uint4*>(q_tile + r * 16 + c * 2048) =
            make_uint4(prmt(w[0], w[2], 0x5410), prmt(w[0], w[2], 0x7632), prmt(w[1], w[3], 0x5410),
                       prmt(w[1], w[3], 0x7632));
      }
      s_ex[qt * 128 + r] = bad ? INT32_MAX : ex;
      fence_proxy_async_shared();
      mbar_arrive(q_ready + qt);
    };

    uint32_t ph_s = 0, ph_o = 0;
    ChunkWalk<TK, ROWS> ahead = walk;
    ChunkPart nx;
    bool more = ahead.next(nx);
    if (more) load_q(nx);
    while (more && ok) {
      u = nx;
      const int rr = u.row + qt * 128 + r, m = rr / rep, hq = u.h * rep + rr - m * rep;
      const int ex = s_ex[qt * 128 + r];
      const bool bad = ex == INT32_MAX;
      const int see = m < u.n_new ? u.len - u.n_new + m + 1 : 0;
      // log2 e * scale in units of S; never 0, so that -inf stays -inf
      const float sl2 = fmaxf(ldexpf(fabsf(P.scale) * 1.4426950408889634f, bad ? 0 : -ex), 1e-37f);
      float unit = 0.f, lim = -INFINITY, l = 0.f;  // weights are 2^(S sl2 - unit); S past lim moves the unit
      for (int j = u.t0; j < u.t1; ++j) {
        if (!wait(s_full + qt, ph_s)) break;
        ph_s ^= 1;
        tc_fence_after();
        const int vis = see - j * TK;  // columns of the tile that this row sees
        const bool full = __all_sync(~0u, vis >= TK);
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          float x[32];
          tmem_ld32(tS + c * 32, x);
          tmem_wait_ld();
          if (full) {
#pragma unroll
            for (int k = 0; k < 32; ++k) mx = fmaxf(mx, x[k]);
          } else {
#pragma unroll
            for (int k = 0; k < 32; ++k) mx = fmaxf(mx, c * 32 + k < vis ? x[k] : -INFINITY);
          }
        }
        const bool move = mx > lim;
        if (__any_sync(~0u, move)) {
          float f = 1.f;
          if (move) {
            const float now = fmaf(mx, sl2, -kChunkTop);
            f = lim == -INFINITY ? 0.f : exp2f(unit - now);
            unit = now;
            lim = (now + kChunkMost) / sl2;
            l *= f;
          }
          if (j > u.t0) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
              tmem_ld32(tO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= f;
              tmem_st32(tO + c * 32, o);
            }
          }
        }
        uint64_t sum = 0;
        const uint64_t sl22 = f2_make(sl2, sl2), un2 = f2_make(-unit, -unit);
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          float x[32];
          tmem_ld32(tS + c * 32, x);
          tmem_wait_ld();
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float2 y = f2_split(f2_fma(f2_make(x[2 * k], x[2 * k + 1]), sl22, un2));
            y.x = fast_exp2(y.x);
            y.y = fast_exp2(y.y);
            if (!full) {
              if (c * 32 + 2 * k >= vis) y.x = 0.f;
              if (c * 32 + 2 * k + 1 >= vis) y.y = 0.f;
            }
            sum = f2_add(sum, f2_make(y.x, y.y));
            hi[k] = pack_h2(y.x, y.y);
            if constexpr (LO) {
              const float2 b = __half22float2(u32_as_h2(hi[k]));
              lo[k] = pack_h2(y.x - b.x, y.y - b.y);
            }
          }
          if constexpr (LO) {
            tmem_st16u(tS + c * 32, hi);
            tmem_st16u(tS + c * 32 + 16, lo);
          } else {
            tmem_st16u(tS + c * 16, hi);
          }
        }
        const float2 s2 = f2_split(sum);
        l += s2.x + s2.y;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_ready + qt);
      }
      more = ahead.next(nx);
      if (more && ok) load_q(nx);  // every S of this part is out: its queries are done with
      if (!wait(o_full + qt, ph_o)) break;
      ph_o ^= 1;
      tc_fence_after();
      const bool whole = u.t0 == 0 && u.t1 == u.tiles;
      const bool in = m < P.M;
      const int64_t row = static_cast<int64_t>(u.i) * P.o_sr + static_cast<int64_t>(hq) * P.o_sh + m * P.o_sm;
      const float nan = bad && see > 0 ? NAN : 0.f;
      const float inv = l > 0.f ? 1.f / l : 0.f;
      const bool dead = l == 0.f;  // sees nothing (a sum of NaN stays one)
      const int slot = 2 * blockIdx.x + (u.t0 == 0 ? 1 : 0);
      float* part = P.part + static_cast<int64_t>(slot) * ROWS * D + (qt * 128 + r) * 4;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        if (whole) {
          if (!in) continue;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[k] = dead ? 0.f : (l == l ? o[8 * b + (k & 3) * 2 + (k >> 2)] * inv : NAN) + nan;
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = P.bf16 ? pack_elems<true>(v[2 * k], v[2 * k + 1]) : pack_elems<false>(v[2 * k], v[2 * k + 1]);
            uint16_t* dst = P.out + row + c * 32 + b * 8;
            if (P.o16) {
              *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
#pragma unroll
              for (int k = 0; k < 8; ++k) dst[k] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
            }
          }
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              *reinterpret_cast<float4*>(part + static_cast<int64_t>((c * 4 + b) * 2 + hf) * ROWS * 4) =
                  make_float4(o[8 * b + hf] + nan, o[8 * b + 2 + hf] + nan, o[8 * b + 4 + hf] + nan, o[8 * b + 6 + hf] + nan);
        }
      }
      if (whole) {
        if (in && P.lse)
          P.lse[(static_cast<int64_t>(u.i) * P.Hq + hq) * P.M + m] =
              dead ? -INFINITY : (unit + log2f(l)) * 0.6931471805599453f + nan;
      } else {
        P.ml[static_cast<int64_t>(slot) * ROWS + qt * 128 + r] = make_float2(lim == -INFINITY ? -INFINITY : unit, l + nan);
        if (t == 0 && u.t0 == 0) P.meta[blockIdx.x] = make_int4(u.e, u.h, u.last, 1);
      }
      tc_fence_before();
    }
  } else if (warp < 4 * NQ + 4) {
    // ================================================================ values
    const int r = (t & 127) % TK, part = (t & 127) / TK;  // token of the tile, channels part * CH on
    constexpr int NW = S::CH / 8;                          // code words of the thread
    constexpr Int4Layout L = int4_layout(D, G);
    uint32_t kw[NW], vw[NW], kp[S::NG], vp[S::NG];
    const int g0 = part * S::CH / (D / G);                 // its first group
    const uint8_t* rec = nullptr;  // the token's record; nullptr: no token there
    auto fetch_k = [&](const ChunkPart& x, int tile) {
      const int tok = tile * TK + r;
      rec = nullptr;
      if (tok < x.len) {
        int p = __ldg(P.c.table + x.seq * P.c.table_stride + tok / kBlockTokens);
        if (p < 0 || p >= P.c.n_pages) {
          set_status(P.status, AKV_ERR_SHAPE);
          p = 0;
        }
        rec = P.c.pool + p * P.c.page_stride + x.h * P.c.head_stride;
      }
      const int slot = tok % kBlockTokens;
#pragma unroll
      for (int k = 0; k < NW / 4; ++k) {
        const uint4 v = rec ? ldg_nc_v4(rec + L.kc + slot * (D / 2) + part * (S::CH / 2) + 16 * k) : make_uint4(0, 0, 0, 0);
        kw[4 * k] = v.x, kw[4 * k + 1] = v.y, kw[4 * k + 2] = v.z, kw[4 * k + 3] = v.w;
      }
#pragma unroll
      for (int k = 0; k < S::NG; ++k)
        kp[k] = rec ? __ldg(reinterpret_cast<const uint32_t*>(rec + L.kp) + slot * G + g0 + k) : 0u;
    };
    auto fetch_v = [&](int tile) {
      const int slot = (tile * TK + r) % kBlockTokens;
#pragma unroll
      for (int k = 0; k < NW / 4; ++k) {
        const uint4 v = rec ? ldg_nc_v4(rec + L.vc + slot * (D / 2) + part * (S::CH / 2) + 16 * k) : make_uint4(0, 0, 0, 0);
        vw[4 * k] = v.x, vw[4 * k + 1] = v.y, vw[4 * k + 2] = v.z, vw[4 * k + 3] = v.w;
      }
#pragma unroll
      for (int k = 0; k < S::NG; ++k)
        vp[k] = rec ? __ldg(reinterpret_cast<const uint32_t*>(rec + L.vp) + slot * G + g0 + k) : 0u;
    };
    constexpr int STEP = TK * 16;  // between column blocks
    unsigned char* at = smem + r * 16 + part * (S::CH / 8) * STEP;
    int ks = 0, vs = 0;
    uint32_t kph = 1, vph = 1;  // a fresh barrier passes a wait for the phase before its first
    bool more = walk.next(u);
    int j = u.t0;
    if (more) {
      fetch_k(u, j);
      fetch_v(j);
    }
    while (more && ok) {
      ChunkPart nx = u;
      int nj = j + 1;
      bool again = true;
      if (nj == u.t1) {
        again = walk.next(nx);
        nj = nx.t0;
      }
      if (!wait(k_free + ks, kph)) break;
      store_values<NW, S::NG, LO>(kw, kp, at + S::OFF_K + ks * S::KB, STEP, S::VB);
      fence_proxy_async_shared();
      mbar_arrive(k_full + ks);
      if (++ks == S::KS) ks = 0, kph ^= 1;
      if (again) fetch_k(nx, nj);
      if (!wait(v_free + vs, vph)) break;
      store_values<NW, S::NG, false>(vw, vp, at + S::OFF_V + vs * S::VB, STEP, 0);
      fence_proxy_async_shared();
      mbar_arrive(v_full + vs);
      if (++vs == S::VS) vs = 0, vph ^= 1;
      if (again) fetch_v(nj);
      u = nx;
      j = nj;
      more = again;
    }
  } else if (lane == 0) {
    // ================================================================ MMA
    auto wait = [&](uint64_t* bar, uint32_t phase) {  // by this thread alone
      if (ok) ok = mbar_wait(bar, phase, P.status);
      return ok;
    };
    const uint32_t idesc_s = instr_desc(128, TK, 0);  // S = Q K^T: B (= K) K-major
    const uint32_t idesc_o = instr_desc(128, D, 1);   // O = P V: B (= V) MN-major
    const uint32_t base = smem_u32(smem);
    constexpr uint32_t STEP = TK * 16;
    int ks = 0, vs = 0;
    uint32_t kph = 0, vph = 0, ph_p = 0, ph_q = 0;
    auto qk = [&](int q) {
      const uint32_t k_addr = base + S::OFF_K + ks * S::KB;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint64_t a = smem_desc(base + q * S::QB + k * 4096, 2048, 128);
        umma_f16(tmem + S::T_S + q * TK, a, smem_desc(k_addr + k * 2 * STEP, STEP, 128), idesc_s, k > 0 ? 1u : 0u);
        if constexpr (LO)
          umma_f16(tmem + S::T_S + q * TK, a, smem_desc(k_addr + S::VB + k * 2 * STEP, STEP, 128), idesc_s, 1u);
      }
      umma_commit(s_full + q);
    };
    while (ok && walk.next(u)) {
      for (int q = 0; q < NQ; ++q) wait(q_ready + q, ph_q);
      ph_q ^= 1;
      if (!wait(k_full + ks, kph)) break;
      tc_fence_after();
      for (int q = 0; q < NQ; ++q) qk(q);
      umma_commit(k_free + ks);
      if (++ks == S::KS) ks = 0, kph ^= 1;
      for (int j = u.t0; j < u.t1; ++j) {
        if (!wait(v_full + vs, vph)) break;
        const bool again = j + 1 < u.t1;
        const uint32_t v_addr = base + S::OFF_V + vs * S::VB;
        for (int q = 0; q < NQ; ++q) {
          if (!wait(p_ready + q, ph_p)) break;
          tc_fence_after();
          const uint32_t tP = tmem + S::T_S + q * TK, tO = tmem + S::T_O + q * D;
#pragma unroll
          for (int k = 0; k < TK / 16; ++k) {
            const uint64_t b = smem_desc(v_addr + k * 256, 128, STEP);  // tokens = K, channels = N
            const uint32_t on = j > u.t0 || k > 0 ? 1u : 0u;
            if constexpr (LO) {
              const uint32_t col = 32 * (k >> 1) + 8 * (k & 1);
              umma_f16_ts(tO, tP + col, b, idesc_o, on);
              umma_f16_ts(tO, tP + col + 16, b, idesc_o, 1u);
            } else {
              umma_f16_ts(tO, tP + 8 * k, b, idesc_o, on);
            }
          }
          if (q == NQ - 1) umma_commit(v_free + vs);
          if (again) {
            if (q == 0 && !wait(k_full + ks, kph)) break;
            tc_fence_after();
            qk(q);
          } else {
            umma_commit(o_full + q);
          }
        }
        if (!ok) break;
        if (++vs == S::VS) vs = 0, vph ^= 1;
        ph_p ^= 1;
        if (again) {
          umma_commit(k_free + ks);
          if (++ks == S::KS) ks = 0, kph ^= 1;
        }
      }
    }
    if (!ok) {  // a wait ran out: see what was issued end before the tensor memory goes
      umma_commit(drained);
      mbar_wait(drained, 0, P.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------ joining parts
// Block (c, k): 32 query rows of the unit whose first part CTA c holds; its
// parts lie in the slots 2c + 1, 2 (c + 1), ..., 2 last.
template <int D, int ROWS>
__global__ void __launch_bounds__(128) int4_chunk_join_kernel(const ChunkParams P) {
  const int4 meta = P.meta[blockIdx.x];
  if (!meta.w) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int H = P.c.kv_heads, rep = P.Hq / H;
  const int n = blockIdx.y * 32 + lane;  // query row of the tile
  const int e = meta.x, i = P.row0 + e / P.tiles;
  const int rr = e % P.tiles * ROWS + n, m = rr / rep, hq = meta.y * rep + rr - m * rep;
  const int c0 = blockIdx.x, parts = meta.z - c0 + 1;
  auto slot = [&](int s) -> int64_t { return s == 0 ? 2 * c0 + 1 : 2 * (c0 + s); };
  float top = -INFINITY;
  for (int s = 0; s < parts; ++s) top = fmaxf(top, __ldcg(&P.ml[slot(s) * ROWS + n].x));
  float L = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float2 x = __ldcg(&P.ml[slot(s) * ROWS + n]);
    L += x.x == -INFINITY ? x.y : exp2f(x.x - top) * x.y;
  }
  const bool dead = L == 0.f, in = m < P.M;
  const float inv = 1.f / L;
  for (int b = warp; b < D / 8; b += 4) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) {
      const float x = __ldcg(&P.ml[slot(s) * ROWS + n].x);
      const float f = x == -INFINITY ? 0.f : exp2f(x - top);
      const float4* at = reinterpret_cast<const float4*>(P.part) + slot(s) * ROWS * (D / 4) + n;
      const float4 a = __ldcg(at + static_cast<int64_t>(2 * b) * ROWS), c = __ldcg(at + static_cast<int64_t>(2 * b + 1) * ROWS);
      // channels 0..3 and 4..7 of the block
      v[0] = fmaf(f, a.x, v[0]), v[1] = fmaf(f, a.y, v[1]), v[2] = fmaf(f, a.z, v[2]), v[3] = fmaf(f, a.w, v[3]);
      v[4] = fmaf(f, c.x, v[4]), v[5] = fmaf(f, c.y, v[5]), v[6] = fmaf(f, c.z, v[6]), v[7] = fmaf(f, c.w, v[7]);
    }
    if (!in) continue;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = dead ? 0.f : v[2 * k] * inv, c = dead ? 0.f : v[2 * k + 1] * inv;
      w[k] = P.bf16 ? pack_elems<true>(a, c) : pack_elems<false>(a, c);
    }
    uint16_t* dst = P.out + i * P.o_sr + hq * P.o_sh + m * P.o_sm + b * 8;
    if (P.o16) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) dst[k] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
    }
  }
  if (in && P.lse && warp == 0)
    P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = dead ? -INFINITY : (top + log2f(L)) * 0.6931471805599453f;
}

template <int D, int G, int LO>
static int chunk_launch(const ChunkParams& P, cudaStream_t st) {
  using S = ChunkShape<D, G, LO>;
  const int smem = S::smem(P.R, P.R * P.tiles);
  if (!ensure_dynamic_smem<int4_chunk_kernel<D, G, LO>>(smem)) return AKV_ERR_LAUNCH;
  int4_chunk_kernel<D, G, LO><<<kChunkSMs, S::THREADS, smem, st>>>(P);
  int4_chunk_join_kernel<D, S::ROWS><<<dim3(kChunkSMs, S::ROWS / 32), 128, 0, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

template <int D>
static int chunk_dispatch(const ChunkParams& P, cudaStream_t st) {
  switch (D / P.c.group) {
    case 1: return P.bf16 ? chunk_launch<D, 1, 0>(P, st) : chunk_launch<D, 1, 1>(P, st);
    case 2: return P.bf16 ? chunk_launch<D, 2, 0>(P, st) : chunk_launch<D, 2, 1>(P, st);
    default: return P.bf16 ? chunk_launch<D, 4, 0>(P, st) : chunk_launch<D, 4, 1>(P, st);
  }
}

int int4_chunk_64(const ChunkParams& P, cudaStream_t st);
int int4_chunk_128(const ChunkParams& P, cudaStream_t st);
int int4_chunk_256(const ChunkParams& P, cudaStream_t st);

}  // namespace akv
