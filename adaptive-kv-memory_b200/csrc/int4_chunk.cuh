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
//   MMA      one warp: S = Q K^T from shared memory, O += P V with P from
//            tensor memory
// While one tile's softmax runs, the other's MMAs do.
//
// Roundings.  Queries are scaled per row by a power of two into fp16's middle
// range (bf16; exact unless 2^-24 of the row's largest) or taken as they are
// (fp16).  For a bf16 output K, V and the weights enter the MMAs as one fp16
// term each, every one an eighth of the output's own rounding.  For an fp16
// output (LO) K and the weights are two terms, the second the first's error,
// and V one: its rounding and the output's are alike.  The accumulators, the
// maximum (its weight stands at 2^7 and up, so that small weights keep their
// bits) and the sums are fp32.
//
// Shared-memory operands have the 128-byte swizzle: 64 channels of a row in 128
// bytes, rows 128 B apart, the 16-byte pieces of row r permuted by r % 8 (XOR),
// the next 64 channels of all rows behind.  So a value thread's stores (its row,
// piece after piece) meet no bank twice, and one layout serves as the K-major
// operand (Q, K) and the MN-major one (V: tokens = K, channels = N).
// Within a block of 8 channels they stand as the codes come out of a word,
// 0 4 1 5 2 6 3 7, in Q and K alike; V's order is undone when O is stored.
//
// Measured.  2 x 2,048 tokens over 32K, 32 / 8 heads of 128, bf16: 1.93 ms in a
// short burst, 1.10 PFLOP/s of the 1.68 that a matrix product reaches, 2.2 ms (970
// TFLOP/s of its 1.40) in steady repetition, where power holds the clock.  Bursts:
// heads of 64 1.73 ms, of 256 7.5 ms (half the TFLOP/s: one query tile a CTA),
// fp16 (three products for two, tiles of half the size) 3.3 ms.  A tile of 128 tokens takes
// the two query tiles some 3,850 cycles, their MMAs 2,048: what remains is the
// chain from a score to its weight and back to the tensor cores, and the value
// warpgroup's unpacking, 128 tokens in about the tile's time.  Tried and slower:
// two score buffers a query tile with 64-token tiles, an MMA warp for each query
// tile, softmax warps in pairs per row, a part of the exponentials by polynomial.
#pragma once

#include "int4.cuh"
#include "umma.cuh"

namespace akv {

constexpr int kChunkSMs = 148;      // CTAs: one an SM
constexpr int kChunkEntries = 4096; // (row, tile) pairs of one launch
constexpr int kChunkRowsMax = 1024; // call rows of one launch
constexpr int kChunkRep = 4096;     // query heads of a group, at most (the division below)
constexpr int kChunkSetup = 4;      // token tiles that a unit's set-up counts for
// A CTA's share is this many tiles at least, or as few as leave a unit kChunkParts
// parts: more of them take the join longer than their CTAs save (64 new tokens
// after 1,100, 2 heads of 128: shares of 4 32 us, 2 29.4, 1 27.9; one token of 12
// heads over 4,096: 4 31 us, 2 29.5).
constexpr int kChunkShare = 4, kChunkParts = 32;
// A row's maximum stands at 2^7 when its unit is set, and a tile's weights sum up
// to 2^15 at most before it moves: fp16 holds them down to 2^-21 of the maximum
// with all their bits.  A sum says so without the tile's maximum: that is formed
// only where the unit moves.
constexpr float kChunkTop = 7.f, kChunkMost = 32768.f;

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
  uint32_t rep_inv;  // 2^32 / (query heads of a group), rounded up; 0 for one head
  int4* meta;     // per CTA: (entry, head, last CTA, 1) of the unit whose first part it holds
  float* part;    // [2 * CTA + (first part ? 1 : 0)][D / 4][rows][4]
  float2* ml;     // [slot][rows]: log2 of the maximum's unit, sum
  int* status;
};

template <int D, int G, int LO>
struct ChunkShape {
  static constexpr int NQ = D == 256 ? 1 : 2;
  static constexpr int TK = D == 256 || LO ? 64 : 128;
  static constexpr int ROWS = 128 * NQ;
  static constexpr int QB = 128 * D * 2;            // a query tile
  static constexpr int VB = TK * D * 2;             // a tile of V
  static constexpr int KB = VB * (LO ? 2 : 1);      // of K: one or two terms
  static constexpr int KS = D == 256 && LO ? 1 : 2; // ring slots
  static constexpr int VS = 2;
  static constexpr int THREADS = 128 * NQ + 128 + 128;
  // registers of a softmax / value / MMA thread; with 512 threads the launch gives 128 each
  static constexpr bool SPLIT = THREADS == 512;
  static constexpr int R_SOFT = 176, R_VAL = 104, R_MMA = 56;
  static_assert(2 * R_SOFT + R_VAL + R_MMA == 4 * 128, "register shares");
  static constexpr int PARTS = 128 / TK;            // value threads of a token
  static constexpr int CH = D / PARTS;              // channels of a value thread
  static constexpr int NG = CH * G / D < 1 ? 1 : CH * G / D;  // groups among them
  static constexpr int OFF_K = NQ * QB;
  static constexpr int OFF_V = OFF_K + KS * KB;
  static constexpr int OFF_EX = OFF_V + VS * VB;    // per row: exponent, or a mark for a query that is not finite
  static constexpr int OFF_BAR = OFF_EX + ROWS * 4;
  static constexpr int OFF_ROWS = OFF_BAR + 160;    // lengths, new tokens, prefix sums
  static constexpr int smem(int rows, int entries) { return 1024 + OFF_ROWS + (2 * rows + entries + 1) * 4; }
  // tensor memory: S (and P) of each tile, then O
  static constexpr int T_S = 0, T_O = NQ * TK;
  static_assert(NQ * (TK + D) <= 512, "tensor memory");
  static_assert(smem(kChunkRowsMax, kChunkEntries) <= 227 * 1024, "shared memory");
};

// The part of a unit that a CTA takes: tiles [t0, t1) of `tiles`.
struct ChunkPart {
  int e, h, i, len, n_new, row;  // row: first query row of the tile
  int t0, t1, tiles, unit_end;   // unit_end: where the unit ends in the list
};

// What the walk over the CTA's share needs, in shared memory: a role keeps its
// position only.
struct ChunkList {
  const int *len, *n_new, *pref;  // per call row; per entry
  int share, end;
};
struct ChunkPos {
  int pos, e, h;   // the entry and head that pos stands in
  int r, tile;     // the entry's call row and its tile
};

// query row rr of a (row, head): its token, exact for rr * heads < 2^32
AKV_DEV int chunk_token(const ChunkParams& P, int rr) {
  return P.rep_inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(rr), P.rep_inv)) : rr;
}

template <int TK, int ROWS>
AKV_DEV int chunk_tiles(int len, int n_new, int rep, int tile) {
  const int first = tile * ROWS / rep;  // its first query token
  const int last = min((tile * ROWS + ROWS - 1) / rep, n_new - 1);
  const int see = len - n_new + last + 1;
  return first <= last && see > 0 ? (see + TK - 1) / TK : 0;
}

// where the list's position pos stands
AKV_DEV ChunkPos chunk_at(const ChunkParams& P, const ChunkList& L, int pos) {
  const int H = P.c.kv_heads, entries = P.R * P.tiles;
  int lo = 0, hi = entries;  // the last entry that starts at or before pos
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (L.pref[mid] * H <= pos) lo = mid; else hi = mid;
  }
  const int weight = L.pref[lo + 1] - L.pref[lo];
  return ChunkPos{pos, lo, weight ? (pos - L.pref[lo] * H) / weight : 0, lo / P.tiles, lo % P.tiles};
}

// The part at w, which moves past it; false at the share's end.
template <int ROWS>
AKV_DEV bool chunk_next(const ChunkParams& P, const ChunkList& L, ChunkPos& w, ChunkPart& u) {
  const int H = P.c.kv_heads;
  while (w.pos < L.end) {
    const int first = L.pref[w.e], weight = L.pref[w.e + 1] - first;
    if (weight == 0 || w.h == H) {
      w.h = 0;
      ++w.e;
      if (++w.tile == P.tiles) w.tile = 0, ++w.r;
      continue;
    }
    const int unit = first * H + w.h * weight, off = w.pos - unit, stop = min(unit + weight, L.end);
    u.h = w.h;
    u.e = w.e;
    u.i = P.row0 + w.r;
    u.len = L.len[w.r];
    u.n_new = L.n_new[w.r];
    u.row = w.tile * ROWS;
    u.tiles = weight - kChunkSetup;
    u.t0 = max(0, off - kChunkSetup);
    u.t1 = stop - unit - kChunkSetup;
    u.unit_end = unit + weight;
    w.pos = stop;
    if (stop == u.unit_end) ++w.h;
    if (u.t1 > u.t0) return true;
  }
  return false;
}

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

// whether a value of the groups reaches `most` in magnitude
template <int NG>
AKV_DEV bool far_values(const uint32_t (&pair)[NG], float most) {
  bool far = false;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float2 sz = __half22float2(u32_as_h2(pair[g]));
    far |= !(fmaxf(fabsf(sz.y), fabsf(fmaf(15.f, sz.x, sz.y))) < most);
  }
  return far;
}

// A row of one or two terms, its first 64 channels at `dst`, the next `next` bytes
// on, its pieces permuted by x / 16: c*s + z rounded to fp16, or (TWO) a coarser first term and, `second` bytes
// on, what it leaves.
//
// Two terms: with 2^E above the group's magnitudes, M = 1.5 * 2^(E + 1) and z =
// z1 + z2, z1 = (z + M) - M, both exact, the first term hi = fma(c, s, z1 + M) - M
// is a multiple of 2^(E - 9), as z1 is, so that z1 - hi is exact, and the second
// is fma(c, s, z1 - hi) + z2: together 2^(E - 20) or better.  Groups that reach
// 2^13 (FAR) take the exact difference in halves instead.
template <int NW, int NG, bool TWO, bool FAR>
AKV_DEV void store_rows(const uint32_t (&w)[NW], const uint32_t (&pair)[NG], unsigned char* dst, int x, int next, int second) {
  constexpr int PER = NW / NG;  // words (of 8 channels) of a group
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const uint32_t sz = pair[g];
    const __half2 s = u32_as_h2(prmt(sz, sz, 0x1010)), z = u32_as_h2(prmt(sz, sz, 0x3232));
    __half2 big = z, z1 = z, z1m = z, z2 = z, sh = s, zh = z;
    if constexpr (TWO && !FAR) {
      const float2 f = __half22float2(u32_as_h2(sz));
      const float most = fmaxf(fabsf(f.y), fabsf(fmaf(15.f, f.x, f.y)));
      // 2^(E + 1) with 2^(E - 1) <= most < 2^E, 2^-13 at least
      const int e = max((static_cast<int>(__float_as_uint(most)) >> 23) - 127 + 2, -13);
      big = __float2half2_rn(__int_as_float((127 + e) << 23) * 1.5f);
      z1m = __hadd2(z, big);
      z1 = __hsub2(z1m, big);
      z2 = __hsub2(z, z1);
    }
    if constexpr (TWO && FAR) {
      const __half2 half = u32_as_h2(0x38003800u);
      sh = __hmul2(s, half), zh = __hmul2(z, half);
    }
#pragma unroll
    for (int i = g * PER; i < (g + 1) * PER; ++i) {
      __half2 c[4], v[4], r[4];
      codes_of_word(w[i], c);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (!TWO) {
          v[k] = __hfma2(c[k], s, z);
          if constexpr (FAR) v[k] = hold(v[k]);
        } else if constexpr (!FAR) {
          v[k] = __hsub2(__hfma2(c[k], s, z1m), big);
          r[k] = __hadd2(__hfma2(c[k], s, __hsub2(z1, v[k])), z2);
        } else {
          // z - v = d + e exactly, both halved; c*s + d is what v left out, but for e
          v[k] = hold(__hfma2(c[k], s, z));
          const __half2 vh = __hmul2_rn(v[k], u32_as_h2(0x38003800u)), d = __hsub2(zh, vh), b = __hsub2(d, zh);
          const __half2 e = __hsub2(__hsub2(zh, __hsub2(d, b)), __hadd2(vh, b));
          const __half2 h = __hadd2(__hfma2(c[k], sh, d), e);
          r[k] = __hadd2(h, h);
        }
      }
      unsigned char* at = dst + (i >> 3) * next + ((i & 7) * 16 ^ x);
      *reinterpret_cast<uint4*>(at) =
          make_uint4(h2_as_u32(v[0]), h2_as_u32(v[1]), h2_as_u32(v[2]), h2_as_u32(v[3]));
      if constexpr (TWO)
        *reinterpret_cast<uint4*>(at + second) =
            make_uint4(h2_as_u32(r[0]), h2_as_u32(r[1]), h2_as_u32(r[2]), h2_as_u32(r[3]));
    }
  }
}

template <int NW, int NG, bool TWO>
AKV_DEV void store_values(const uint32_t (&w)[NW], const uint32_t (&pair)[NG], unsigned char* dst, int x, int next, int second) {
  if (__any_sync(~0u, far_values(pair, TWO ? 8192.f : 65000.f))) store_rows<NW, NG, TWO, true>(w, pair, dst, x, next, second);
  else store_rows<NW, NG, TWO, false>(w, pair, dst, x, next, second);
}

// Lane i of four holds piece k of its row in w[k]: afterwards piece i of row k.
AKV_DEV void transpose4(uint4 (&w)[4]) {
  const int lane = threadIdx.x & 31;
  auto swap = [&](int a, int b, int bit) {
    const bool up = lane & bit;
    const uint4 give = up ? w[a] : w[b];
    const uint4 got = make_uint4(__shfl_xor_sync(~0u, give.x, bit), __shfl_xor_sync(~0u, give.y, bit),
                                 __shfl_xor_sync(~0u, give.z, bit), __shfl_xor_sync(~0u, give.w, bit));
    (up ? w[a] : w[b]) = got;
  };
  swap(0, 1, 1), swap(2, 3, 1), swap(0, 2, 2), swap(1, 3, 2);
}

// ------------------------------------------------------------------ the kernel
template <int D, int G, int LO>
__global__ void __launch_bounds__(ChunkShape<D, G, LO>::THREADS, 1) int4_chunk_kernel(const ChunkParams P) {
  using S = ChunkShape<D, G, LO>;
  constexpr int NQ = S::NQ, TK = S::TK, ROWS = S::ROWS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // the swizzle goes by the address: tiles start on 1 KB
  unsigned char* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
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
  __shared__ ChunkList s_list;
  __shared__ ChunkPos s_begin;

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
        x = chunk_tiles<TK, ROWS>(s_len[e / P.tiles], s_new[e / P.tiles], rep, e % P.tiles);
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
    if (t == 0) {
      s_pref[0] = 0;
      const int total = base * H;
      int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
      const int each = (total + entries * H - 1) / (entries * H);  // tiles of a unit
      share = max(share, max(1, min(kChunkShare, (each + kChunkParts - 1) / kChunkParts)));
      const int begin = static_cast<int>(min(static_cast<int64_t>(share) * blockIdx.x, static_cast<int64_t>(total)));
      s_list = ChunkList{s_len, s_new, s_pref, share, total - begin > share ? begin + share : total};
      s_begin = chunk_at(P, s_list, begin);
    }
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

  ChunkPos walk = s_begin;
  auto next = [&](ChunkPart& x) { return chunk_next<ROWS>(P, s_list, walk, x); };
  bool ok = true;  // no bounded wait of this warp has run out
  auto wait = [&](uint64_t* bar, uint32_t phase) {  // by whole warps
    if (ok) ok = mbar_wait_warp(bar, phase, P.status);
    return ok;
  };

  if (warp < 4 * NQ) {
    // ================================================================ softmax
    if constexpr (S::SPLIT) regs_up<S::R_SOFT>();
    const int qt = warp >> 2, r = t & 127;        // query tile, row = TMEM lane
    unsigned char* q_tile = smem + qt * S::QB;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + S::T_S + qt * TK, tO = tmem + lanes + S::T_O + qt * D;

    // The warp's 32 query rows into shared memory, as fp16; their exponents for
    // later.  A load takes 64 bytes of 8 rows, a store 8 rows of a column block.
    auto load_q = [&](const ChunkPart& x) {
      constexpr int IT = D / 32;             // loads of a row
      constexpr int GR = D == 256 ? 2 : 4;   // groups of 8 rows in flight
      const int piece = lane >> 3;
#pragma unroll
      for (int g0 = 0; g0 < 4; g0 += GR) {
        uint4 v[GR][IT];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const int rr = x.row + qt * 128 + (warp & 3) * 32 + (g0 + g) * 8 + (lane & 7);
          const int m = chunk_token(P, rr), hq = x.h * rep + rr - m * rep;
          const uint16_t* src = P.q + x.i * P.q_sr + hq * P.q_sh + m * P.q_sm + piece * 8;
          if (m >= x.n_new) {
#pragma unroll
            for (int k = 0; k < IT; ++k) v[g][k] = make_uint4(0u, 0u, 0u, 0u);
          } else if (P.q16) {
#pragma unroll
            for (int k = 0; k < IT; ++k) v[g][k] = *reinterpret_cast<const uint4*>(src + 32 * k);
          } else {
#pragma unroll
            for (int k = 0; k < IT; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int c = 0; c < 4; ++c)
                w[c] = src[32 * k + 2 * c] | static_cast<uint32_t>(src[32 * k + 2 * c + 1]) << 16;
              v[g][k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const int row = (warp & 3) * 32 + (g0 + g) * 8 + (lane & 7);
          uint32_t top = 0u;  // largest magnitude of the row, as the 15 bits of the type
#pragma unroll
          for (int k = 0; k < IT; ++k)
            top = __vmaxu2(__vmaxu2(top, v[g][k].x & 0x7FFF7FFFu),
                           __vmaxu2(v[g][k].y & 0x7FFF7FFFu, __vmaxu2(v[g][k].z & 0x7FFF7FFFu, v[g][k].w & 0x7FFF7FFFu)));
          top = max(top & 0xFFFFu, top >> 16);
          top = max(top, __shfl_xor_sync(~0u, top, 8));
          top = max(top, __shfl_xor_sync(~0u, top, 16));
          const bool bad = top >= (LO ? 0x7C00u : 0x7F80u);  // no softmax: computed as zeros, NaN at the end
          int ex = 0;  // bf16: 2^ex brings the largest into [2^9, 2^10)
          if (!LO && top && !bad) ex = 9 - (static_cast<int>(top >> 7) - 127);
          ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
          const float up = __int_as_float((127 + ex) << 23) * (P.scale < 0.f ? -1.f : 1.f);
          const uint32_t flip = P.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
          for (int k = 0; k < IT; ++k) {
            uint32_t w[4] = {v[g][k].x, v[g][k].y, v[g][k].z, v[g][k].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if constexpr (!LO)
                w[c] = pack_h2(__uint_as_float(w[c] << 16) * up, __uint_as_float(w[c] & 0xFFFF0000u) * up);
              else
                w[c] ^= flip;
              if (bad) w[c] = 0u;
            }
            *reinterpret_cast<uint4*>(q_tile + (k >> 1) * (128 * 128) + row * 128 + (((4 * (k & 1) + piece) ^ (lane & 7)) * 16)) =
                make_uint4(prmt(w[0], w[2], 0x5410), prmt(w[0], w[2], 0x7632), prmt(w[1], w[3], 0x5410),
                           prmt(w[1], w[3], 0x7632));
          }
          if (piece == 0) s_ex[qt * 128 + row] = bad ? INT32_MAX : ex;
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      mbar_arrive(q_ready + qt);
    };

    uint32_t ph_s = 0, ph_o = 0;
    ChunkPos here = walk;  // where the part at hand is decoded from: its fields are not kept over the tiles
    bool more;
    {
      ChunkPart u;
      more = next(u);
      if (more) load_q(u);
    }
    while (more && ok) {
      int see, t0, t1;
      {
        ChunkPart u;
        ChunkPos w = here;
        chunk_next<ROWS>(P, s_list, w, u);
        const int m = chunk_token(P, u.row + qt * 128 + r);
        see = m < u.n_new ? u.len - u.n_new + m + 1 : 0;
        t0 = u.t0, t1 = u.t1;
      }
      const int ex = s_ex[qt * 128 + r];
      const bool bad = ex == INT32_MAX;
      // log2 e * scale in units of S; never 0, so that -inf stays -inf
      const float sl2 = fmaxf(ldexpf(fabsf(P.scale) * 1.4426950408889634f, bad ? 0 : -ex), 1e-37f);
      float unit = 0.f, l = 0.f;  // weights are 2^(S sl2 - unit), l their sum
      bool fresh = true;          // no token seen: the unit is not set
      for (int j = t0; j < t1; ++j) {
        if (!wait(s_full + qt, ph_s)) break;
        ph_s ^= 1;
        tc_fence_after();
        const int vis = see - j * TK;  // columns of the tile that this row sees
        const bool full = __all_sync(~0u, vis >= TK);
        uint32_t hi[TK / 32][16], lo[LO ? TK / 32 : 1][16];
        float part = 0.f;
        // 0: the unit is set first; 1: weights by the unit there is; 2: again, by a new one
        for (int round = __any_sync(~0u, fresh && vis > 0) ? 0 : 1;; round = 2) {
          if (round != 1) {
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < TK / 16; ++c) {
              float x[16];
              tmem_ld16(tS + c * 16, x);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) mx = fmaxf(mx, c * 16 + k < vis ? x[k] : -INFINITY);
            }
            const float now = fmaf(mx, sl2, -kChunkTop);
            float f = 1.f;
            if (mx > -INFINITY && (fresh || now > unit)) {
              f = fresh ? 0.f : exp2f(unit - now);
              unit = now;
              l *= f;
              fresh = false;
            }
            if (j > t0) {
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                float o[16];
                tmem_ld16(tO + c * 16, o);
                tmem_wait_ld();
                uint32_t w[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(o[k] * f);
                tmem_st16u(tO + c * 16, w);
              }
            }
          }
          uint64_t sum = 0;
          const uint64_t sl22 = f2_make(sl2, sl2), un2 = f2_make(-unit, -unit);
          float x[2][32];
          tmem_ld32(tS, x[0]);
#pragma unroll
          for (int c = 0; c < TK / 32; ++c) {
            tmem_wait_ld();
            if (c + 1 < TK / 32) tmem_ld32(tS + (c + 1) * 32, x[(c + 1) & 1]);
            float(&v)[32] = x[c & 1];
            if (!full) {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = c * 32 + k < vis ? v[k] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float2 y = f2_split(f2_fma(f2_make(v[2 * k], v[2 * k + 1]), sl22, un2));
              y.x = fast_exp2(y.x);
              y.y = fast_exp2(y.y);
              sum = f2_add(sum, f2_make(y.x, y.y));
              hi[c][k] = pack_h2(y.x, y.y);
              if constexpr (LO) {
                const float2 b = __half22float2(u32_as_h2(hi[c][k]));
                lo[c][k] = pack_h2(y.x - b.x, y.y - b.y);
              }
            }
          }
          const float2 s2 = f2_split(sum);
          part = s2.x + s2.y;
          if (round != 1 || __all_sync(~0u, part <= kChunkMost)) break;
        }
        l += part;
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          if constexpr (LO) {
            tmem_st16u(tS + c * 32, hi[c]);
            tmem_st16u(tS + c * 32 + 16, lo[c]);
          } else {
            tmem_st16u(tS + c * 16, hi[c]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_ready + qt);
      }
      if (fresh) l = 0.f;
      ChunkPart u;
      chunk_next<ROWS>(P, s_list, here, u);
      here = walk;
      {
        ChunkPart nx;
        more = next(nx);
        if (more && ok) load_q(nx);  // every S of this part is out: its queries are done with
      }
      const int rr = u.row + qt * 128 + r, m = chunk_token(P, rr), hq = u.h * rep + rr - m * rep;
      if (!wait(o_full + qt, ph_o)) break;
      ph_o ^= 1;
      tc_fence_after();
      const bool whole = u.t0 == 0 && u.t1 == u.tiles;
      const bool in = m < P.M;
      const int64_t row = static_cast<int64_t>(u.i) * P.o_sr + static_cast<int64_t>(hq) * P.o_sh + m * P.o_sm;
      const float nan = bad && see > 0 ? NAN : 0.f;
      const float inv = 1.f / l;
      const bool dead = l == 0.f;  // sees nothing
      int64_t at[4];  // output rows of the four lanes' query rows; -1: none
#pragma unroll
      for (int k = 0; k < 4; ++k) at[k] = __shfl_sync(~0u, in ? row : -1, (lane & 28) + k);
      const int slot = 2 * blockIdx.x + (u.t0 == 0 ? 1 : 0);
      float* part = P.part + static_cast<int64_t>(slot) * ROWS * D + (qt * 128 + r) * 4;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        if (whole) {
          uint4 w[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = dead ? 0.f : o[8 * b + (k & 3) * 2 + (k >> 2)] * inv + nan;
            w[b] = make_uint4(pack_elems<!LO>(v[0], v[1]), pack_elems<!LO>(v[2], v[3]), pack_elems<!LO>(v[4], v[5]),
                              pack_elems<!LO>(v[6], v[7]));
          }
          if (P.o16) {
            // four lanes exchange, so that a store takes 64 bytes of 8 rows
            transpose4(w);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (at[k] >= 0) *reinterpret_cast<uint4*>(P.out + at[k] + c * 32 + (lane & 3) * 8) = w[k];
          } else if (in) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const uint32_t x[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
              for (int k = 0; k < 8; ++k) P.out[row + c * 32 + b * 8 + k] = static_cast<uint16_t>(x[k / 2] >> (16 * (k & 1)));
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
        P.ml[static_cast<int64_t>(slot) * ROWS + qt * 128 + r] = make_float2(fresh ? -INFINITY : unit, l + nan);
        if (t == 0 && u.t0 == 0) P.meta[blockIdx.x] = make_int4(u.e, u.h, (u.unit_end - 1) / s_list.share, 1);
      }
      tc_fence_before();
    }
  } else if (warp < 4 * NQ + 4) {
    // ================================================================ values
    if constexpr (S::SPLIT) regs_down<S::R_VAL>();
    const int r = (t & 127) % TK, part = (t & 127) / TK;  // token of the tile, channels part * CH on
    constexpr int NW = S::CH / 8;                          // code words of the thread
    constexpr Int4Layout L = int4_layout(D, G);
    uint32_t kw[NW], vw[NW], kp[S::NG], vp[S::NG];
    const int g0 = part * S::CH / (D / G);                 // its first group
    const uint8_t* rec = nullptr;  // the token's record; nullptr: no token there
    auto page_of = [&](const ChunkPart& x, int tile) -> int {  // of the thread's token, as the table has it
      const int tok = tile * TK + r;
      const int seq = P.rows ? __ldg(P.rows + x.i) : x.i;  // in range: it has tiles
      return tok < x.len ? __ldg(P.c.table + seq * P.c.table_stride + tok / kBlockTokens) : 0;
    };
    auto fetch_k = [&](const ChunkPart& x, int tile, int p) {
      const int tok = tile * TK + r;
      rec = nullptr;
      if (tok < x.len) {
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
    constexpr int NEXT = TK * 128;  // from 64 channels to the next
    unsigned char* at = smem + r * 128 + part * (S::CH / 64) * NEXT;
    const int swz = ((r ^ part * (S::CH / 8)) & 7) * 16;  // half a row of 64 channels starts at its fifth piece
    int ks = 0, vs = 0;
    uint32_t kph = 1, vph = 1;  // a fresh barrier passes a wait for the phase before its first
    ChunkPart u{};
    bool more = next(u);
    int j = u.t0;
    int page = 0;  // of the tile after the next
    if (more) {
      fetch_k(u, j, page_of(u, j));
      fetch_v(j);
      if (j + 1 < u.t1) page = page_of(u, j + 1);
    }
    while (more && ok) {
      ChunkPart nx = u;
      int nj = j + 1;
      bool again = true;
      if (nj == u.t1) {
        again = next(nx);
        nj = nx.t0;
      }
      if (!wait(k_free + ks, kph)) break;
      store_values<NW, S::NG, LO>(kw, kp, at + S::OFF_K + ks * S::KB, swz, NEXT, S::VB);
      fence_proxy_async_shared();
      mbar_arrive(k_full + ks);
      if (++ks == S::KS) ks = 0, kph ^= 1;
      if (again) {
        fetch_k(nx, nj, nj == nx.t0 ? page_of(nx, nj) : page);
        if (nj + 1 < nx.t1) page = page_of(nx, nj + 1);
      }
      if (!wait(v_free + vs, vph)) break;
      store_values<NW, S::NG, false>(vw, vp, at + S::OFF_V + vs * S::VB, swz, NEXT, 0);
      fence_proxy_async_shared();
      mbar_arrive(v_full + vs);
      if (++vs == S::VS) vs = 0, vph ^= 1;
      if (again) fetch_v(nj);
      u = nx;
      j = nj;
      more = again;
    }
  } else {
    // ================================================================ MMA
    if constexpr (S::SPLIT) regs_down<S::R_MMA>();
    if (warp == 4 * NQ + 4) {
    const uint32_t lead = elect_one();
    constexpr uint32_t NEXT = TK * 128;  // from 64 channels to the next
    constexpr uint32_t HI = desc_hi_sw128(1024);
    constexpr uint32_t IDESC_S = instr_desc(128, TK, 0);  // S = Q K^T: B (= K) K-major
    constexpr uint32_t IDESC_O = instr_desc(128, D, 1);   // O = P V: B (= V) MN-major
    const uint32_t base = smem_u32(smem);
    int ks = 0, vs = 0;
    uint32_t kph = 0, vph = 0, ph_p = 0, ph_q = 0;
    auto qk = [&](int q) {
      const uint32_t a = desc_lo(base + q * S::QB, 16), b = desc_lo(base + S::OFF_K + ks * S::KB, 16);
      const uint32_t d = tmem + S::T_S + q * TK;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t ak = a + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16, bk = b + ((k >> 2) * NEXT + (k & 3) * 32) / 16;
        umma_ss<HI, HI, IDESC_S>(d, ak, bk, k > 0 ? 1u : 0u, lead);
        if constexpr (LO) umma_ss<HI, HI, IDESC_S>(d, ak, bk + S::VB / 16, 1u, lead);
      }
      umma_commit(s_full + q, lead);
    };
    ChunkPart u;
    while (ok && next(u)) {
      for (int q = 0; q < NQ; ++q) wait(q_ready + q, ph_q);
      ph_q ^= 1;
      if (!wait(k_full + ks, kph)) break;
      tc_fence_after();
      for (int q = 0; q < NQ; ++q) qk(q);
      umma_commit(k_free + ks, lead);
      if (++ks == S::KS) ks = 0, kph ^= 1;
      for (int j = u.t0; j < u.t1; ++j) {
        if (!wait(v_full + vs, vph)) break;
        const bool again = j + 1 < u.t1;
        const uint32_t v = desc_lo(base + S::OFF_V + vs * S::VB, NEXT);
        for (int q = 0; q < NQ; ++q) {
          if (!wait(p_ready + q, ph_p)) break;
          tc_fence_after();
          const uint32_t tP = tmem + S::T_S + q * TK, tO = tmem + S::T_O + q * D;
#pragma unroll
          for (int k = 0; k < TK / 16; ++k) {
            const uint32_t on = j > u.t0 || k > 0 ? 1u : 0u;
            if constexpr (LO) {
              const uint32_t col = 32 * (k >> 1) + 8 * (k & 1);
              umma_ts<HI, IDESC_O>(tO, tP + col, v + k * 128, on, lead);
              umma_ts<HI, IDESC_O>(tO, tP + col + 16, v + k * 128, 1u, lead);
            } else {
              umma_ts<HI, IDESC_O>(tO, tP + 8 * k, v + k * 128, on, lead);
            }
          }
          if (q == NQ - 1) umma_commit(v_free + vs, lead);
          if (again) {
            if (q == 0 && !wait(k_full + ks, kph)) break;
            tc_fence_after();
            qk(q);
          } else {
            umma_commit(o_full + q, lead);
          }
        }
        if (!ok) break;
        if (++vs == S::VS) vs = 0, vph ^= 1;
        ph_p ^= 1;
        if (again) {
          umma_commit(k_free + ks, lead);
          if (++ks == S::KS) ks = 0, kph ^= 1;
        }
      }
    }
    if (!ok) {  // a wait ran out: see what was issued end before the tensor memory goes
      umma_commit(drained, lead);
      mbar_wait(drained, 0, P.status);
    }
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
__global__ void __launch_bounds__(D * 4) int4_chunk_join_kernel(const ChunkParams P) {
  __shared__ float2 s_ml[kChunkSMs][32];
  const int4 meta = P.meta[blockIdx.x];
  if (!meta.w) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int H = P.c.kv_heads, rep = P.Hq / H;
  const int n = blockIdx.y * 32 + lane;  // query row of the tile
  const int e = meta.x, i = P.row0 + e / P.tiles;
  const int rr = e % P.tiles * ROWS + n, m = rr / rep, hq = meta.y * rep + rr - m * rep;
  const int c0 = blockIdx.x, parts = meta.z - c0 + 1;
  auto slot = [&](int s) -> int64_t { return s == 0 ? 2 * c0 + 1 : 2 * (c0 + s); };
  for (int s = warp; s < parts; s += D / 8) s_ml[s][lane] = __ldcg(&P.ml[slot(s) * ROWS + n]);
  __syncthreads();
  float top = -INFINITY;
  for (int s = 0; s < parts; ++s) top = fmaxf(top, s_ml[s][lane].x);
  float L = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float2 x = s_ml[s][lane];
    L += x.x == -INFINITY ? x.y : exp2f(x.x - top) * x.y;
  }
  const bool dead = L == 0.f, in = m < P.M;
  const float inv = 1.f / L;
  const int b = warp;  // the warp's 8 channels
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float x = s_ml[s][lane].x;
    const float f = x == -INFINITY ? 0.f : exp2f(x - top);
    const float4* at = reinterpret_cast<const float4*>(P.part) + slot(s) * ROWS * (D / 4) + n;
    const float4 a = __ldcg(at + static_cast<int64_t>(2 * b) * ROWS), c = __ldcg(at + static_cast<int64_t>(2 * b + 1) * ROWS);
    // channels 0..3 and 4..7 of the block
    v[0] = fmaf(f, a.x, v[0]), v[1] = fmaf(f, a.y, v[1]), v[2] = fmaf(f, a.z, v[2]), v[3] = fmaf(f, a.w, v[3]);
    v[4] = fmaf(f, c.x, v[4]), v[5] = fmaf(f, c.y, v[5]), v[6] = fmaf(f, c.z, v[6]), v[7] = fmaf(f, c.w, v[7]);
  }
  if (!in) return;
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
  if (in && P.lse && warp == 0)
    P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = dead ? -INFINITY : (top + log2f(L)) * 0.6931471805599453f;
}

template <int D, int G, int LO>
static int chunk_launch(const ChunkParams& P, cudaStream_t st) {
  using S = ChunkShape<D, G, LO>;
  const int smem = S::smem(P.R, P.R * P.tiles);
  if (!ensure_dynamic_smem<int4_chunk_kernel<D, G, LO>>(smem)) return AKV_ERR_LAUNCH;
  int4_chunk_kernel<D, G, LO><<<kChunkSMs, S::THREADS, smem, st>>>(P);
  int4_chunk_join_kernel<D, S::ROWS><<<dim3(kChunkSMs, S::ROWS / 32), D * 4, 0, st>>>(P);
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
