// Eviction from the 4-bit paged cache by accumulated attention weight.
//
//   score[t] = fp32(sum over layers of weights[l][s][t], summed in fp64)
// (one rounding: the order of the layers does not decide a tie), the first
// `first` and last `recent` tokens above all others; the `keep` largest stay,
// the lowest token first among equal ones, and move together in their order, in
// every layer and head.
//
// Five steps, each a launch: scores; the keep-th largest score by a radix
// select, the list of the kept tokens and the pages that are shared and would be
// written, a CTA a row; new pages for those (their other holders keep the old
// ones), in the order of the rows; the moves; tables, lengths and reference counts.
//
// Moves in place.  The kept tokens of page j come from pages >= j, so taking
// the pages in ascending order a CTA may read ahead freely; it only has to have
// read all of a page's sources before it writes that page.  A CTA owns the K or
// the V of one (row, layer, head), and four 16-byte pieces a thread stand in
// registers between read and write.  Pages before the first token that goes are
// left alone.
//
// Bound by the moves: 16 rows of 1K to 7K tokens brought to 2,000 in 16 layers of
// 8 heads of 128, 1.1 GB read and written, 204 us of the call's 225 to 260, by the
// lengths drawn (170 at the memory's rate); by five launches in a chain where they are few: one row of
// 4,352 to 4,096 in 28 layers of 2 heads 46 us (scores 6, selection 13, pages 4,
// moves 17, tables 4).
#include "int4.cuh"

namespace akv {

constexpr int kSelectThreads = 1024;
constexpr int kMovePieces = 4;  // 16-byte pieces of a thread between read and write

// What a step of the eviction knows of a call row.
struct EvictRow {
  int seq;    // -1: refused
  int len;    // tokens before
  int left;   // tokens after
  int start;  // first page that is written; pages [start, end) are
  int end;
  int need;   // of them shared: each gets a new page
  int off;    // the row's first new page in the list
  int pad;
};

struct EvictParams {
  akv_page_table T;
  uint8_t* pool;
  int64_t layer_stride, page_bytes;
  int n_layers, kv_heads, head_dim, n_groups;
  float* weights;
  int64_t w_layer, w_row;
  const int32_t* rows;
  int n, keep, first, recent;
  int32_t* kept;
  // workspace
  EvictRow* info;
  uint32_t* score;   // [n][max_blocks * 32] order of the scores
  int32_t* list;     // new pages
  int32_t* to;       // [n][max_blocks] what each page of the row becomes: new_page()
  int* status;
};

AKV_DEV int max_tokens(const EvictParams& P) { return P.T.max_blocks * kBlockTokens; }

// Sequence and length of call row i; seq -1 for one that is refused (a bad or
// repeated row, a bad length).  All threads of the block call it.
AKV_DEV int2 evict_row(const EvictParams& P, int i) {
  const int seq = P.rows ? P.rows[i] : i;
  bool bad = seq < 0 || seq >= P.T.max_seqs;
  if (P.rows)
    for (int s = threadIdx.x; s < i; s += blockDim.x) bad |= P.rows[s] == seq;
  bad = __syncthreads_or(bad);
  const int len = bad ? 0 : P.T.lens[seq];
  if (bad || len < 0 || len > max_tokens(P)) {
    if (threadIdx.x == 0) set_status(P.status, AKV_ERR_SHAPE);
    return make_int2(-1, 0);
  }
  return make_int2(seq, len);
}

AKV_DEV uint32_t score_order(float x) {
  if (x != x) return 0u;  // NaN: below all others
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

// ---------------------------------------------------------------- scores
__global__ void __launch_bounds__(256) evict_score_kernel(const EvictParams P) {
  const int i = blockIdx.y;
  const int seq = P.rows ? P.rows[i] : i;
  if (seq < 0 || seq >= P.T.max_seqs) return;
  const int len = P.T.lens[seq];
  if (len <= P.keep || len > max_tokens(P)) return;
  for (int t = blockIdx.x * 256 + threadIdx.x; t < len; t += gridDim.x * 256) {
    uint32_t k = 0xFFFFFFFFu;
    if (t >= P.first && t < len - P.recent) {
      const float* w = P.weights + seq * P.w_row + t;
      double sum = 0.0;
      int l = 0;
      for (; l + 8 <= P.n_layers; l += 8) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = w[(l + j) * P.w_layer];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[j];
      }
      for (; l < P.n_layers; ++l) sum += w[l * P.w_layer];
      k = score_order(__double2float_rn(sum));
    }
    P.score[static_cast<int64_t>(i) * max_tokens(P) + t] = k;
  }
}

// inclusive sum over the block; total gets the block's sum
AKV_DEV int select_scan(int x, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums may still be read from an earlier scan
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int s = lane < static_cast<int>(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(~0u, s, o);
    if (lane >= o) s += y;
  }
  total = __shfl_sync(~0u, s, 31);
  const int before = __shfl_sync(~0u, s, warp ? warp - 1 : 0);
  return x + (warp ? before : 0);
}

// ---------------------------------------------------------------- selection
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams P) {
  __shared__ int s_hist[256], s_warp[32];
  __shared__ int s_bin, s_above, s_first;
  const int i = blockIdx.x, t = threadIdx.x;
  if (t == 0) s_first = INT32_MAX;
  const int2 row = evict_row(P, i);
  const int seq = row.x, len = row.y;
  const int left = len < P.keep ? len : P.keep;
  int32_t* kept = P.kept + static_cast<int64_t>(i) * P.keep;
  for (int j = left + t; j < P.keep; j += kSelectThreads) kept[j] = -1;
  if (seq < 0 || len <= P.keep) {
    for (int j = t; j < left; j += kSelectThreads) kept[j] = j;
    if (t == 0) P.info[i] = EvictRow{seq, len, left, 0, 0, 0, 0, 0};
    return;
  }
  const uint32_t* key = P.score + static_cast<int64_t>(i) * max_tokens(P);
  // the keep-th largest key, a byte at a time from the top
  uint32_t prefix = 0;
  int want = P.keep;  // still to be found among the keys that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) s_hist[t] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
    for (int j = t; j < len; j += kSelectThreads) {
      const uint32_t k = key[j];
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    int total;
    const int mine = t < 256 ? s_hist[255 - t] : 0;  // from the largest byte down
    const int upto = select_scan(mine, s_warp, total);
    if (t < 256 && upto >= want && upto - mine < want) {
      s_bin = 255 - t;
      s_above = upto - mine;
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(s_bin) << shift;
    want -= s_above;
    __syncthreads();
  }
  // in order: the keys above it, and the first `want` equal to it; a thread takes a run of keys
  const int run = (len + 4 * kSelectThreads - 1) / (4 * kSelectThreads) * 4;
  const int j0 = t * run, j1 = min(len, j0 + run);
  int n_eq = 0, n_gt = 0;
  for (int j = j0; j < j1; j += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(key + j);
    const uint32_t k[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      n_eq += j + e < j1 && k[e] == prefix;
      n_gt += j + e < j1 && k[e] > prefix;
    }
  }
  int total;
  int equal = select_scan(n_eq, s_warp, total) - n_eq;  // before this run
  const int on = n_gt + max(0, min(n_eq, want - equal));
  int at = select_scan(on, s_warp, total) - on;
  for (int j = j0; j < j1; j += 4) {
    const uint4 q = *reinterpret_cast<const uint4*>(key + j);
    const uint32_t k[4] = {q.x, q.y, q.z, q.w};
    int gone = len;
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (j + e < j1 && k[e] < prefix) gone = j + e;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (j + e >= j1) continue;
      const bool stays = k[e] > prefix || (k[e] == prefix && equal < want);
      if (k[e] == prefix && ++equal > want) gone = min(gone, j + e);
      if (stays) kept[at++] = j + e;
    }
    if (gone < s_first) atomicMin(&s_first, gone);
  }
  __syncthreads();
  const int end = (left + kBlockTokens - 1) / kBlockTokens;
  const int start = s_first < left ? s_first / kBlockTokens : end;  // past the kept tokens: none moves
  int need = 0;
  for (int b0 = start; b0 < end; b0 += kSelectThreads) {
    const int b = b0 + t;
    const int p = b < end ? P.T.table[seq * P.T.table_stride + b] : -1;
    const bool ok = p >= 0 && p < P.T.n_pages, shared = ok && P.T.refs[p] > 1;
    if (b < end && !ok) set_status(P.status, AKV_ERR_SHAPE);
    int n;
    const int rank = need + select_scan(shared, s_warp, n) - shared;
    if (b < end) P.to[static_cast<int64_t>(i) * P.T.max_blocks + b] = shared ? -2 - rank : ok ? p : -1;
    need += n;
  }
  if (t == 0) P.info[i] = EvictRow{seq, len, left, start, end, need, 0, 0};
}

// Page that page b of call row i becomes: its own, or where that is shared one from
// the list, the row's -2 - to[b]-th; -1 for one that is no page.
AKV_DEV int new_page(const EvictParams& P, const EvictRow& r, int i, int b) {
  const int p = P.to[static_cast<int64_t>(i) * P.T.max_blocks + b];
  return p < -1 ? P.list[r.off - 2 - p] : p;
}

// ---------------------------------------------------------------- new pages
// The lowest free pages, in the order of the rows and of their pages, until the
// pool runs out: that row and all after it are refused.
__global__ void __launch_bounds__(kSelectThreads) evict_plan_kernel(const EvictParams P) {
  __shared__ int s_warp[32];
  __shared__ int s_found, s_base, s_fail;
  const int t = threadIdx.x, words = (P.T.n_pages + 31) / 32;
  if (t == 0) s_base = 0, s_fail = P.n;
  __syncthreads();
  // each row's place in the list
  for (int i0 = 0; i0 < P.n; i0 += kSelectThreads) {
    const int i = i0 + t;
    const int need = i < P.n ? P.info[i].need : 0;
    int total;
    const int upto = select_scan(need, s_warp, total);
    if (i < P.n) P.info[i].off = s_base + upto - need;
    __syncthreads();
    if (t == 0) s_base += total;
    __syncthreads();
  }
  const int total = s_base;
  if (t == 0) s_found = 0;
  __syncthreads();
  for (int base = 0; base < words && s_found < total; base += kSelectThreads) {
    const int w = base + t;
    uint32_t bits = w < words ? P.T.free_bits[w] : 0u;
    const int past = P.T.n_pages - w * 32;  // bits past the pool are no pages
    if (past < 32) bits &= past <= 0 ? 0u : (1u << past) - 1u;
    int sum;
    int rank = s_found + select_scan(__popc(bits), s_warp, sum) - __popc(bits);
    for (; bits && rank < total; bits &= bits - 1) P.list[rank++] = w * 32 + __ffs(bits) - 1;
    __syncthreads();
    if (t == 0) s_found += sum;
    __syncthreads();
  }
  const int have = s_found < total ? s_found : total;
  for (int i = t; i < P.n; i += kSelectThreads) {
    const EvictRow r = P.info[i];
    if (r.need > 0 && r.off + r.need > have) atomicMin(&s_fail, i);
  }
  __syncthreads();
  const int fail = s_fail;
  if (t == 0 && fail < P.n) set_status(P.status, AKV_ERR_EXHAUSTED);
  for (int i = fail + t; i < P.n; i += kSelectThreads) P.info[i].seq = -1;
  const int used = fail < P.n ? P.info[fail].off : total;
  for (int k = t; k < used; k += kSelectThreads) {
    const int p = P.list[k];
    atomicAnd(P.T.free_bits + (p >> 5), ~(1u << (p & 31)));
    P.T.refs[p] = 1;
  }
}

// ---------------------------------------------------------------- moves
template <int B>
struct MoveWord;
template <>
struct MoveWord<4> { using type = uint32_t; };
template <>
struct MoveWord<8> { using type = uint2; };
template <>
struct MoveWord<16> { using type = uint4; };

// Block x: K (even) or V of head x / 2; the last one the weights.
template <int D, int G, int NT>
__global__ void __launch_bounds__(NT) evict_move_kernel(const EvictParams P) {
  constexpr Int4Layout L = int4_layout(D, G);
  constexpr int CH = D / 32;                    // 16-byte pieces of a token's codes
  constexpr int TOK = NT * kMovePieces / CH;    // tokens of a step
  constexpr int PER = (TOK + NT - 1) / NT;      // tokens whose place and (scale, zero) pairs a thread takes
  using Pairs = typename MoveWord<G * 4>::type;
  __shared__ int2 s_from[2][TOK];               // page and slot of the step's sources
  __shared__ int s_to[2][TOK / kBlockTokens];
  const int t = threadIdx.x;
  const int layer = blockIdx.y, i = blockIdx.z;
  const EvictRow r = P.info[i];
  if (r.seq < 0 || r.start >= r.end) return;
  const int32_t* kept = P.kept + static_cast<int64_t>(i) * P.keep;
  const int first = r.start * kBlockTokens;
  if (blockIdx.x == 2 * P.kv_heads) {  // the weights move like a head
    float* w = P.weights + layer * P.w_layer + r.seq * P.w_row;
    for (int j0 = first; j0 < r.left; j0 += 4 * NT) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * NT + t;
        v[k] = j < r.left ? w[kept[j]] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * NT + t;
        if (j < r.left) w[j] = v[k];
      }
    }
    return;
  }
  const int32_t* table = P.T.table + r.seq * P.T.table_stride;
  const bool is_v = blockIdx.x & 1;
  uint8_t* pool = P.pool + layer * P.layer_stride + (blockIdx.x >> 1) * static_cast<int64_t>(L.bytes);
  uint8_t* codes = pool + (is_v ? L.vc : L.kc);
  uint8_t* pairs = pool + (is_v ? L.vp : L.kp);
  // where the tokens of a step come from and go to; page -1: nowhere
  auto places = [&](int j0, int buf) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int x = k * NT + t, j = j0 + x;
      if (x >= TOK) break;
      int2 from = make_int2(-1, 0);
      if (j < r.left) {
        const int src = kept[j], p = table[src / kBlockTokens];
        if (p >= 0 && p < P.T.n_pages) from = make_int2(p, src % kBlockTokens);
        else set_status(P.status, AKV_ERR_SHAPE);
      }
      s_from[buf][x] = from;
    }
    if (t < TOK / kBlockTokens) {
      const int b = j0 / kBlockTokens + t;
      s_to[buf][t] = b < r.end ? new_page(P, r, i, b) : -1;
    }
  };
  places(first, 0);
  int buf = 0;
  for (int j0 = first; j0 < r.left; j0 += TOK, buf ^= 1) {
    __syncthreads();  // the places stand; the last step's writes are behind its reads
    uint4 c[kMovePieces];
    Pairs z[PER];
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) {
      const int x = k * NT + t;
      const int2 from = s_from[buf][x / CH];
      if (from.x >= 0) c[k] = *reinterpret_cast<const uint4*>(codes + from.x * P.page_bytes + from.y * (D / 2) + x % CH * 16);
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int x = k * NT + t;
      if (x >= TOK) break;
      const int2 from = s_from[buf][x];
      if (from.x >= 0) z[k] = *reinterpret_cast<const Pairs*>(pairs + from.x * P.page_bytes + from.y * (G * 4));
    }
    if (j0 + TOK < r.left) places(j0 + TOK, buf ^ 1);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kMovePieces; ++k) {
      const int x = k * NT + t, y = x / CH, p = s_to[buf][y / kBlockTokens];
      if (p >= 0 && s_from[buf][y].x >= 0)
        *reinterpret_cast<uint4*>(codes + p * P.page_bytes + y % kBlockTokens * (D / 2) + x % CH * 16) = c[k];
    }
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int x = k * NT + t;
      if (x >= TOK) break;
      const int p = s_to[buf][x / kBlockTokens];
      if (p >= 0 && s_from[buf][x].x >= 0)
        *reinterpret_cast<Pairs*>(pairs + p * P.page_bytes + x % kBlockTokens * (G * 4)) = z[k];
    }
  }
}

// ---------------------------------------------------------------- tables
__global__ void __launch_bounds__(256) evict_finish_kernel(const EvictParams P) {
  const int i = blockIdx.x, t = threadIdx.x;
  const EvictRow r = P.info[i];
  if (r.seq < 0) {
    for (int j = t; j < P.keep; j += 256) P.kept[static_cast<int64_t>(i) * P.keep + j] = -1;
    return;
  }
  if (r.left == r.len) return;
  int32_t* table = P.T.table + r.seq * P.T.table_stride;
  const int pages = (r.len + kBlockTokens - 1) / kBlockTokens;
  for (int b = r.start + t; b < pages; b += 256) {
    const int old = table[b], now = b < r.end ? new_page(P, r, i, b) : -1;
    if (old == now) continue;
    table[b] = now;
    if (old < 0 || old >= P.T.n_pages) {
      set_status(P.status, AKV_ERR_SHAPE);
      continue;
    }
    if (atomicSub(P.T.refs + old, 1) == 1) atomicOr(P.T.free_bits + (old >> 5), 1u << (old & 31));
  }
  if (t == 0) P.T.lens[r.seq] = r.left;
}

// ---------------------------------------------------------------- weights of new and forked tokens
// 0 for the last n_new[i] tokens of row rows[i], in every layer
__global__ void __launch_bounds__(128) weights_clear_kernel(float* weights, int64_t w_layer, int64_t w_row, int n_layers,
                                                            const int32_t* lens, int max_seqs, int max_tok,
                                                            const int32_t* rows, const int32_t* n_new) {
  const int i = blockIdx.x, seq = rows ? rows[i] : i;
  if (seq < 0 || seq >= max_seqs) return;
  const int add = n_new[i], len = lens[seq];
  if (add <= 0 || len < add || len > max_tok) return;
  for (int l = blockIdx.y; l < n_layers; l += gridDim.y)
    for (int t = len - add + threadIdx.x; t < len; t += 128) weights[l * w_layer + seq * w_row + t] = 0.f;
}

// an empty row takes the weights of the row that it is about to be forked from
__global__ void __launch_bounds__(128) weights_fork_kernel(float* weights, int64_t w_layer, int64_t w_row, int n_layers,
                                                           const int32_t* lens, int max_seqs, int max_tok,
                                                           const int32_t* parents, const int32_t* children) {
  const int i = blockIdx.x, par = parents[i], kid = children[i];
  if (par < 0 || par >= max_seqs || kid < 0 || kid >= max_seqs || par == kid || lens[kid] != 0) return;
  bool again = false;  // the first of two requests for a row counts
  for (int s = threadIdx.x; s < i; s += 128) again |= children[s] == kid;
  if (__syncthreads_or(again)) return;
  const int len = lens[par];
  if (len < 0 || len > max_tok) return;
  for (int l = blockIdx.y; l < n_layers; l += gridDim.y)
    for (int t = threadIdx.x; t < len; t += 128)
      weights[l * w_layer + kid * w_row + t] = weights[l * w_layer + par * w_row + t];
}

static int evict_launched() { return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH; }

template <int D, int NT>
static void launch_move(const EvictParams& P, cudaStream_t st) {
  const dim3 grid(2 * P.kv_heads + 1, P.n_layers, P.n);
  switch (P.n_groups) {
    case 1: evict_move_kernel<D, 1, NT><<<grid, NT, 0, st>>>(P); break;
    case 2: evict_move_kernel<D, 2, NT><<<grid, NT, 0, st>>>(P); break;
    default: evict_move_kernel<D, 4, NT><<<grid, NT, 0, st>>>(P); break;
  }
}

static size_t up16(size_t x) { return (x + 15) / 16 * 16; }

static int weights_check(const float* w, int64_t w_layer, int64_t w_row, int n_layers, int max_blocks) {
  if (!w) return AKV_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(w) & 3) return AKV_ERR_ALIGN;
  if (n_layers <= 0 || n_layers > 65535 || w_layer < 0 || w_row < static_cast<int64_t>(max_blocks) * kBlockTokens)
    return AKV_ERR_SHAPE;
  return AKV_OK;
}

static int rows_check(const akv_page_table* t) {
  if (!t || !t->table || !t->lens || !t->refs || !t->free_bits) return AKV_ERR_NULL;
  if (t->max_seqs <= 0 || t->max_blocks <= 0 || t->n_pages <= 0 || t->table_stride < t->max_blocks)
    return AKV_ERR_SHAPE;
  return t->max_blocks > (1 << 20) ? AKV_ERR_UNSUPPORTED : AKV_OK;
}

}  // namespace akv

using namespace akv;

extern "C" size_t akv_int4_evict_workspace_bytes(int n, int max_blocks, int n_pages) {
  if (n <= 0 || max_blocks <= 0 || max_blocks > (1 << 20) || n_pages <= 0) return 0;
  const size_t rows = static_cast<size_t>(n);
  return up16(rows * sizeof(EvictRow)) + up16(rows * max_blocks * kBlockTokens * 4) +
         up16(static_cast<size_t>(n_pages) * 4) + up16(rows * max_blocks * 4);
}

extern "C" int akv_int4_evict(const akv_int4_evict_args* a, void* stream) {
  if (!a) return AKV_ERR_NULL;
  int rc = rows_check(a->table);
  if (rc) return rc;
  const akv_page_table& T = *a->table;
  if ((rc = weights_check(a->weights, a->w_layer, a->w_row, a->n_layers, T.max_blocks))) return rc;
  if (a->n < 0 || a->n > 65535 || a->keep <= 0 || a->first < 0 || a->recent < 0 ||
      static_cast<int64_t>(a->first) + a->recent > a->keep || a->kv_heads <= 0)
    return AKV_ERR_SHAPE;
  if (!int4_shape_ok(a->head_dim, a->group)) return AKV_ERR_SHAPE;
  if (!a->pool) return AKV_ERR_NULL;
  const Int4Layout L = int4_layout(a->head_dim, a->head_dim / a->group);
  if (a->page_bytes != static_cast<int64_t>(L.bytes) * a->kv_heads) return AKV_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->pool) | static_cast<uintptr_t>(a->layer_stride)) & 15) return AKV_ERR_ALIGN;
  if (a->n == 0) return AKV_OK;
  if (!a->kept || !a->workspace) return AKV_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return AKV_ERR_ALIGN;
  if (a->workspace_bytes < akv_int4_evict_workspace_bytes(a->n, T.max_blocks, T.n_pages)) return AKV_ERR_WORKSPACE;
  EvictParams p{};
  p.T = T;
  p.pool = a->pool;
  p.layer_stride = a->layer_stride;
  p.page_bytes = a->page_bytes;
  p.n_layers = a->n_layers;
  p.kv_heads = a->kv_heads;
  p.head_dim = a->head_dim;
  p.n_groups = a->head_dim / a->group;
  p.weights = a->weights;
  p.w_layer = a->w_layer;
  p.w_row = a->w_row;
  p.rows = a->rows;
  p.n = a->n;
  p.keep = a->keep;
  p.first = a->first;
  p.recent = a->recent;
  p.kept = a->kept;
  p.status = a->status;
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  p.info = reinterpret_cast<EvictRow*>(ws);
  ws += up16(sizeof(EvictRow) * static_cast<size_t>(a->n));
  p.score = reinterpret_cast<uint32_t*>(ws);
  ws += up16(static_cast<size_t>(a->n) * T.max_blocks * kBlockTokens * 4);
  p.list = reinterpret_cast<int32_t*>(ws);
  ws += up16(static_cast<size_t>(T.n_pages) * 4);
  p.to = reinterpret_cast<int32_t*>(ws);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int most = (T.max_blocks * kBlockTokens + 255) / 256;
  evict_score_kernel<<<dim3(most < 256 ? most : 256, a->n), 256, 0, st>>>(p);
  evict_select_kernel<<<a->n, kSelectThreads, 0, st>>>(p);
  evict_plan_kernel<<<1, kSelectThreads, 0, st>>>(p);
  // few blocks: more threads each, so that a block's steps, one after the other,
  // are fewer: 112 blocks 54 -> 45 us; 4,096 blocks 247 -> 259 us
  const bool few = static_cast<int64_t>(a->n) * a->n_layers * a->kv_heads * 2 <= 148 * 2;
  switch (a->head_dim) {
    case 64: few ? launch_move<64, 1024>(p, st) : launch_move<64, 256>(p, st); break;
    case 128: few ? launch_move<128, 1024>(p, st) : launch_move<128, 256>(p, st); break;
    default: few ? launch_move<256, 1024>(p, st) : launch_move<256, 256>(p, st); break;
  }
  evict_finish_kernel<<<a->n, 256, 0, st>>>(p);
  return evict_launched();
}

extern "C" int akv_int4_weights_clear(const akv_page_table* t, float* weights, int64_t w_layer, int64_t w_row,
                                      int n_layers, const int32_t* rows, const int32_t* n_new, int n, void* stream) {
  int rc = rows_check(t);
  if (rc) return rc;
  if ((rc = weights_check(weights, w_layer, w_row, n_layers, t->max_blocks))) return rc;
  if (n < 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  if (!n_new) return AKV_ERR_NULL;
  weights_clear_kernel<<<dim3(n, n_layers < 16 ? n_layers : 16), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      weights, w_layer, w_row, n_layers, t->lens, t->max_seqs, t->max_blocks * kBlockTokens, rows, n_new);
  return evict_launched();
}

extern "C" int akv_int4_weights_fork(const akv_page_table* t, float* weights, int64_t w_layer, int64_t w_row,
                                     int n_layers, const int32_t* parents, const int32_t* children, int n,
                                     void* stream) {
  int rc = rows_check(t);
  if (rc) return rc;
  if ((rc = weights_check(weights, w_layer, w_row, n_layers, t->max_blocks))) return rc;
  if (n < 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  if (!parents || !children) return AKV_ERR_NULL;
  weights_fork_kernel<<<dim3(n, n_layers < 64 ? n_layers : 64), 128, 0, static_cast<cudaStream_t>(stream)>>>(
      weights, w_layer, w_row, n_layers, t->lens, t->max_seqs, t->max_blocks * kBlockTokens, parents, children);
  return evict_launched();
}
