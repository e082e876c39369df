// Eviction from the 4-bit paged cache by accumulated attention weight.
//
//   score[t] = fp32(sum over layers of weights[l][s][t], summed in fp64)
// (one rounding: the order of the layers does not decide a tie), the first
// `first` and last `recent` tokens above all others; the `keep` largest stay,
// the lowest token first among equal ones, and move together in their order, in
// every layer and head.
//
// Five steps, each a launch: scores; the keep-th largest score by a radix
// select and the list of the kept tokens, a CTA a row; pages for those that are
// shared and would be written (their other holders keep them), in the order of
// the rows; the moves; tables, lengths and reference counts.
//
// Moves in place.  The kept tokens of page j come from pages >= j, so taking
// the pages in ascending order a CTA may read ahead freely; it only has to have
// read all of a page's sources before it writes that page.  A CTA owns one
// (row, layer, head) and its four pages at a time stand in registers between
// read and write; rows x layers x heads run side by side.  Pages before the
// first token that goes are left alone.
#include "int4.cuh"

namespace akv {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kMovePages = 4;
constexpr int kMoveTokens = kMovePages * kBlockTokens;

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
  int32_t* to;       // [n][max_blocks] page each page of the row becomes
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
  __shared__ int s_bin, s_above, s_first, s_need;
  const int i = blockIdx.x, t = threadIdx.x;
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
  // in order: the keys above it, and the first `want` equal to it
  if (t == 0) s_first = len, s_need = 0;
  int out = 0, equal = 0;
  for (int j0 = 0; j0 < len; j0 += kSelectThreads) {
    const int j = j0 + t;
    const uint32_t k = j < len ? key[j] : 0u;
    const bool eq = j < len && k == prefix, gt = j < len && k > prefix;
    int n_eq, n_on;
    const int before = select_scan(eq, s_warp, n_eq) - eq + equal;
    const bool on = gt || (eq && before < want);
    const int at = select_scan(on, s_warp, n_on) - on + out;
    if (on) kept[at] = j;
    else if (j < len) atomicMin(&s_first, j);
    out += n_on;
    equal += n_eq;
  }
  __syncthreads();
  const int end = (left + kBlockTokens - 1) / kBlockTokens;
  const int start = s_first < left ? s_first / kBlockTokens : end;  // past the kept tokens: none moves
  int need = 0;
  for (int b = start + t; b < end; b += kSelectThreads) {
    const int p = P.T.table[seq * P.T.table_stride + b];
    if (p >= 0 && p < P.T.n_pages) need += P.T.refs[p] > 1;
  }
  if (need) atomicAdd(&s_need, need);
  __syncthreads();
  if (t == 0) P.info[i] = EvictRow{seq, len, left, start, end, s_need, 0, 0};
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
// Page that page b of the row becomes: its own, or a new one where it is shared.
__global__ void __launch_bounds__(kSelectThreads) evict_target_kernel(const EvictParams P) {
  __shared__ int s_warp[32];
  const int i = blockIdx.x, t = threadIdx.x;
  const EvictRow r = P.info[i];
  if (r.seq < 0) {
    for (int j = t; j < P.keep; j += kSelectThreads) P.kept[static_cast<int64_t>(i) * P.keep + j] = -1;
    return;
  }
  int taken = r.off;
  for (int b0 = r.start; b0 < r.end; b0 += kSelectThreads) {
    const int b = b0 + t;
    const int p = b < r.end ? P.T.table[r.seq * P.T.table_stride + b] : -1;
    const bool ok = p >= 0 && p < P.T.n_pages, shared = ok && r.need > 0 && P.T.refs[p] > 1;
    if (b < r.end && !ok) set_status(P.status, AKV_ERR_SHAPE);
    int total;
    const int rank = select_scan(shared, s_warp, total) - shared;
    if (b < r.end) P.to[static_cast<int64_t>(i) * P.T.max_blocks + b] = shared ? P.list[taken + rank] : (ok ? p : -1);
    taken += total;
  }
}

template <int D, int G>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictParams P) {
  constexpr Int4Layout L = int4_layout(D, G);
  constexpr int CH = D / 32;                 // 16-byte pieces of a token's K (V) codes
  constexpr int PIECES = kMoveTokens * CH / kMoveThreads * 2;
  constexpr int PAIRS = kMoveTokens * G * 2; // 4-byte (scale, zero) pairs, K then V
  constexpr int PW = (PAIRS + kMoveThreads - 1) / kMoveThreads;
  const int t = threadIdx.x;
  const int h = blockIdx.x, layer = blockIdx.y, i = blockIdx.z;
  const EvictRow r = P.info[i];
  if (r.seq < 0 || r.start >= r.end) return;
  const int32_t* kept = P.kept + static_cast<int64_t>(i) * P.keep;
  if (h == P.kv_heads) {  // the weights move like a head
    float* w = P.weights + layer * P.w_layer + r.seq * P.w_row;
    for (int j0 = r.start * kBlockTokens; j0 < r.left; j0 += 4 * kMoveThreads) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * kMoveThreads + t;
        v[k] = j < r.left ? w[kept[j]] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = j0 + k * kMoveThreads + t;
        if (j < r.left) w[j] = v[k];
      }
    }
    return;
  }
  const int32_t* table = P.T.table + r.seq * P.T.table_stride;
  const int32_t* to = P.to + static_cast<int64_t>(i) * P.T.max_blocks;
  uint8_t* pool = P.pool + layer * P.layer_stride + h * static_cast<int64_t>(L.bytes);
  auto record = [&](const int32_t* pages, int tok) -> uint8_t* {
    const int p = pages[tok / kBlockTokens];
    return p >= 0 && p < P.T.n_pages ? pool + p * P.page_bytes : nullptr;
  };
  for (int j0 = r.start * kBlockTokens; j0 < r.left; j0 += kMoveTokens) {
    uint4 c[PIECES];
    uint32_t z[PW];
    // thread t: piece t % CH of token t / CH and every (kMoveThreads / CH)-th on
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int v = k >= PIECES / 2, x = (v ? k - PIECES / 2 : k) * kMoveThreads + t;
      const int j = j0 + x / CH;
      if (j < r.left) {
        const int src = kept[j];
        const uint8_t* rec = record(table, src);
        if (rec) c[k] = *reinterpret_cast<const uint4*>(rec + (v ? L.vc : L.kc) + src % kBlockTokens * (D / 2) + x % CH * 16);
        else set_status(P.status, AKV_ERR_SHAPE);
      }
    }
#pragma unroll
    for (int k = 0; k < PW; ++k) {
      const int x = k * kMoveThreads + t, v = x >= PAIRS / 2, y = v ? x - PAIRS / 2 : x;
      const int j = j0 + y / G;
      if (x < PAIRS && j < r.left) {
        const int src = kept[j];
        const uint8_t* rec = record(table, src);
        if (rec) z[k] = *reinterpret_cast<const uint32_t*>(rec + (v ? L.vp : L.kp) + (src % kBlockTokens * G + y % G) * 4);
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int v = k >= PIECES / 2, x = (v ? k - PIECES / 2 : k) * kMoveThreads + t;
      const int j = j0 + x / CH;
      if (j < r.left) {
        uint8_t* rec = record(to, j);
        if (rec && record(table, kept[j]))
          *reinterpret_cast<uint4*>(rec + (v ? L.vc : L.kc) + j % kBlockTokens * (D / 2) + x % CH * 16) = c[k];
      }
    }
#pragma unroll
    for (int k = 0; k < PW; ++k) {
      const int x = k * kMoveThreads + t, v = x >= PAIRS / 2, y = v ? x - PAIRS / 2 : x;
      const int j = j0 + y / G;
      if (x < PAIRS && j < r.left) {
        uint8_t* rec = record(to, j);
        if (rec && record(table, kept[j]))
          *reinterpret_cast<uint32_t*>(rec + (v ? L.vp : L.kp) + (j % kBlockTokens * G + y % G) * 4) = z[k];
      }
    }
  }
}

// ---------------------------------------------------------------- tables
__global__ void __launch_bounds__(256) evict_finish_kernel(const EvictParams P) {
  const int i = blockIdx.x, t = threadIdx.x;
  const EvictRow r = P.info[i];
  if (r.seq < 0 || r.left == r.len) return;
  int32_t* table = P.T.table + r.seq * P.T.table_stride;
  const int pages = (r.len + kBlockTokens - 1) / kBlockTokens;
  for (int b = r.start + t; b < pages; b += 256) {
    const int old = table[b], now = b < r.end ? P.to[static_cast<int64_t>(i) * P.T.max_blocks + b] : -1;
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

template <int D>
static void launch_move(const EvictParams& P, cudaStream_t st) {
  const dim3 grid(P.kv_heads + 1, P.n_layers, P.n);
  switch (P.n_groups) {
    case 1: evict_move_kernel<D, 1><<<grid, kMoveThreads, 0, st>>>(P); break;
    case 2: evict_move_kernel<D, 2><<<grid, kMoveThreads, 0, st>>>(P); break;
    default: evict_move_kernel<D, 4><<<grid, kMoveThreads, 0, st>>>(P); break;
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
  evict_target_kernel<<<a->n, kSelectThreads, 0, st>>>(p);
  switch (a->head_dim) {
    case 64: launch_move<64>(p, st); break;
    case 128: launch_move<128>(p, st); break;
    default: launch_move<256>(p, st); break;
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
