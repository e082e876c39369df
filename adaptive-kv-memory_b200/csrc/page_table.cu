// Page ownership of a paged cache, kept on the device: fork, reserve (copy on
// write), truncate, compact, copy.
//
// Integer bookkeeping around page copies.  A page has refs[p] holders; a page
// with none has its bit set in free_bits.  Allocation is deterministic: the
// free pages are taken lowest first, in the order of the requests, which a
// prefix sum over the popcounts of free_bits gives (one bit a page, so one
// CTA reads the state of 32,768 pages with one load per thread).
//
// The copies are bound by memory: 256 pages of 34.8 KB in 16 layers (285 MB
// read and written) in 34 us, the writes partly still in L2; a compaction that
// moves 428 MB in 68 us (6.3 TB/s).  The plans are one CTA's latencies, 9 to
// 14 us for 5 to 288 requests or 8,192 pages.
#include "int4.cuh"

namespace akv {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;                                     // 16-byte pieces in flight per thread
constexpr int kCopyChunk = kCopyThreads * kCopyUnroll * 16;        // bytes per work item

// workspace: count, then src / dst pairs, then one int per page
struct PageWs {
  int32_t* count;
  int32_t* src;
  int32_t* dst;
  int32_t* list;
};

__host__ __device__ inline size_t page_ws_pairs(int n_pages, int n) { return n > n_pages ? n : n_pages; }

inline PageWs page_ws(void* ws, int n_pages, int n) {
  PageWs w;
  const size_t m = page_ws_pairs(n_pages, n);
  w.count = static_cast<int32_t*>(ws);
  w.src = w.count + 4;
  w.dst = w.src + m;
  w.list = w.dst + m;
  return w;
}

// inclusive sum over the block; total gets the block's sum
AKV_DEV int block_scan(int x, int* warp_sums, int& total) {
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

AKV_DEV uint32_t page_mask(int w, int n_pages) {  // the bits of word w that are pages
  const int left = n_pages - w * 32;
  return left >= 32 ? ~0u : (left <= 0 ? 0u : (1u << left) - 1u);
}

// ---------------------------------------------------------------- reserve
// Requests go through 1,024 at a time, in order; what one round takes, copies
// and refuses the next one sees (free bits and reference counts are read from
// L2, where this CTA's atomics change them).
__global__ void __launch_bounds__(kPlanThreads) reserve_plan_kernel(akv_page_table T, const int32_t* rows,
                                                                    const int32_t* n_new, int n_new_all, int n_all,
                                                                    int32_t* granted, PageWs ws, int* status) {
  __shared__ int s_row[kPlanThreads], s_page[kPlanThreads], s_off[kPlanThreads + 1], s_block[kPlanThreads];
  __shared__ int s_warp[32];
  __shared__ int s_found, s_fail, s_copies;
  const int t = threadIdx.x;
  const int words = (T.n_pages + 31) / 32;
  if (t == 0) s_copies = 0;
  int first = 0;
  for (; first < n_all; first += kPlanThreads) {
    const int n = n_all - first < kPlanThreads ? n_all - first : kPlanThreads, i = first + t;
    // the request of this thread
    int row = -1, add = 0, len = 0, nb0 = 0, nb1 = 0, last = -1;
    bool ok = false, part = false;
    if (t < n) {
      row = rows ? rows[i] : i;
      add = n_new ? n_new[i] : n_new_all;
      ok = row >= 0 && row < T.max_seqs && add >= 0;
    }
    s_row[t] = row;
    if (t == 0) s_found = 0, s_fail = n;
    if (ok) {
      len = T.lens[row];
      const int64_t end = static_cast<int64_t>(len) + add;
      ok = len >= 0 && (end + kBlockTokens - 1) / kBlockTokens <= T.max_blocks;
      if (ok) {
        nb0 = (len + kBlockTokens - 1) / kBlockTokens;
        nb1 = static_cast<int>((end + kBlockTokens - 1) / kBlockTokens);
        part = add > 0 && len % kBlockTokens != 0;
        if (part) {
          last = T.table[row * T.table_stride + nb0 - 1];
          ok = last >= 0 && last < T.n_pages;
        }
      }
    }
    __syncthreads();
    if (ok && rows) {
      bool twice = false;
      for (int s = 0; s < first; ++s) twice |= rows[s] == row;
      for (int s = 0; s < t; ++s) twice |= s_row[s] == row;
      ok = !twice;
    }
    if (!ok) {
      if (t < n) set_status(status, AKV_ERR_SHAPE);
      add = nb0 = nb1 = 0;
      part = false;
    }
    s_page[t] = part ? last : -1;
    __syncthreads();
    bool cow = false;
    if (part) {  // earlier requests that share this page leave it before this one
      int before = 0;
      for (int s = 0; s < t; ++s) before += s_page[s] == last;
      cow = __ldcg(T.refs + last) - before > 1;
    }
    const int need = nb1 - nb0 + (cow ? 1 : 0);
    int total;
    const int off = block_scan(need, s_warp, total) - need;
    s_off[t] = off;
    s_block[t] = nb0 - (cow ? 1 : 0);
    // the first `total` free pages, lowest first
    for (int base = 0; base < words; base += kPlanThreads) {
      const int w = base + t;
      // a bit past the pool, of a state from elsewhere, is no page
      uint32_t bits = w < words ? __ldcg(T.free_bits + w) & page_mask(w, T.n_pages) : 0u;
      int sum;
      int rank = s_found + block_scan(__popc(bits), s_warp, sum) - __popc(bits);
      while (bits && rank < total) {
        ws.list[rank++] = w * 32 + __ffs(bits) - 1;
        bits &= bits - 1;
      }
      __syncthreads();
      if (t == 0) s_found += sum;
      __syncthreads();
      if (s_found >= total) break;
    }
    const int have = s_found < total ? s_found : total;
    // in order until the pool runs out
    if (t < n && need > 0 && off + need > have) atomicMin(&s_fail, t);
    __syncthreads();
    const int fail = s_fail;
    const int used = fail < n ? s_off[fail] : total;
    if (t == 0 && fail < n) set_status(status, AKV_ERR_EXHAUSTED);
    if (t < n) granted[i] = t < fail ? add : 0;
    if (t < fail && ok) {
      T.lens[row] = len + add;
      if (cow) {
        const int k = atomicAdd(&s_copies, 1);
        ws.src[k] = last;
        ws.dst[k] = ws.list[off];
        atomicSub(T.refs + last, 1);
      }
    }
    for (int k = t; k < used; k += kPlanThreads) {
      const int page = ws.list[k];
      atomicAnd(T.free_bits + (page >> 5), ~(1u << (page & 31)));
      T.refs[page] = 1;
      int lo = 0, hi = n;  // the last request whose first page is at or before k
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_off[mid] <= k) lo = mid; else hi = mid;
      }
      T.table[s_row[lo] * T.table_stride + s_block[lo] + (k - s_off[lo])] = page;
    }
    __syncthreads();
    if (fail < n) break;
  }
  // the pool ran out: whatever follows is refused
  for (int i = first + kPlanThreads + t; i < n_all; i += kPlanThreads) granted[i] = 0;
  if (t == 0) *ws.count = s_copies;
}

// ---------------------------------------------------------------- page copies
// Pairs (src[i], dst[i]), i < *count, in every layer, as a grid-stride loop
// over 16 KB pieces; first, for compaction, the table entries above *n_live
// are renamed (remap non-null).
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(uint8_t* pool, int n_layers, int64_t layer_stride,
                                                                  int64_t page_bytes, const int32_t* src,
                                                                  const int32_t* dst, const int32_t* count, int n_fixed,
                                                                  int n_pages, int32_t* table, int64_t table_stride,
                                                                  int max_seqs, int max_blocks, const int32_t* remap,
                                                                  const int32_t* n_live, int* status) {
  if (remap) {
    const int live = *n_live;
    const int64_t entries = static_cast<int64_t>(max_seqs) * max_blocks;
    for (int64_t e = blockIdx.x * static_cast<int64_t>(kCopyThreads) + threadIdx.x; e < entries;
         e += static_cast<int64_t>(gridDim.x) * kCopyThreads) {
      int32_t* at = table + (e / max_blocks) * table_stride + e % max_blocks;
      const int p = *at;
      if (p >= live && p < n_pages) *at = remap[p];
    }
  }
  const int64_t n = count ? *count : n_fixed;
  const int64_t pieces = (page_bytes + kCopyChunk - 1) / kCopyChunk;
  const int64_t items = n * n_layers * pieces;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t piece = it % pieces, rest = it / pieces;
    const int64_t pair = rest / n_layers, layer = rest % n_layers;
    const int a = src[pair], b = dst[pair];
    if (a < 0 || a >= n_pages || b < 0 || b >= n_pages) {
      if (threadIdx.x == 0) set_status(status, AKV_ERR_SHAPE);
      continue;
    }
    const int64_t at = piece * kCopyChunk;
    const uint8_t* from = pool + layer * layer_stride + a * page_bytes + at;
    uint8_t* to = pool + layer * layer_stride + b * page_bytes + at;
    const int64_t left = page_bytes - at;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k) {
      const int o = (k * kCopyThreads + threadIdx.x) * 16;
      if (o < left) v[k] = __ldcs(reinterpret_cast<const uint4*>(from + o));
    }
#pragma unroll
    for (int k = 0; k < kCopyUnroll; ++k) {
      const int o = (k * kCopyThreads + threadIdx.x) * 16;
      if (o < left) *reinterpret_cast<uint4*>(to + o) = v[k];
    }
  }
}

// ---------------------------------------------------------------- fork
__global__ void __launch_bounds__(128) fork_kernel(akv_page_table T, const int32_t* parents, const int32_t* children,
                                                   int n, int* status) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int par = parents[i], kid = children[i];
  bool bad = par < 0 || par >= T.max_seqs || kid < 0 || kid >= T.max_seqs;
  for (int s = t; s < n; s += 128) {
    const int c = children[s];
    bad |= c == par || (s < i && c == kid);
  }
  int len = 0;
  if (!bad) {
    len = T.lens[par];
    bad = T.lens[kid] != 0 || len < 0 || len > T.max_blocks * kBlockTokens;
  }
  if (__syncthreads_or(bad)) {
    if (t == 0) set_status(status, AKV_ERR_SHAPE);
    return;
  }
  const int nb = (len + kBlockTokens - 1) / kBlockTokens;
  for (int j = t; j < nb; j += 128) {
    const int p = T.table[par * T.table_stride + j];
    T.table[kid * T.table_stride + j] = p;
    if (p >= 0 && p < T.n_pages) atomicAdd(T.refs + p, 1);
    else set_status(status, AKV_ERR_SHAPE);
  }
  if (t == 0) T.lens[kid] = len;
}

// ---------------------------------------------------------------- truncate
__global__ void __launch_bounds__(128) truncate_kernel(akv_page_table T, const int32_t* rows, const int32_t* new_lens,
                                                       int* status) {
  const int i = blockIdx.x, t = threadIdx.x;
  const int row = rows ? rows[i] : i;
  bool bad = row < 0 || row >= T.max_seqs;
  if (rows)
    for (int s = t; s < i; s += 128) bad |= rows[s] == row;
  const int keep = new_lens ? new_lens[i] : 0;
  const int len = bad ? 0 : T.lens[row];
  bad |= keep < 0 || keep > len || len > T.max_blocks * kBlockTokens;
  if (__syncthreads_or(bad)) {
    if (t == 0) set_status(status, AKV_ERR_SHAPE);
    return;
  }
  const int nb0 = (keep + kBlockTokens - 1) / kBlockTokens, nb1 = (len + kBlockTokens - 1) / kBlockTokens;
  for (int j = nb0 + t; j < nb1; j += 128) {
    int32_t* at = T.table + row * T.table_stride + j;
    const int p = *at;
    *at = -1;
    if (p < 0 || p >= T.n_pages) {
      set_status(status, AKV_ERR_SHAPE);
      continue;
    }
    if (atomicSub(T.refs + p, 1) == 1) atomicOr(T.free_bits + (p >> 5), 1u << (p & 31));
  }
  if (t == 0) T.lens[row] = keep;
}

// ---------------------------------------------------------------- compact
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(akv_page_table T, int32_t* n_live, PageWs ws) {
  __shared__ int s_warp[32];
  __shared__ int s_below;  // live pages below n_live
  const int t = threadIdx.x;
  const int words = (T.n_pages + 31) / 32;
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = t * per, w1 = w0 + per < words ? w0 + per : words;
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(~T.free_bits[w] & page_mask(w, T.n_pages));
  int live;
  const int before = block_scan(mine, s_warp, live) - mine;
  const int wl = live >> 5;
  if (t == 0) s_below = live;  // when every page is live
  __syncthreads();
  if (wl >= w0 && wl < w1) {
    int b = before;
    for (int w = w0; w < wl; ++w) b += __popc(~T.free_bits[w] & page_mask(w, T.n_pages));
    s_below = b + __popc(~T.free_bits[wl] & page_mask(wl, T.n_pages) & ((1u << (live & 31)) - 1u));
  }
  __syncthreads();
  const int below = s_below, moves = live - below;
  int lb = before;  // live pages before the current word
  for (int w = w0; w < w1; ++w) {
    const uint32_t mask = page_mask(w, T.n_pages);
    const uint32_t on = ~T.free_bits[w] & mask;
    // pages of this word that stay below n_live
    const uint32_t low = w < wl ? ~0u : (w > wl ? 0u : (1u << (live & 31)) - 1u);
    for (uint32_t b = ~on & mask & low; b; b &= b - 1) {
      const int k = __ffs(b) - 1;
      ws.dst[w * 32 + k - lb - __popc(on & ((1u << k) - 1u))] = w * 32 + k;
    }
    for (uint32_t b = on & ~low; b; b &= b - 1) {
      const int k = __ffs(b) - 1;
      ws.src[lb + __popc(on & ((1u << k) - 1u)) - below] = w * 32 + k;
    }
    lb += __popc(on);
    T.free_bits[w] = mask & ~low;
  }
  __syncthreads();
  for (int i = t; i < moves; i += kPlanThreads) {
    const int a = ws.src[i], b = ws.dst[i];
    ws.list[a] = b;
    T.refs[b] = T.refs[a];
    T.refs[a] = 0;
  }
  if (t == 0) {
    *ws.count = moves;
    *n_live = live;
  }
}

}  // namespace akv

using namespace akv;

static int table_check(const akv_page_table* t) {
  if (!t || !t->table || !t->lens || !t->refs || !t->free_bits) return AKV_ERR_NULL;
  if (t->max_seqs <= 0 || t->max_blocks <= 0 || t->n_pages <= 0 || t->table_stride < t->max_blocks)
    return AKV_ERR_SHAPE;
  if (t->max_blocks > (1 << 20)) return AKV_ERR_UNSUPPORTED;  // the plan's page sums are 32-bit
  return AKV_OK;
}

static int pool_check(const uint8_t* pool, int n_layers, int64_t layer_stride, int64_t page_bytes) {
  if (!pool) return AKV_ERR_NULL;
  if (n_layers <= 0 || page_bytes <= 0) return AKV_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(pool) | static_cast<uintptr_t>(layer_stride) | static_cast<uintptr_t>(page_bytes)) & 15)
    return AKV_ERR_ALIGN;
  return AKV_OK;
}

static int launched() { return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH; }

// CTAs for at most `items` pieces of a copy whose real count only the device knows
static int copy_grid(int64_t items) {
  const int64_t most = 148 * 8;
  return static_cast<int>(items < 1 ? 1 : (items < most ? items : most));
}

extern "C" size_t akv_pages_workspace_bytes(int n_pages, int n) {
  if (n_pages <= 0 || n < 0) return 0;
  return 4 * (4 + 2 * page_ws_pairs(n_pages, n) + static_cast<size_t>(n_pages));
}

extern "C" int akv_pages_fork(const akv_page_table* t, const int32_t* parents, const int32_t* children, int n,
                              int* status, void* stream) {
  int rc = table_check(t);
  if (rc) return rc;
  if (n < 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  if (!parents || !children) return AKV_ERR_NULL;
  fork_kernel<<<n, 128, 0, static_cast<cudaStream_t>(stream)>>>(*t, parents, children, n, status);
  return launched();
}

extern "C" int akv_pages_reserve_many(const akv_page_table* t, const int32_t* rows, const int32_t* n_new,
                                      int n_new_all, int n, int32_t* granted, uint8_t* pool, int n_layers,
                                      int64_t layer_stride, int64_t page_bytes, void* workspace,
                                      size_t workspace_bytes, int* status, void* stream) {
  int rc = table_check(t);
  if (rc) return rc;
  if ((rc = pool_check(pool, n_layers, layer_stride, page_bytes))) return rc;
  if (n < 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  if (!granted || !workspace) return AKV_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return AKV_ERR_ALIGN;
  if (workspace_bytes < akv_pages_workspace_bytes(t->n_pages, n)) return AKV_ERR_WORKSPACE;
  const PageWs ws = page_ws(workspace, t->n_pages, n);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  reserve_plan_kernel<<<1, kPlanThreads, 0, st>>>(*t, rows, n_new, n_new_all, n, granted, ws, status);
  const int64_t pieces = (page_bytes + kCopyChunk - 1) / kCopyChunk;
  copy_pages_kernel<<<copy_grid(pieces * n_layers * n), kCopyThreads, 0, st>>>(
      pool, n_layers, layer_stride, page_bytes, ws.src, ws.dst, ws.count, 0, t->n_pages, nullptr, 0, 0, 1, nullptr,
      nullptr, status);
  return launched();
}

extern "C" int akv_pages_reserve(const akv_page_table* t, const int32_t* rows, const int32_t* n_new, int n_new_all,
                                 int n, int32_t* granted, uint8_t* pool, int n_layers, int64_t layer_stride,
                                 int64_t page_bytes, void* workspace, size_t workspace_bytes, int* status,
                                 void* stream) {
  if (t && n > kPlanThreads) return AKV_ERR_UNSUPPORTED;
  return akv_pages_reserve_many(t, rows, n_new, n_new_all, n, granted, pool, n_layers, layer_stride, page_bytes,
                                workspace, workspace_bytes, status, stream);
}

extern "C" int akv_pages_truncate(const akv_page_table* t, const int32_t* rows, const int32_t* new_lens, int n,
                                  int* status, void* stream) {
  int rc = table_check(t);
  if (rc) return rc;
  if (n < 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  truncate_kernel<<<n, 128, 0, static_cast<cudaStream_t>(stream)>>>(*t, rows, new_lens, status);
  return launched();
}

extern "C" int akv_pages_compact(const akv_page_table* t, uint8_t* pool, int n_layers, int64_t layer_stride,
                                 int64_t page_bytes, int32_t* n_live, void* workspace, size_t workspace_bytes,
                                 int* status, void* stream) {
  int rc = table_check(t);
  if (rc) return rc;
  if ((rc = pool_check(pool, n_layers, layer_stride, page_bytes))) return rc;
  if (!n_live || !workspace) return AKV_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return AKV_ERR_ALIGN;
  if (workspace_bytes < akv_pages_workspace_bytes(t->n_pages, 0)) return AKV_ERR_WORKSPACE;
  const PageWs ws = page_ws(workspace, t->n_pages, 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(*t, n_live, ws);
  const int64_t pieces = (page_bytes + kCopyChunk - 1) / kCopyChunk;
  copy_pages_kernel<<<copy_grid(pieces * n_layers * t->n_pages), kCopyThreads, 0, st>>>(
      pool, n_layers, layer_stride, page_bytes, ws.src, ws.dst, ws.count, 0, t->n_pages, t->table, t->table_stride,
      t->max_seqs, t->max_blocks, ws.list, n_live, status);
  return launched();
}

extern "C" int akv_pages_copy(uint8_t* pool, int n_layers, int64_t layer_stride, int64_t page_bytes, int n_pages,
                              const int32_t* src, const int32_t* dst, int n, int* status, void* stream) {
  const int rc = pool_check(pool, n_layers, layer_stride, page_bytes);
  if (rc) return rc;
  if (n < 0 || n_pages <= 0) return AKV_ERR_SHAPE;
  if (n == 0) return AKV_OK;
  if (!src || !dst) return AKV_ERR_NULL;
  const int64_t pieces = (page_bytes + kCopyChunk - 1) / kCopyChunk;
  copy_pages_kernel<<<copy_grid(pieces * n_layers * n), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      pool, n_layers, layer_stride, page_bytes, src, dst, nullptr, n, n_pages, nullptr, 0, 0, 1, nullptr, nullptr,
      status);
  return launched();
}
