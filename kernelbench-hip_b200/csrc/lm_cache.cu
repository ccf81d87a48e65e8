// lm_cache.cu — the page operations of a paged key/value cache, kept and
// decided on the GPU: no call waits for the host.
//
// State: a pool [planes, pages, page bytes] (planes: keys and values of each
// layer), a table [slots, width] of page ids (-1: none), the number of keys
// lens[slots], and refs[pages], the number of table entries that hold each
// page (0: free).  A slot holds ceil(lens / page_size) pages from the start
// of its row, and more where its program has lowered lens (drafts that were
// rejected): they stay in the row until its next reserve uses them or it is
// freed.  A page that is not full belongs to one slot alone.
//
//   reserve  grows slots by `tokens` keys, taking pages
//   append   writes keys and values at a slot's last `tokens` places, where
//            the request that made them was granted
//   fork     makes child slots copies of parent slots: full pages are
//            shared, a last page that is not full is copied
//   free     empties slots
//   compact  moves the live pages to the low end of the pool
//   copy     copies listed pages between pools
//
// Free pages are taken in ascending order, requests are served in their
// order, and a request is granted while the pages asked for up to and
// including it are there: results do not depend on timing.  Page ids and
// slots read from device memory are checked before use; one out of range is
// passed over.
//
// The decisions are one CTA's (a chain of a few latencies, 5-7 us); the copies
// run at HBM speed (64 children of one parent in 64 planes of 32 KB pages: 27
// us for 134 MB written, the parent's page from L2).  Each launch starts while
// the one before ends.  A fork of few table entries is two launches, the plan's
// CTA writing the rows as well (4 children of 63 pages, with the reserve and the
// append that follow, in a graph: 12.4 against 14.4 us in three, 10.3 by now; 32 of
// 101 pages: 16.4 against 14.4, 14.5 by now).
// Else rows of children that share their pages meet in refs: a thread takes one
// column of 16 rows and adds a page's changes up before its atomic.
#include "lm_common.cuh"

namespace kb {
namespace lm {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMaxPages = 1 << 20, kMaxSlots = 1 << 20;
constexpr int64_t kMaxKeys = 0x3fffffff;  // of a row: a page more is still a number of 32 bits
constexpr int kSharedSlots = 4096;  // slots whose owners shared memory holds
constexpr int kWholeRows = 2048;    // table entries that the fork's planning CTA writes itself

// Changes of pages' counts that a thread meets one after the other, added up
// while the page stays the same.
struct Run {
  int* refs;
  int pages, page = -1, by = 0;
  __device__ Run(int* r, int n) : refs(r), pages(n) {}
  __device__ void flush() {
    if (by) atomicAdd(&refs[page], by);
    by = 0;
  }
  __device__ void add(int p, int v) {
    if (p < 0 || p >= pages) return;
    if (p != page) flush();
    page = p;
    by += v;
  }
};
constexpr int kColumns = 128, kRowsAtOnce = 16;  // of a table: a CTA's part where rows share pages

// Exclusive prefix sum over the block, and the total.
__device__ __forceinline__ int block_scan(int v, int* red, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  if (lane == 31) red[warp] = inc;
  __syncthreads();
  int w = lane < (int)(blockDim.x >> 5) ? red[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += n;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  __syncthreads();
  return before + inc - v;
}

// list[r] = the r-th lowest page with refs == 0, for r < want; returns how
// many there are, at most `want`.  `first`: refs[threadIdx.x], loaded ahead
// (nonzero past the pages).
__device__ int free_pages(const int* refs, int pages, int want, int* list, int* red, int first) {
  int found = 0;
  for (int base = 0; base < pages && found < want; base += kPlanThreads) {
    const int p = base + threadIdx.x;
    const int is_free = p < pages && (base == 0 ? first : refs[p]) == 0;
    int total;
    const int at = found + block_scan(is_free, red, total);
    if (is_free && at < want) list[at] = p;
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

// ------------------------------------------------------------------ fork
struct ForkArgs {
  int *table, *lens, *refs;
  const int *parents, *children;
  int* granted;
  int n, slots, width, pages, page_size;
  int *owner;   // [slots] lowest request that names the slot as its child
  int *list;    // [n] free pages
  int *src, *dst;  // [n] page to copy and where to, or -1
  int *len;     // [n] the child's new length, or -1 where nothing changes
  int *rows;    // [n][width] the children's new rows
  bool whole;   // the plan's CTA writes the rows, too
};

// Entry j of the row of a child of `len` keys whose last page, if it was copied, is `dst`.
__device__ __forceinline__ int new_entry(const ForkArgs& a, int len, int dst, int parent, int j) {
  const int held = (len + a.page_size - 1) / a.page_size;
  return j >= held ? -1 : (dst >= 0 && j == held - 1) ? dst : a.table[(int64_t)parent * a.width + j];
}

// A chain of latencies: what does not depend on another load is loaded at the
// start, and the slots' owners and the free pages stay in shared memory where
// they fit.
__global__ void __launch_bounds__(kPlanThreads) fork_plan(ForkArgs a) {
  __shared__ int red[32];
  __shared__ int s_owner[kSharedSlots], s_list[kPlanThreads];
  __shared__ int s_child[kPlanThreads], s_len[kPlanThreads], s_dst[kPlanThreads];  // of the one-CTA case
  allow_next();
  wait_for_previous();
  int* owner = a.slots <= kSharedSlots ? s_owner : a.owner;
  int* list = a.n <= kPlanThreads ? s_list : a.list;
  const int mine = threadIdx.x;
  const int first = mine < a.pages ? a.refs[mine] : 1;
  const int parent0 = mine < a.n ? a.parents[mine] : -1, child0 = mine < a.n ? a.children[mine] : -1;
  const int len0 = parent0 >= 0 && parent0 < a.slots ? a.lens[parent0] : 0;
  for (int i = mine; i < a.slots; i += kPlanThreads) owner[i] = a.n;
  __syncthreads();
  for (int i = mine; i < a.n; i += kPlanThreads) {
    const int c = i == mine ? child0 : a.children[i];
    if (c >= 0 && c < a.slots) atomicMin(&owner[c], i);
  }
  const int have = free_pages(a.refs, a.pages, a.n, list, red, first);  // ends with a barrier
  __syncthreads();                                                      // where there was no page to look at
  int asked = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + mine;
    int need = 0, len = -1, ok = 0, src = -1;
    if (i < a.n) {
      const int p = base ? a.parents[i] : parent0, c = base ? a.children[i] : child0;
      ok = p >= 0 && p < a.slots && c >= 0 && c < a.slots && owner[c] == i;
      if (ok && p != c) {
        len = max(0, min(base ? a.lens[p] : len0, a.width * a.page_size));
        if (len % a.page_size) {
          src = a.table[(int64_t)p * a.width + len / a.page_size];
          need = src >= 0 && src < a.pages;
        }
      }
    }
    int total;
    const int rank = asked + block_scan(need, red, total);
    asked += total;
    if (i < a.n) {
      if (need && rank >= have) ok = 0, len = -1, need = 0;
      a.granted[i] = ok;
      a.len[i] = len;
      a.src[i] = need ? src : -1;
      a.dst[i] = need ? list[rank] : -1;
      if (a.whole) s_child[i] = child0, s_len[i] = len, s_dst[i] = need ? list[rank] : -1;
    }
  }
  if (!a.whole) return;
  // the rows as well: all are read before any is written
  __shared__ int s_parent[kPlanThreads];
  s_parent[mine] = parent0;
  __syncthreads();
  constexpr int kEach = kWholeRows / kPlanThreads;
  const int entries = a.n * a.width;
  int before[kEach], after[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = mine + k * kPlanThreads, i = at / max(a.width, 1), j = at - i * a.width;
    before[k] = after[k] = -1;
    if (at >= entries || s_len[i] < 0) continue;
    before[k] = a.table[(int64_t)s_child[i] * a.width + j];
    after[k] = new_entry(a, s_len[i], s_dst[i], s_parent[i], j);
  }
  __syncthreads();
  if (mine < a.n && s_len[mine] >= 0) a.lens[child0] = s_len[mine];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = mine + k * kPlanThreads, i = at / max(a.width, 1), j = at - i * a.width;
    if (at >= entries || s_len[i] < 0) continue;
    a.table[(int64_t)s_child[i] * a.width + j] = after[k];
    if (before[k] >= 0 && before[k] < a.pages) atomicSub(&a.refs[before[k]], 1);
    if (after[k] >= 0 && after[k] < a.pages) atomicAdd(&a.refs[after[k]], 1);
  }
}

// The children's new rows, from the parents' before any of them is replaced.
__device__ void fork_row(const ForkArgs& a, int i) {
  const int len = a.len[i];
  if (len < 0) return;
  const int dst = a.dst[i], parent = a.parents[i];
  int* to = a.rows + (int64_t)i * a.width;
  for (int j = threadIdx.x; j < a.width; j += blockDim.x) to[j] = new_entry(a, len, dst, parent, j);
}

__global__ void __launch_bounds__(kColumns) fork_commit(ForkArgs a) {
  allow_next();
  wait_for_previous();
  const int j = blockIdx.y * kColumns + threadIdx.x, first = blockIdx.x * kRowsAtOnce;  // rows in x: up to 2^16 blocks
  __shared__ int child[kRowsAtOnce];  // or -1 where nothing changes
  if (threadIdx.x < kRowsAtOnce) {
    const int i = first + threadIdx.x, len = i < a.n ? a.len[i] : -1;
    child[threadIdx.x] = len >= 0 ? a.children[i] : -1;
    if (len >= 0 && blockIdx.y == 0) a.lens[a.children[i]] = len;
  }
  __syncthreads();
  if (j >= a.width) return;
  int before[kRowsAtOnce], after[kRowsAtOnce];  // all in flight at once
#pragma unroll
  for (int k = 0; k < kRowsAtOnce; ++k) {
    before[k] = child[k] >= 0 ? a.table[(int64_t)child[k] * a.width + j] : -1;
    after[k] = child[k] >= 0 ? a.rows[(int64_t)(first + k) * a.width + j] : -1;
  }
  Run gone(a.refs, a.pages), come(a.refs, a.pages);
#pragma unroll
  for (int k = 0; k < kRowsAtOnce; ++k) {
    gone.add(before[k], -1);
    come.add(after[k], 1);
    if (child[k] >= 0) a.table[(int64_t)child[k] * a.width + j] = after[k];
  }
  gone.flush();
  come.flush();
}

// ------------------------------------------------------------------ copy
struct CopyArgs {
  const char* from;
  char* to;
  const int *src, *dst;
  const int* count;  // device, or null: n pairs
  int n;
  int64_t planes, page_bytes, from_pages, to_pages;
};
// Copies pages src[i] -> dst[i] of every plane, shared out over `blocks` CTAs.
// Pairs with an id out of range are passed over.
__device__ void copy_pages(const CopyArgs& a, int64_t block, int64_t blocks) {
  const int64_t pairs = a.count ? min(*a.count, a.n) : a.n;
  const bool wide = a.page_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(a.from) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(a.to) & 15) == 0;
  for (int64_t it = block; it < pairs * a.planes; it += blocks) {
    const int64_t i = it / a.planes, plane = it - i * a.planes;
    const int s = a.src[i], d = a.dst[i];
    if (s < 0 || s >= a.from_pages || d < 0 || d >= a.to_pages) continue;
    const char* x = a.from + (plane * a.from_pages + s) * a.page_bytes;
    char* y = a.to + (plane * a.to_pages + d) * a.page_bytes;
    if (wide) {
      const int64_t vecs = a.page_bytes / 16;
      const uint4* xv = reinterpret_cast<const uint4*>(x);
      uint4* yv = reinterpret_cast<uint4*>(y);
      int64_t j = threadIdx.x;
      for (; j + 3 * blockDim.x < vecs; j += 4 * blockDim.x) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = xv[j + k * blockDim.x];
#pragma unroll
        for (int k = 0; k < 4; ++k) yv[j + k * blockDim.x] = v[k];
      }
      for (; j < vecs; j += blockDim.x) yv[j] = xv[j];
    } else {
      for (int64_t j = threadIdx.x; j < a.page_bytes; j += blockDim.x) y[j] = x[j];
    }
  }
}
__global__ void __launch_bounds__(256) copy_kernel(CopyArgs a) {
  allow_next();
  wait_for_previous();
  copy_pages(a, blockIdx.x, gridDim.x);
}
// The first n CTAs write the children's new rows, the others copy the pages.
__global__ void __launch_bounds__(256) fork_rows(ForkArgs a, CopyArgs copy) {
  allow_next();
  wait_for_previous();
  if ((int)blockIdx.x < a.n)
    fork_row(a, blockIdx.x);
  else
    copy_pages(copy, blockIdx.x - a.n, gridDim.x - a.n);
}

// ------------------------------------------------------------------ reserve
struct ReserveArgs {
  int *table, *lens, *refs;
  const int* seqs;
  int* granted;
  int n, tokens, slots, width, pages, page_size;
  int *owner, *list;
};

__global__ void __launch_bounds__(kPlanThreads) reserve_kernel(ReserveArgs a) {
  __shared__ int red[32];
  __shared__ int s_owner[kSharedSlots], s_list[kPlanThreads];
  allow_next();
  wait_for_previous();
  // no slot takes more pages than its row is wide, nor all more than there are
  const int most = (int)min((int64_t)a.pages, (int64_t)a.n * min(a.width, a.tokens / a.page_size + 1));
  int* owner = a.slots <= kSharedSlots ? s_owner : a.owner;
  int* list = most <= kPlanThreads ? s_list : a.list;
  const int mine = threadIdx.x;
  const int first = mine < a.pages ? a.refs[mine] : 1;
  const int seq0 = mine < a.n ? a.seqs[mine] : -1;
  const int len0 = seq0 >= 0 && seq0 < a.slots ? a.lens[seq0] : -1;
  // the entry past the slot's pages, on its way while the free pages are looked for
  const bool inside = len0 >= 0 && len0 < a.width * a.page_size;
  const int next0 = inside ? a.table[(int64_t)seq0 * a.width + (len0 + a.page_size - 1) / a.page_size % a.width] : -1;
  for (int i = mine; i < a.slots; i += kPlanThreads) owner[i] = a.n;
  __syncthreads();
  for (int i = mine; i < a.n; i += kPlanThreads) {
    const int c = i == mine ? seq0 : a.seqs[i];
    if (c >= 0 && c < a.slots) atomicMin(&owner[c], i);
  }
  const int have = free_pages(a.refs, a.pages, most, list, red, first);
  __syncthreads();
  int asked = 0;
  for (int base = 0; base < a.n; base += kPlanThreads) {
    const int i = base + mine;
    int need = 0, kept = 0, ok = 0, held = 0, len = 0, c = -1;
    if (i < a.n) {
      c = base ? a.seqs[i] : seq0;
      ok = c >= 0 && c < a.slots && owner[c] == i;
      if (ok) {
        len = base ? a.lens[c] : len0;
        ok = len >= 0 && (int64_t)len + a.tokens <= (int64_t)a.width * a.page_size;
      }
      if (ok) {
        held = (len + a.page_size - 1) / a.page_size;
        // capped past the pool, so that sums over a block stay in 32 bits
        need = min((len + a.tokens + a.page_size - 1) / a.page_size - held, a.pages + 1);
        // pages that the row still holds from before lens was lowered
        const int* row = a.table + (int64_t)c * a.width + held;
        if (base || next0 >= 0)
          while (kept < need && row[kept] >= 0 && row[kept] < a.pages) ++kept;
        held += kept;
        need -= kept;
      }
    }
    int total;
    const int rank = asked + block_scan(need, red, total);
    asked = (int)min((int64_t)asked + total, (int64_t)1 << 26);
    if (i < a.n) {
      if (need && rank + need > have) ok = 0;
      a.granted[i] = ok;
      if (ok) {
        for (int j = 0; j < need; ++j) {
          const int p = list[rank + j];
          a.table[(int64_t)c * a.width + held + j] = p;
          a.refs[p] = 1;
        }
        a.lens[c] = len + a.tokens;
      }
    }
  }
}

// ------------------------------------------------------------------ append
struct AppendArgs {
  const char *k, *v;
  char *k_pages, *v_pages;
  const int *table, *lens, *seqs;
  const int* granted;  // of the reserve that made the places, or null: all of them
  int64_t k_stride_seq, k_stride_tok, v_stride_seq, v_stride_tok;  // bytes
  int64_t page_bytes, key_bytes;  // a page, and one token's heads, of one plane
  int n, tokens, slots, width, pages, page_size;
};

__global__ void __launch_bounds__(128) append_kernel(AppendArgs a) {
  allow_next();
  wait_for_previous();
  const int64_t i = blockIdx.x / a.tokens;
  const int t = (int)(blockIdx.x - i * a.tokens);
  const int c = a.seqs[i];
  // A refused slot has not grown: its last places are older keys, which other slots may share.
  if (c < 0 || c >= a.slots || (a.granted && !a.granted[i])) return;
  const int pos = max(a.lens[c], 0) - a.tokens + t;  // the least number stays below zero
  if (pos < 0 || pos / a.page_size >= a.width) return;
  const int p = a.table[(int64_t)c * a.width + pos / a.page_size];
  if (p < 0 || p >= a.pages) return;
  const int64_t at = p * a.page_bytes + (pos % a.page_size) * a.key_bytes;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const char* x = kv ? a.v + i * a.v_stride_seq + t * a.v_stride_tok : a.k + i * a.k_stride_seq + t * a.k_stride_tok;
    char* y = (kv ? a.v_pages : a.k_pages) + at;
    if (a.key_bytes % 16 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0) {
      for (int64_t j = threadIdx.x; j < a.key_bytes / 16; j += blockDim.x)
        reinterpret_cast<uint4*>(y)[j] = reinterpret_cast<const uint4*>(x)[j];
    } else {
      for (int64_t j = threadIdx.x; j < a.key_bytes; j += blockDim.x) y[j] = x[j];
    }
  }
}

// ------------------------------------------------------------------ free
__global__ void free_kernel(int* table, int* lens, int* refs, const int* seqs, int slots, int width, int pages) {
  allow_next();
  wait_for_previous();
  const int c = seqs[blockIdx.x];
  if (c < 0 || c >= slots) return;
  if (threadIdx.x == 0) lens[c] = 0;
  int* row = table + (int64_t)c * width;
  for (int j = threadIdx.x; j < width; j += blockDim.x) {
    const int p = atomicExch(&row[j], -1);  // a slot that is listed twice gives its pages back once
    if (p >= 0 && p < pages) atomicSub(&refs[p], 1);
  }
}

// ------------------------------------------------------------------ compact
struct CompactArgs {
  int *table, *refs;
  int* live;
  int64_t entries;
  int pages;
  int *src, *dst, *count;  // the moves
  int* map;                // [pages] where a moved page goes, or -1
};

__global__ void __launch_bounds__(kPlanThreads) compact_plan(CompactArgs a) {
  __shared__ int red[32];
  allow_next();
  wait_for_previous();
  int mine = 0, live;
  for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) mine += a.refs[p] > 0;
  block_scan(mine, red, live);
  int holes = 0, moved = 0;
  for (int base = 0; base < a.pages; base += kPlanThreads) {
    const int p = base + threadIdx.x;
    const bool used = p < a.pages && a.refs[p] > 0;
    const int hole = p < live && !used, move = p >= live && used;
    int total;
    const int h = holes + block_scan(hole, red, total);
    holes += total;
    const int m = moved + block_scan(move, red, total);
    moved += total;
    if (hole) a.dst[h] = p;
    if (move) a.src[m] = p;
  }
  // as many holes below the live count as live pages above it
  __syncthreads();
  for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) a.map[p] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < moved; i += kPlanThreads) {
    const int s = a.src[i], d = a.dst[i];
    a.map[s] = d;
    a.refs[d] = a.refs[s];
    a.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    *a.count = moved;
    *a.live = live;
  }
}

// The first `table_blocks` CTAs rewrite the table, the others move the pages.
__global__ void __launch_bounds__(256) compact_moves(CompactArgs a, CopyArgs copy, int table_blocks) {
  allow_next();
  wait_for_previous();
  if ((int)blockIdx.x >= table_blocks) {
    copy_pages(copy, blockIdx.x - table_blocks, gridDim.x - table_blocks);
    return;
  }
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < a.entries;
       i += (int64_t)table_blocks * blockDim.x) {
    const int p = a.table[i];
    if (p >= 0 && p < a.pages && a.map[p] >= 0) a.table[i] = a.map[p];
  }
}

unsigned copy_grid(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, sm_count() * 8)); }

size_t ints(int64_t n) { return (size_t)ceil_div(n, 4) * 16; }

}  // namespace
}  // namespace lm
}  // namespace kb

extern "C" {

#define KB_CACHE_COMMON(n)                                                                                       \
  KB_REQUIRE((n) >= 0 && slots >= 0 && width >= 0 && pages >= 0, KB_ERR_INVALID_ARG, "%s: negative size", name); \
  KB_REQUIRE(slots <= kMaxSlots && width <= kMaxSlots && pages <= kMaxPages && (n) <= kMaxSlots,                  \
             KB_ERR_UNSUPPORTED, "%s: more than %d pages or %d slots, entries of a row or requests", name,        \
             kMaxPages, kMaxSlots)

#define KB_CACHE_WORKSPACE(need)                                                                       \
  KB_REQUIRE(workspace && workspace_bytes >= (need), KB_ERR_WORKSPACE,                                 \
             "%s: workspace of %zu bytes needed, %zu given", name, (size_t)(need), workspace_bytes);   \
  KB_REQUIRE(kb::aligned16(workspace), KB_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name)

size_t kb_cache_fork_workspace_size(int64_t n, int64_t slots, int64_t width) {
  if (n <= 0 || slots < 0 || width < 0) return 0;
  return kb::lm::ints(slots) + 4 * kb::lm::ints(n) + kb::lm::ints(n * width);
}

int kb_cache_fork(void* pool, int32_t* table, int32_t* lens, int32_t* refs, const int32_t* parents,
                  const int32_t* children, int32_t* granted, int64_t n, int64_t slots, int64_t width, int64_t planes,
                  int64_t pages, int64_t page_size, int64_t page_bytes, void* workspace, size_t workspace_bytes,
                  kbStream stream) {
  const char* name = "kb_cache_fork";
  using namespace kb::lm;
  KB_CACHE_COMMON(n);
  KB_REQUIRE(planes >= 0 && page_bytes >= 0 && page_size >= 1, KB_ERR_INVALID_ARG, "%s: bad page", name);
  KB_REQUIRE(page_size <= kMaxKeys && page_size * width <= kMaxKeys && planes <= 0x7fffffff, KB_ERR_UNSUPPORTED,
             "%s: too many keys or planes", name);
  if (n == 0) return KB_OK;
  KB_REQUIRE(parents && children && granted && (!slots || (lens && (!width || table))) && (!pages || refs),
             KB_ERR_INVALID_ARG, "%s: null pointer", name);
  KB_REQUIRE(pool || !planes || !pages || !page_bytes, KB_ERR_INVALID_ARG, "%s: null pool", name);
  KB_CACHE_WORKSPACE(kb_cache_fork_workspace_size(n, slots, width));
  char* w = static_cast<char*>(workspace);
  ForkArgs a{table, lens, refs, parents, children, granted, (int)n, (int)slots, (int)width, (int)pages, (int)page_size,
             nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, false};
  auto take = [&](int64_t m) {
    int* p = reinterpret_cast<int*>(w);
    w += ints(m);
    return p;
  };
  a.owner = take(slots), a.list = take(n), a.src = take(n), a.dst = take(n), a.len = take(n), a.rows = take(n * width);
  a.whole = n <= kPlanThreads && n * width <= kWholeRows;
  if (int st = launch_after(fork_plan, dim3(1), (unsigned)kPlanThreads, 0, stream, a)) return st;
  CopyArgs copy{static_cast<const char*>(pool), static_cast<char*>(pool), a.src, a.dst, nullptr, (int)n, planes,
                page_bytes, pages, pages};
  const unsigned copies = planes && page_bytes && pages ? copy_grid(n * planes) : 0;
  if (a.whole) return copies ? launch_after(copy_kernel, dim3(copies), 256u, 0, stream, copy) : (int)KB_OK;
  if (int st = launch_after(fork_rows, dim3((unsigned)n + copies), 256u, 0, stream, a, copy)) return st;
  return launch_after(fork_commit, dim3((unsigned)kb::ceil_div(n, kRowsAtOnce),
                                        (unsigned)std::max<int64_t>(1, kb::ceil_div(width, kColumns))),
                      (unsigned)kColumns, 0, stream, a);
}

size_t kb_cache_reserve_workspace_size(int64_t n, int64_t tokens, int64_t slots, int64_t width, int64_t pages,
                                       int64_t page_size) {
  if (n <= 0 || slots < 0 || width < 0 || pages < 0 || tokens < 0 || page_size < 1) return 0;
  const int64_t most = std::min<int64_t>(pages, n * std::min<int64_t>(width, tokens / page_size + 1));
  return kb::lm::ints(slots) + kb::lm::ints(most);
}

int kb_cache_reserve(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* seqs, int32_t* granted, int64_t n,
                     int64_t tokens, int64_t slots, int64_t width, int64_t pages, int64_t page_size, void* workspace,
                     size_t workspace_bytes, kbStream stream) {
  const char* name = "kb_cache_reserve";
  using namespace kb::lm;
  KB_CACHE_COMMON(n);
  KB_REQUIRE(tokens >= 0 && page_size >= 1, KB_ERR_INVALID_ARG, "%s: bad page or token count", name);
  KB_REQUIRE(page_size <= kMaxKeys && page_size * width <= kMaxKeys && tokens <= kMaxKeys, KB_ERR_UNSUPPORTED,
             "%s: too many keys", name);
  if (n == 0) return KB_OK;
  KB_REQUIRE(seqs && granted && (!slots || (lens && (!width || table))) && (!pages || refs), KB_ERR_INVALID_ARG,
             "%s: null pointer", name);
  KB_CACHE_WORKSPACE(kb_cache_reserve_workspace_size(n, tokens, slots, width, pages, page_size));
  ReserveArgs a{table, lens, refs, seqs, granted, (int)n, (int)tokens, (int)slots, (int)width, (int)pages,
                (int)page_size, static_cast<int*>(workspace),
                reinterpret_cast<int*>(static_cast<char*>(workspace) + ints(slots))};
  return launch_after(reserve_kernel, dim3(1), (unsigned)kPlanThreads, 0, stream, a);
}

int kb_cache_append_granted(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                            const int32_t* lens, const int32_t* seqs, const int32_t* granted, int64_t n,
                            int64_t tokens, int64_t slots, int64_t width, int64_t pages, int64_t page_size,
                            int64_t page_bytes, int64_t key_bytes, int64_t k_stride_seq, int64_t k_stride_token,
                            int64_t v_stride_seq, int64_t v_stride_token, kbStream stream) {
  const char* name = "kb_cache_append";
  using namespace kb::lm;
  KB_CACHE_COMMON(n);
  KB_REQUIRE(tokens >= 0 && page_size >= 1 && key_bytes >= 0 && page_bytes / page_size >= key_bytes,
             KB_ERR_INVALID_ARG, "%s: bad page or token count", name);
  KB_REQUIRE(page_size <= 0x7fffffff && tokens <= 0x7fffffff && n * tokens <= 0x7fffffff, KB_ERR_UNSUPPORTED,
             "%s: too many tokens", name);
  if (n == 0 || tokens == 0 || key_bytes == 0 || slots == 0 || width == 0 || pages == 0) return KB_OK;
  KB_REQUIRE(k && v && k_pages && v_pages && table && lens && seqs, KB_ERR_INVALID_ARG, "%s: null pointer", name);
  AppendArgs a{static_cast<const char*>(k), static_cast<const char*>(v), static_cast<char*>(k_pages),
               static_cast<char*>(v_pages), table, lens, seqs, granted, k_stride_seq, k_stride_token, v_stride_seq,
               v_stride_token, page_bytes, key_bytes, (int)n, (int)tokens, (int)slots, (int)width, (int)pages,
               (int)page_size};
  return launch_after(append_kernel, dim3((unsigned)(n * tokens)), 128u, 0, stream, a);
}

int kb_cache_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* table,
                    const int32_t* lens, const int32_t* seqs, int64_t n, int64_t tokens, int64_t slots, int64_t width,
                    int64_t pages, int64_t page_size, int64_t page_bytes, int64_t key_bytes, int64_t k_stride_seq,
                    int64_t k_stride_token, int64_t v_stride_seq, int64_t v_stride_token, kbStream stream) {
  return kb_cache_append_granted(k, v, k_pages, v_pages, table, lens, seqs, nullptr, n, tokens, slots, width, pages,
                                 page_size, page_bytes, key_bytes, k_stride_seq, k_stride_token, v_stride_seq,
                                 v_stride_token, stream);
}

int kb_cache_free(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* seqs, int64_t n, int64_t slots,
                  int64_t width, int64_t pages, kbStream stream) {
  const char* name = "kb_cache_free";
  using namespace kb::lm;
  KB_CACHE_COMMON(n);
  if (n == 0 || slots == 0) return KB_OK;
  KB_REQUIRE(lens && seqs && (!width || table) && (!pages || refs), KB_ERR_INVALID_ARG, "%s: null pointer", name);
  return launch_after(free_kernel, dim3((unsigned)n), 256u, 0, stream, table, lens, refs, seqs, (int)slots, (int)width,
                      (int)pages);
}

size_t kb_cache_compact_workspace_size(int64_t pages) {
  return pages > 0 ? 3 * kb::lm::ints(pages) + 16 : 16;
}

int kb_cache_compact(void* pool, int32_t* table, int32_t* refs, int32_t* live, int64_t slots, int64_t width,
                     int64_t planes, int64_t pages, int64_t page_bytes, void* workspace, size_t workspace_bytes,
                     kbStream stream) {
  const char* name = "kb_cache_compact";
  using namespace kb::lm;
  KB_CACHE_COMMON(0);
  KB_REQUIRE(planes >= 0 && page_bytes >= 0, KB_ERR_INVALID_ARG, "%s: negative size", name);
  KB_REQUIRE(planes <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: too many planes", name);
  KB_REQUIRE(live && (!pages || refs) && (!slots || !width || table), KB_ERR_INVALID_ARG, "%s: null pointer", name);
  KB_REQUIRE(pool || !planes || !pages || !page_bytes, KB_ERR_INVALID_ARG, "%s: null pool", name);
  KB_CACHE_WORKSPACE(kb_cache_compact_workspace_size(pages));
  char* w = static_cast<char*>(workspace);
  CompactArgs a{table, refs, live, slots * width, (int)pages, nullptr, nullptr, nullptr, nullptr};
  a.count = reinterpret_cast<int*>(w);
  a.src = reinterpret_cast<int*>(w + 16);
  a.dst = reinterpret_cast<int*>(w + 16 + ints(pages));
  a.map = reinterpret_cast<int*>(w + 16 + 2 * ints(pages));
  if (int st = launch_after(compact_plan, dim3(1), (unsigned)kPlanThreads, 0, stream, a)) return st;
  if (pages == 0) return KB_OK;
  CopyArgs copy{static_cast<const char*>(pool), static_cast<char*>(pool), a.src, a.dst, a.count, (int)pages, planes,
                page_bytes, pages, pages};
  const unsigned copies = planes && page_bytes ? copy_grid(pages * planes) : 0;
  const unsigned rows = a.entries ? copy_grid(kb::ceil_div(a.entries, 1024)) : 0;
  if (copies + rows == 0) return KB_OK;
  return launch_after(compact_moves, dim3(rows + copies), 256u, 0, stream, a, copy, (int)rows);
}

int kb_cache_copy(const void* src_pool, const int32_t* src, void* dst_pool, const int32_t* dst, int64_t n,
                  int64_t planes, int64_t page_bytes, int64_t src_pages, int64_t dst_pages, kbStream stream) {
  const char* name = "kb_cache_copy";
  using namespace kb::lm;
  KB_REQUIRE(n >= 0 && planes >= 0 && page_bytes >= 0 && src_pages >= 0 && dst_pages >= 0, KB_ERR_INVALID_ARG,
             "%s: negative size", name);
  KB_REQUIRE(n <= 0x7fffffff && planes <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: too many pages or planes", name);
  if (n == 0 || planes == 0 || page_bytes == 0 || src_pages == 0 || dst_pages == 0) return KB_OK;
  KB_REQUIRE(src_pool && dst_pool && src && dst, KB_ERR_INVALID_ARG, "%s: null pointer", name);
  const CopyArgs copy{static_cast<const char*>(src_pool), static_cast<char*>(dst_pool), src, dst, nullptr, (int)n,
                      planes, page_bytes, src_pages, dst_pages};
  return launch_after(copy_kernel, dim3(copy_grid(n * planes)), 256u, 0, stream, copy);
}

}  // extern "C"
