// lm_attention.cuh — what the kernels of attention over the paged cache share:
// their arguments, work items and the running softmax's exponential.
#pragma once

#include <type_traits>

#include "lm_common.cuh"

namespace kb {
namespace lm {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The weights exp2(s - m) are rounded to the values' type.  fp16 keeps 10 bits
// down to 2^-14 only, so its weights are held 2^kShift higher (far below its
// largest), and small ones do not lose bits; bf16 has fp32's range.
template <typename T>
constexpr float kShift = std::is_same_v<T, __half> ? 7.0f : 0.0f;

// What the tensor-core kernels multiply raw scores by after they have put -inf in
// the masked ones' place: |c|, but the least normal number for a c of zero (a
// scale of zero), since -inf x 0 would be a NaN.
__device__ __forceinline__ float score_factor(float c) { return c == 0.0f ? 0x1p-126f : fabsf(c); }

// exp2(s c - m) as one multiply-add keeps the product exact but not m = s' c of
// the reference s', and the difference, half a unit in m's last place, is the
// same factor for all of a row's weights.  Where m is so large that this factor
// could leave fp32 or fp16 (from 2^25 on), weights are exp2((s - s') c) instead.
constexpr float kFar = 0x1p20f;

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;
  const int *prefix, *table, *lens;
  int batch, queries, heads_q, heads_kv, group, dim;
  int prefix_pages, width, pages, page_size, page_shift;  // page_shift: its logarithm, or -1
  int64_t q_b, q_t, q_h, k_p, k_s, k_h, v_p, v_s, v_h;  // strides in elements
  float scale_log2;                                      // scale * log2(e)
  int prefix_tiles, prefix_splits, prefix_chunk;         // row tiles per key head; ranges and keys per range
  int own_tiles, own_splits, own_chunk, splits;
  int64_t prefix_items, first_item;                      // items of the prefix come first; the launch's first one
  float *part_o, *part_lse;  // [splits][rows][dim], [rows][splits] (rows: batch * queries * heads_q); null: one range
};

// A work item: rows r of key head h, query of row r = base + r / group, head
// h * group + r % group; keys [k0, k1) through `pages`.
struct Item {
  int h, base, row0, rows, k0, k1, split;
  const int* pages;
};
__device__ __forceinline__ Item item_at(const AttnArgs& a, int64_t id, int tile_rows) {
  Item w;
  const int P = a.prefix_pages * a.page_size;
  if (id < a.prefix_items) {  // key head fastest: CTAs that run together read different heads of the same pages
    w.h = (int)(id % a.heads_kv);
    id /= a.heads_kv;
    const int tile = (int)(id % a.prefix_tiles), s = (int)(id / a.prefix_tiles);
    w.base = 0;
    w.row0 = tile * tile_rows;
    w.rows = min(tile_rows, a.batch * a.queries * a.group - w.row0);
    w.k0 = s * a.prefix_chunk;
    w.k1 = min(w.k0 + a.prefix_chunk, P);
    w.split = s;
    w.pages = a.prefix;
  } else {
    id -= a.prefix_items;
    w.h = (int)(id % a.heads_kv);
    id /= a.heads_kv;
    const int tile = (int)(id % a.own_tiles);
    id /= a.own_tiles;
    const int b = (int)(id % a.batch), s = (int)(id / a.batch);
    w.base = b * a.queries;
    w.row0 = tile * tile_rows;
    w.rows = min(tile_rows, a.queries * a.group - w.row0);
    w.k0 = P + s * a.own_chunk;
    w.k1 = min(w.k0 + a.own_chunk, a.width * a.page_size);
    w.split = a.prefix_splits + s;
    w.pages = a.table + (int64_t)b * a.width;
  }
  return w;
}
__device__ __forceinline__ int visible(const AttnArgs& a, int bt) {
  const int b = bt / a.queries, t = bt - b * a.queries;
  return max(a.lens[b], 0) - a.queries + t + 1;  // the least number stays below zero
}
// Row r of the item in the tensors' order [batch, queries, heads_q].
__device__ __forceinline__ int64_t row_index(const AttnArgs& a, const Item& w, int r) {
  const int rr = w.row0 + r;
  return (int64_t)(w.base + rr / a.group) * a.heads_q + w.h * a.group + rr % a.group;
}
__device__ __forceinline__ const void* query_of(const AttnArgs& a, const Item& w, int r, int element_size) {
  const int rr = w.row0 + r, bt = w.base + rr / a.group;
  return static_cast<const char*>(a.q) +
         ((int64_t)(bt / a.queries) * a.q_b + (int64_t)(bt % a.queries) * a.q_t +
          (int64_t)(w.h * a.group + rr % a.group) * a.q_h) * element_size;
}

// Infinite and NaN values.  In a product of a tile of weights with a tile of
// values a masked key has weight 0, and 0 x NaN is NaN: such a value would reach
// rows that do not see its key.  So in a tile of which some rows see more than
// others the values that are not finite are replaced by 0 in shared memory, and
// at the end, if there were any, their keys are gone through once more: where a
// row sees one, that is its sum (weights are positive).
// `least`: the fewest keys seen by a row that sees any of the item's.  The first
// tile of `keys` keys, from w.k0 on, that needs this:
__device__ __forceinline__ int uneven_from(const Item& w, int least, int keys) {
  return w.k0 + (least - w.k0) / keys * keys;
}
// Whether a 32-bit word of T holds something that is not finite: an exponent of
// ones, to which one more carries into the sign's place.
template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint32_t x) {
  constexpr uint32_t kOne = std::is_same_v<T, float> ? 0x00800000u : std::is_same_v<T, __half> ? 0x04000400u : 0x00800080u;
  constexpr uint32_t kSign = std::is_same_v<T, float> ? 0x80000000u : 0x80008000u;
  return (((x & (kSign - kOne)) + kOne) & kSign) != 0;
}
__device__ __forceinline__ uint4 load_shared(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
// Replaces what is not finite among the 16 bytes at p; whether there was any.
template <typename T>
__device__ __forceinline__ bool replace_nonfinite(uint32_t p, uint4 v) {
  if (!(has_nonfinite<T>(v.x) | has_nonfinite<T>(v.y) | has_nonfinite<T>(v.z) | has_nonfinite<T>(v.w))) return false;
  union {
    uint4 v;
    T t[16 / sizeof(T)];
  } u;
  u.v = v;
#pragma unroll
  for (int i = 0; i < (int)(16 / sizeof(T)); ++i)
    if (!isfinite(to_f32(u.t[i]))) u.t[i] = from_f32<T>(0.0f);
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(p), "r"(u.v.x), "r"(u.v.y), "r"(u.v.z), "r"(u.v.w) : "memory");
  return true;
}
// The same for every STEP-th vector, from the `first` on, of ROWS rows of PER
// vectors, LD elements apart.
template <typename T, int ROWS, int PER, int LD, int STEP>
__device__ __forceinline__ bool replace_nonfinite_rows(uint32_t p, int first) {
  bool any = false;
#pragma unroll 4
  for (int i = first; i < ROWS * PER; i += STEP) {
    const uint32_t at = p + (i / PER * LD) * (int)sizeof(T) + i % PER * 16;
    any |= replace_nonfinite<T>(at, load_shared(at));
  }
  return any;
}
// The item of a launch's block, worked out again: what of it is needed at the end
// only, and hardly ever, takes no registers on the way there.
__device__ __forceinline__ Item item_again(const AttnArgs& a, int64_t first_item, int tile_rows) {
  int block = blockIdx.x;
  asm volatile("" : "+r"(block));
  return item_at(a, first_item + block, tile_rows);
}
constexpr int kNoKey = 0x7fffffff;  // first key whose values were replaced, where there is none
// Columns first to last - 1 of the item's row r, which this thread or one before a
// __syncwarp has written: the values that are not finite of keys `from` to its last.
template <typename T>
__device__ __forceinline__ void write_nonfinite(const AttnArgs& a, const Item& w, int r, int from, int first, int last) {
  if (r >= w.rows) return;
  const int64_t at = row_index(a, w, r), n_rows = (int64_t)a.batch * a.queries * a.heads_q;
  const int end = min(w.k1, visible(a, w.base + (w.row0 + r) / a.group));
#pragma unroll 1
  for (int c = first; c < min(last, a.dim); ++c) {
    float sum = 0.0f;
#pragma unroll 1
    for (int j = from; j < end; ++j) {
      const int pj = j / a.page_size;
      const int64_t page = min(max(w.pages[pj], 0), a.pages - 1);
      const T* v = static_cast<const T*>(a.v) + page * a.v_p + (int64_t)(j - pj * a.page_size) * a.v_s + w.h * a.v_h;
      const float x = to_f32(v[c]);
      if (!isfinite(x)) sum += x;
    }
    if (isfinite(sum)) continue;
    if (a.part_o) {  // added to what is there: a row of NaN stays one
      a.part_o[((int64_t)w.split * n_rows + at) * a.dim + c] += sum;
    } else {
      T* y = static_cast<T*>(a.out) + at * a.dim + c;
      *y = from_f32<T>(to_f32(*y) + sum);
    }
  }
}

// ------------------------------------------------------------------ tensor-core prefix (lm_attention_tc.cu)
// Whether it can take the prefix (16-bit types, head and page sizes, strides).
bool tc_fits(const AttnArgs& a, int dtype);
// Row tiles it makes of `rows` rows of one key head.
int tc_tile_rows(int64_t rows);
int tc_launch(const AttnArgs& a, int dtype, cudaStream_t stream);
// The device's fault word: nonzero after a wait ran out.
int tc_read_fault(bool clear, int* value);

// ------------------------------------------------------------------ fp32 prefix in halves (lm_attention_tc32.cu)
constexpr int kTc32Rows = 128;  // rows of a row tile
bool tc32_pays(int64_t rows, int64_t heads_kv, int64_t dim, int64_t keys);
size_t tc32_bytes(int64_t heads_kv, int64_t dim, int64_t keys);  // scratch, 16-byte aligned
int tc32_launch(const AttnArgs& a, void* scratch, cudaStream_t stream);
int tc32_read_fault(bool clear, int* value);

}  // namespace attn
}  // namespace lm
}  // namespace kb
