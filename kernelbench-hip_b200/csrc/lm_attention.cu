// lm_attention.cu — attention of a batch of sequences that share a prefix,
// over a paged cache of keys and values.
//
// Key j of sequence b lies in page prefix[j / page_size] for j < P = prefix
// pages * page_size, else in page table[b][j / page_size].  Query t of the
// `queries` newest tokens sees the keys j < lens[b] - queries + t + 1.
//   s_j = scale q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j),
//   lse = log sum_j exp(s_j);   no key: o = 0, lse = -inf
//
// The prefix is the same for all sequences, so all their query rows of one
// key head (batch * queries * group of them) meet each tile of it together:
// it is read once per row tile instead of once per sequence, and the products
// have enough rows for the tensor cores.  Each sequence's own keys meet its
// own rows.  Both axes of keys are cut into ranges; a work item (row tile,
// range) keeps the running maximum and sum of its softmax, in fp32, and writes
// its normalised part of o and its lse, and a second kernel joins the parts:
//   o = sum_i exp(lse_i - L) o_i,  L = log sum_i exp(lse_i).
//
// The kernels here are on mma.sync: `keys` for few rows, bound by the bytes of
// the cache, and `rows` for more of them where the tensor-core kernels of
// lm_attention_tc.cu (16-bit) and lm_attention_tc32.cu (fp32) cannot take the
// prefix or do not pay; plan_part() chooses.  bf16, 32 query and 8 key heads x
// 128, on a B200: 64 samples of an 8192-token prompt with up to 1000 keys of
// their own 64 us (own keys alone 39), 256 samples of 32768 tokens with up to
// 700 of their own 227 us where L2 holds what the call before left (own keys 71,
// at 5.1 TB/s) and 260 where all inputs come from HBM.
//
// Keys at or past what a row tile sees are not read (they count as zeros), so
// what stands in unused slots of a page does not matter; infinite and NaN values
// reach the rows that see their keys only.  Page ids out of range are clamped
// into the pool.
#include <type_traits>

#include "lm_attention.cuh"

namespace kb {
namespace lm {
namespace attn {
namespace {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes from global to shared memory, zeros where `valid` is false.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
  const int bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr size_t kMaxSmem = 227 * 1024;  // of a block, what the kernels declare statically included

// Start of a kernel over keys.  The launch over the sequences' own keys needs
// nothing of the one over the prefix, and its CTAs fill the SMs that that one
// leaves: it reads on without a wait.  So the launch that comes first waits for
// those before it first, and only then lets the next one begin.
__device__ __forceinline__ void begin(const AttnArgs& a) {
  if (a.first_item == 0) wait_for_previous();
  allow_next();
}

// ------------------------------------------------------------------ products
// Fragments of mma.sync: 16 rows x 8 columns of fp32 accumulators per warp.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                      __nv_bfloat16*) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// fp32 as two TF32 values: hi keeps the upper 10 mantissa bits, lo = x - hi
// (0 for a non-finite x, whose hi says it all).
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ Split split(float x) {
  const uint32_t hi = __float_as_uint(x) & 0xffffe000u;
  const float lo = x - __uint_as_float(hi);
  return {hi, isfinite(lo) ? __float_as_uint(lo) : 0u};
}
// hh += A_hi B_hi, x += A_lo B_hi + A_hi B_lo; the sum is A B to fp32 accuracy.
// The tensor cores' accumulation truncates, so chains are kept short and the
// small cross terms apart; the callers add with rounding.
__device__ __forceinline__ void mma_3xtf32(float (&hh)[4], float (&x)[4], const Split (&a)[4], Split b0, Split b1) {
  const uint32_t ah[4] = {a[0].hi, a[1].hi, a[2].hi, a[3].hi}, al[4] = {a[0].lo, a[1].lo, a[2].lo, a[3].lo};
  mma_tf32(x, al, b0.hi, b1.hi);
  mma_tf32(x, ah, b0.lo, b1.lo);
  mma_tf32(hh, ah, b0.hi, b1.hi);
}
constexpr int kChain = 4;  // products of depth 8 chained in one accumulator
constexpr int kWide = 4;   // accumulators in turn: a product does not wait for the one before it
__device__ __forceinline__ uint32_t pack2(float x, float y, __half*) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16*) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// S[16 x NK] = Q (16 rows at `q`) K^T (NK keys at `k`), both row-major with a
// row of LD elements; DP of them counted.
template <typename T, int DP, int NK, int LD>
__device__ __forceinline__ void scores(float (&s)[NK / 8][4], const T* q, const T* k, int lane) {
#pragma unroll
  for (int n = 0; n < NK / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
  if constexpr (std::is_same_v<T, float>) {
    const int r = lane >> 2, c = lane & 3;
#pragma unroll 1
    for (int d0 = 0; d0 < DP; d0 += 8 * kChain) {
      Split qa[kChain][4];
#pragma unroll
      for (int i = 0; i < kChain; ++i) {
        const float* x = q + r * LD + d0 + 8 * i + c;
        qa[i][0] = split(x[0]), qa[i][1] = split(x[8 * LD]), qa[i][2] = split(x[4]), qa[i][3] = split(x[8 * LD + 4]);
      }
#pragma unroll
      for (int n0 = 0; n0 < NK / 8; n0 += kWide) {
        float hh[kWide][4] = {}, x[kWide][4] = {};
#pragma unroll
        for (int i = 0; i < kChain; ++i)
#pragma unroll
          for (int n = 0; n < kWide && n0 + n < NK / 8; ++n) {
            const float* y = k + ((n0 + n) * 8 + r) * LD + d0 + 8 * i + c;
            mma_3xtf32(hh[n], x[n], qa[i], split(y[0]), split(y[4]));
          }
#pragma unroll
        for (int n = 0; n < kWide && n0 + n < NK / 8; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n0 + n][i] += hh[n][i] + x[n][i];
      }
    }
  } else {
    const uint32_t qrow = smem_addr(q + (lane & 15) * LD + (lane >> 4) * 8);
    const uint32_t krow = smem_addr(k + ((lane & 7) + ((lane >> 4) << 3)) * LD + ((lane >> 3) & 1) * 8);
#pragma unroll
    for (int d = 0; d < DP; d += 16) {
      uint32_t qa[4];
      ldmatrix4(qa, qrow + d * 2);
#pragma unroll
      for (int n = 0; n < NK / 16; ++n) {
        uint32_t kb[4];
        ldmatrix4(kb, krow + (n * 16 * LD + d) * 2);
        mma16(s[2 * n], qa, kb[0], kb[1], (T*)nullptr);
        mma16(s[2 * n + 1], qa, kb[2], kb[3], (T*)nullptr);
      }
    }
  }
}

// O[16 x DP] += P[16 x NK] V (NK keys at `v`).  With 16-bit V, P is rounded to
// V's type (the sum that divides it is not); with fp32 V both are split.
template <typename T, int DP, int NK, int LD>
__device__ __forceinline__ void weigh(float (&o)[DP / 8][4], const float (&p)[NK / 8][4], const T* v, int lane) {
  if constexpr (std::is_same_v<T, float>) {
    const int r = lane >> 2, c = lane & 3;
    constexpr int kKeys = NK / 8 < kChain ? NK / 8 : kChain;
#pragma unroll
    for (int n0 = 0; n0 < NK / 8; n0 += kKeys) {
      // the order of keys within a product is free: slot c holds key 2c, slot c + 4 key 2c + 1, as p's registers do
      Split pa[kKeys][4];
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        const float(&x)[4] = p[n0 + i];
        pa[i][0] = split(x[0]), pa[i][1] = split(x[2]), pa[i][2] = split(x[1]), pa[i][3] = split(x[3]);
      }
#pragma unroll
      for (int d0 = 0; d0 < DP / 8; d0 += kWide) {
        float hh[kWide][4] = {}, x[kWide][4] = {};
#pragma unroll
        for (int i = 0; i < kKeys; ++i)
#pragma unroll
          for (int d = 0; d < kWide; ++d) {
            const float* y = v + ((n0 + i) * 8 + 2 * c) * LD + (d0 + d) * 8 + r;
            mma_3xtf32(hh[d], x[d], pa[i], split(y[0]), split(y[LD]));
          }
#pragma unroll
        for (int d = 0; d < kWide; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d0 + d][i] += hh[d][i] + x[d][i];
      }
    }
  } else {
    const uint32_t vrow = smem_addr(v + ((lane & 7) + ((lane >> 3) & 1) * 8) * LD + (lane >> 4) * 8);
#pragma unroll
    for (int n = 0; n < NK / 16; ++n) {
      const uint32_t pa[4] = {pack2(p[2 * n][0], p[2 * n][1], (T*)nullptr), pack2(p[2 * n][2], p[2 * n][3], (T*)nullptr),
                              pack2(p[2 * n + 1][0], p[2 * n + 1][1], (T*)nullptr),
                              pack2(p[2 * n + 1][2], p[2 * n + 1][3], (T*)nullptr)};
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        uint32_t vb[4];
        ldmatrix4_trans(vb, vrow + (n * 16 * LD + d * 16) * 2);
        mma16(o[2 * d], pa, vb[0], vb[1], (T*)nullptr);
        mma16(o[2 * d + 1], pa, vb[2], vb[3], (T*)nullptr);
      }
    }
  }
}

// The running softmax of a warp's 16 rows (two per thread): maximum m in units
// of log2, sum l of this thread's columns.
struct Running {
  float m[2], l[2];
};
template <typename T>
__device__ __forceinline__ float lse_of(float m, float l) {
  return ((m == -INFINITY ? 0.0f : m) - kShift<T>) * kLn2 + logf(l);
}
// Turns scores into weights exp2(s - m + kShift), after masking keys at or past
// vis[row], and rescales o.
template <typename T, int NK, int ND>
__device__ __forceinline__ void softmax_step(float (&s)[NK / 8][4], float (&o)[ND][4], Running& st, float scale_log2,
                                             int key0, const int (&vis)[2], bool masked, int lane) {
  float top[2] = {st.m[0], st.m[1]};
#pragma unroll
  for (int n = 0; n < NK / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[n][i] *= scale_log2;
      if (masked && key0 + n * 8 + (lane & 3) * 2 + (i & 1) >= vis[i >> 1]) s[n][i] = -INFINITY;
      top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
    }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
    top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
  }
  if (__any_sync(0xffffffffu, top[0] != st.m[0] || top[1] != st.m[1])) {  // a maximum has moved
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float keep = ex2(st.m[r] - (top[r] == -INFINITY ? 0.0f : top[r]));
      st.m[r] = top[r];
      st.l[r] *= keep;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        o[d][2 * r] *= keep;
        o[d][2 * r + 1] *= keep;
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) top[r] = (top[r] == -INFINITY ? 0.0f : top[r]) - kShift<T>;
#pragma unroll
  for (int n = 0; n < NK / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[n][i] = ex2(s[n][i] - top[i >> 1]);
      st.l[i >> 1] += s[n][i];
    }
}

// ------------------------------------------------------------------ rows kernel
// Warps of 16 rows each share tiles of NK keys and values, double buffered by
// cp.async.  fp32: eight warps, so that one CTA, which is all that shared
// memory holds at 128 columns, fills the SM.
template <typename T>
constexpr int rows_warps() {
  return sizeof(T) == 4 ? 8 : 4;
}
template <typename T, int DP, int NK>
struct RowsCfg {
  static constexpr int kWarps = rows_warps<T>(), kRows = 16 * kWarps, kThreads = 32 * kWarps;
  static constexpr int LD = DP + 16 / (int)sizeof(T);  // rows 16 bytes apart in the banks
  static constexpr size_t kSmem = sizeof(T) * LD * (kRows + 4 * NK);
  static_assert(kSmem + 1024 <= kMaxSmem, "no block holds this");
};

template <typename T, int DP, int NK>
__global__ void __launch_bounds__(RowsCfg<T, DP, NK>::kThreads) attn_rows_kernel(AttnArgs a) {
  using C = RowsCfg<T, DP, NK>;
  constexpr int LD = C::LD, kVec = 16 / sizeof(T), kPerRow = DP / kVec;
  extern __shared__ __align__(16) uint8_t raw[];
  T* sq = reinterpret_cast<T*>(raw);
  T* sk = sq + C::kRows * LD;
  T* sv = sk + 2 * NK * LD;
  __shared__ int s_max[C::kWarps], s_least[C::kWarps], s_replaced;
  begin(a);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Item w = item_at(a, a.first_item + blockIdx.x, C::kRows);
  const int64_t n_rows = (int64_t)a.batch * a.queries * a.heads_q;

  // this thread's two rows
  const int row[2] = {warp * 16 + (lane >> 2), warp * 16 + (lane >> 2) + 8};
  int vis[2];
  int top = 0, low = 0x7fffffff, least = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    vis[r] = row[r] < w.rows ? visible(a, w.base + (w.row0 + row[r]) / a.group) : 0;
    top = max(top, vis[r]);
    if (row[r] < w.rows) low = min(low, vis[r]);
    if (vis[r] > w.k0) least = min(least, vis[r]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  low = __reduce_min_sync(0xffffffffu, low);
  least = __reduce_min_sync(0xffffffffu, least);
  if (lane == 0) s_max[warp] = top, s_least[warp] = least;
  if (tid == 0) s_replaced = kNoKey;
  __syncthreads();
  int end = 0;
#pragma unroll
  for (int i = 0; i < C::kWarps; ++i) end = max(end, s_max[i]), least = min(least, s_least[i]);
  end = min(end, w.k1);
  const int uneven = least < end ? uneven_from(w, least, NK) : kNoKey;

  const T* kp = static_cast<const T*>(a.k) + w.h * a.k_h;
  const T* vp = static_cast<const T*>(a.v) + w.h * a.v_h;
  for (int i = tid; i < C::kRows * kPerRow; i += C::kThreads) {
    const int r = i / kPerRow, c = (i - r * kPerRow) * kVec;
    const bool in = r < w.rows && c < a.dim;
    cp_async16(sq + r * LD + c, static_cast<const T*>(query_of(a, w, in ? r : 0, sizeof(T))) + (in ? c : 0), in);
  }
  auto load = [&](int key0, int buf) {
    for (int i = tid; i < NK * kPerRow; i += C::kThreads) {
      const int n = i / kPerRow, c = (i - n * kPerRow) * kVec;
      const int j = key0 + n;
      const bool in = j < end && c < a.dim;
      int64_t page = 0;
      int slot = 0;
      if (in) {
        const int pj = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
        slot = j - pj * a.page_size;
        page = min(max(w.pages[pj], 0), a.pages - 1);
      }
      const int cc = in ? c : 0;
      cp_async16(sk + (buf * NK + n) * LD + c, kp + page * a.k_p + slot * a.k_s + cc, in);
      cp_async16(sv + (buf * NK + n) * LD + c, vp + page * a.v_p + slot * a.v_s + cc, in);
    }
    cp_async_commit();
  };

  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[d][i] = 0.0f;
  Running st{{-INFINITY, -INFINITY}, {0.0f, 0.0f}};
  if (w.k0 < end) load(w.k0, 0);
  int buf = 0, key0 = w.k0;
  auto step = [&](auto look) {  // look: at values that not all rows see
    if (key0 + NK < end) {
      load(key0 + NK, buf ^ 1);
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    if constexpr (look) {
      if (replace_nonfinite_rows<T, NK, kPerRow, LD, C::kThreads>(smem_addr(sv + buf * NK * LD), tid)) s_replaced = uneven;
      __syncthreads();
    }
    float s[NK / 8][4];
    scores<T, DP, NK, LD>(s, sq + warp * 16 * LD, sk + buf * NK * LD, lane);
    const int seen[2] = {min(vis[0], end), min(vis[1], end)};
    softmax_step<T, NK, DP / 8>(s, o, st, a.scale_log2, key0, seen, key0 + NK > min(low, end), lane);
    weigh<T, DP, NK, LD>(o, s, sv + buf * NK * LD, lane);
    __syncthreads();
  };
  // two loops, so that the first has nothing to ask
  for (; key0 < min(end, uneven); key0 += NK, buf ^= 1) step(std::false_type{});
  for (; key0 < end; key0 += NK, buf ^= 1) step(std::true_type{});
  cp_async_wait<0>();  // the queries' copies, where there was no key

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    if (row[r] >= w.rows) continue;
    const int64_t at = row_index(a, w, row[r]);
    const bool none = st.l[r] == 0.0f;
    const float inv = none ? 0.0f : 1.0f / st.l[r];
    const float lse = none ? -INFINITY : lse_of<T>(st.m[r], st.l[r]);
    if (a.part_o) {
      const int64_t slot = (int64_t)w.split * n_rows + at;
      if ((lane & 3) == 0) a.part_lse[at * a.splits + w.split] = lse;
      if (none) continue;  // the join does not read it
      float* y = a.part_o + slot * a.dim;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        const int c = d * 8 + (lane & 3) * 2;
        if (c < a.dim) *reinterpret_cast<float2*>(y + c) = make_float2(o[d][2 * r] * inv, o[d][2 * r + 1] * inv);
      }
    } else {
      if ((lane & 3) == 0) a.lse[at] = lse;
      T* y = static_cast<T*>(a.out) + at * a.dim;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        const int c = d * 8 + (lane & 3) * 2;
        if (c < a.dim) {
          y[c] = from_f32<T>(none ? 0.0f : o[d][2 * r] * inv);
          y[c + 1] = from_f32<T>(none ? 0.0f : o[d][2 * r + 1] * inv);
        }
      }
    }
  }
  if (s_replaced != kNoKey) {
    const Item again = item_again(a, a.first_item, C::kRows);
    for (int i = 0; i < 2 * (DP / 8); ++i) {
      const int c = (i >> 1) * 8 + (threadIdx.x & 3) * 2;
      write_nonfinite<T>(a, again, (threadIdx.x >> 5) * 16 + ((threadIdx.x & 31) >> 2) + (i & 1) * 8, s_replaced, c, c + 2);
    }
  }
  wait_for_previous();  // as in the keys kernel
}

// ------------------------------------------------------------------ keys kernel
// Tiles of 16 rows: each of four warps takes every fourth block of NK keys, with
// a ring of its own filled by cp.async (no barrier until the end), and its own
// running softmax; the four are joined in shared memory.  This is the shape of
// decoding: a few query heads per key head against a sequence's own keys,
// bound by the bytes of the cache.  Two stages, and blocks of 8 keys for 128
// columns of fp32: what they leave of shared memory goes to more CTAs per SM.
// Against one more stage (128 columns), 64 sequences of up to 1000 keys: 42
// against 47 us; against four (64 columns): 60 against 89 us for 100 sequences
// of 8 queries in fp32, 26 against 32 us for 64 of one query in fp16; blocks of
// 8 against 16 (fp32, 16 sequences of up to 1024 keys): 27 against 37 us.
// EVEN: the launch has only items whose rows all see the same keys (the own keys of
// one query a sequence); what the others look at cost these 4 to 7 %.
template <typename T, int DP, int NK, int STAGES>
struct KeysCfg {
  static constexpr int kRows = 16, kWarps = 4, kThreads = 128;
  static constexpr int LD = DP + 16 / (int)sizeof(T);
  static constexpr int kStage = 2 * NK * LD;  // elements: keys, values
  static constexpr size_t kRing = sizeof(T) * kWarps * STAGES * kStage;
  static constexpr size_t kJoin = sizeof(float) * kWarps * kRows * (DP + 4);
  static constexpr size_t kSmem = sizeof(T) * kRows * LD + (kRing > kJoin ? kRing : kJoin);
  static_assert(kSmem + 1024 <= kMaxSmem, "no block holds this");
};

template <typename T, int DP, int NK, int STAGES, bool EVEN>
__global__ void __launch_bounds__(128) attn_keys_kernel(AttnArgs a) {
  using C = KeysCfg<T, DP, NK, STAGES>;
  constexpr int LD = C::LD, kVec = 16 / sizeof(T), kPerRow = DP / kVec;
  extern __shared__ __align__(16) uint8_t raw[];
  T* sq = reinterpret_cast<T*>(raw);
  T* ring = sq + C::kRows * LD;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_replaced;
  begin(a);
  if (!EVEN && threadIdx.x == 0) s_replaced = kNoKey;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Item w = item_at(a, a.first_item + blockIdx.x, C::kRows);
  const int64_t n_rows = (int64_t)a.batch * a.queries * a.heads_q;
  const T* kp = static_cast<const T*>(a.k) + w.h * a.k_h;
  const T* vp = static_cast<const T*>(a.v) + w.h * a.v_h;
  T* mine = ring + warp * STAGES * C::kStage;
  // A CTA lives for a few blocks, so its start counts: the queries, the pages
  // and the lengths are read at once, and the keys as soon as those are there
  // (one after the other they took 5 us until the first keys).
  for (int i = tid; i < C::kRows * kPerRow; i += C::kThreads) {
    const int r = i / kPerRow, c = (i - r * kPerRow) * kVec;
    const bool in = r < w.rows && c < a.dim;
    cp_async16(sq + r * LD + c, static_cast<const T*>(query_of(a, w, in ? r : 0, sizeof(T))) + (in ? c : 0), in);
  }
  // Where this lane's key of the block at key0 lies (lanes past NK repeat):
  // looked up once per key, before it is known whether any row sees it.
  const bool alike = a.k_p == a.v_p && a.k_s == a.v_s;
  struct Place {
    int64_t k, v;
  };
  auto place = [&](int key0) {
    const int j = key0 + lane % NK;
    Place p{0, 0};
    if (j < w.k1) {
      const int pj = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
      const int slot = j - pj * a.page_size;
      const int64_t page = min(max(w.pages[pj], 0), a.pages - 1);
      p.k = page * a.k_p + slot * a.k_s;
      p.v = alike ? p.k : page * a.v_p + slot * a.v_s;
    }
    return p;
  };
  constexpr int kStep = C::kWarps * NK;
  const int begin = w.k0 + warp * NK;
  Place first[STAGES];
#pragma unroll
  for (int i = 0; i < STAGES; ++i) first[i] = place(begin + i * kStep);
  const int row[2] = {lane >> 2, (lane >> 2) + 8};
  int vis[2], top = 0, low = 0x7fffffff, least = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    vis[r] = row[r] < w.rows ? visible(a, w.base + (w.row0 + row[r]) / a.group) : 0;
    top = max(top, vis[r]);
    if (row[r] < w.rows) low = min(low, vis[r]);
    if (vis[r] > w.k0) least = min(least, vis[r]);
  }
  const int end = min(w.k1, __reduce_max_sync(0xffffffffu, top));
  low = __reduce_min_sync(0xffffffffu, low);
  least = __reduce_min_sync(0xffffffffu, least);
  const int uneven = !EVEN && least < end ? uneven_from(w, least, NK) : kNoKey;

  auto load = [&](int key0, const Place& p, int stage) {
    T* sk = mine + stage * C::kStage;
    T* sv = sk + NK * LD;
    if (alike && key0 + NK <= end && a.dim == DP && kPerRow <= 32) {
      // a whole block: every copy of a lane has the same column
      constexpr int kRowsAt = kPerRow <= 32 ? 32 / kPerRow : 1;
      const int n0 = lane / kPerRow, c = lane % kPerRow * kVec;
      const uint32_t dst = smem_addr(sk + n0 * LD + c);
#pragma unroll
      for (int i = 0; i < NK / kRowsAt; ++i) {
        const int64_t at = __shfl_sync(0xffffffffu, p.k, i * kRowsAt + n0) + c;
        copy16(dst + i * kRowsAt * LD * (int)sizeof(T), kp + at);
        copy16(dst + (NK + i * kRowsAt) * LD * (int)sizeof(T), vp + at);
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < NK * kPerRow / 32; ++i) {
      const int at = i * 32 + lane, n = at / kPerRow, c = at % kPerRow * kVec;
      const int64_t k = __shfl_sync(0xffffffffu, p.k, n);
      const int64_t v = alike ? k : __shfl_sync(0xffffffffu, p.v, n);
      const bool in = key0 + n < end && c < a.dim;
      const int cc = in ? c : 0;
      cp_async16(sk + n * LD + c, kp + k + cc, in);
      cp_async16(sv + n * LD + c, vp + v + cc, in);
    }
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (begin + i * kStep < end) load(begin + i * kStep, first[i], i);
    cp_async_commit();
  }
  Place next = first[STAGES - 1];

  float o[DP / 8][4];
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[d][i] = 0.0f;
  Running st{{-INFINITY, -INFINITY}, {0.0f, 0.0f}};
  const int seen[2] = {min(vis[0], end), min(vis[1], end)};
  // The queries came with each warp's first copies; a warp without a block meets the others here, too.
  auto queries_there = [&] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
  if (begin >= end) {
    cp_async_wait<0>();
    queries_there();
  }
  int stage = 0, key0 = begin;
  auto step = [&](auto look) {  // look: at values that not all rows see
    const int ahead = key0 + (STAGES - 1) * kStep;
    if (ahead < end) load(ahead, next, stage == 0 ? STAGES - 1 : stage - 1);
    cp_async_commit();
    next = place(ahead + kStep);
    cp_async_wait<STAGES - 1>();
    if (key0 == begin) queries_there();
    __syncwarp();
    const T* sk = mine + stage * C::kStage;
    if constexpr (look) {
      if (replace_nonfinite_rows<T, NK, kPerRow, LD, 32>(smem_addr(sk + NK * LD), lane)) s_replaced = uneven;
      __syncwarp();
    }
    float s[NK / 8][4];
    scores<T, DP, NK, LD>(s, sq, sk, lane);
    softmax_step<T, NK, DP / 8>(s, o, st, a.scale_log2, key0, seen, key0 + NK > min(low, end), lane);
    weigh<T, DP, NK, LD>(o, s, sk + NK * LD, lane);
    __syncwarp();  // all lanes are done with the stage that the next load fills
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  };
  // two loops, so that the first has nothing to ask
  for (; key0 < min(end, uneven); key0 += kStep) step(std::false_type{});
  if constexpr (!EVEN)
    for (; key0 < end; key0 += kStep) step(std::true_type{});
  cp_async_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    if ((lane & 3) == 0) s_m[warp][row[r]] = st.m[r], s_l[warp][row[r]] = st.l[r];
  }
  __syncthreads();  // the rings are free
  float* so = reinterpret_cast<float*>(ring);
  constexpr int LO = DP + 4;
#pragma unroll
  for (int d = 0; d < DP / 8; ++d)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      *reinterpret_cast<float2*>(so + (warp * 16 + row[r]) * LO + d * 8 + (lane & 3) * 2) =
          make_float2(o[d][2 * r], o[d][2 * r + 1]);
  __syncthreads();
  // eight threads a row
  const int r = tid >> 3;
  // Where this launch began before the prefix's had ended: it ends after it, so
  // that the join, which waits for this one, has both.
  if (tid == 127) wait_for_previous();
  if (r >= w.rows) return;
  float m = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
  const float base = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = ex2(s_m[i][r] - base);
    l += f[i] * s_l[i][r];
  }
  const int64_t at = row_index(a, w, r);
  const int64_t slot = (int64_t)w.split * n_rows + at;
  const bool none = l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  const float lse = none ? -INFINITY : lse_of<T>(m, l);
  if ((tid & 7) == 0) (a.part_o ? a.part_lse[at * a.splits + w.split] : a.lse[at]) = lse;
  if (a.part_o && none) return;  // the join does not read it
  for (int d = (tid & 7) * 4; d < a.dim; d += 32) {
    float y[4] = {};
    if (!none) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (f[i] == 0.0f) continue;  // a warp without keys
        const float4 x = *reinterpret_cast<const float4*>(so + (i * 16 + r) * LO + d);
        y[0] += f[i] * x.x, y[1] += f[i] * x.y, y[2] += f[i] * x.z, y[3] += f[i] * x.w;
      }
    }
    if (a.part_o) {
      *reinterpret_cast<float4*>(a.part_o + slot * a.dim + d) = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
    } else {
      T* z = static_cast<T*>(a.out) + at * a.dim + d;
#pragma unroll
      for (int i = 0; i < 4; ++i) z[i] = from_f32<T>(y[i] * inv);
    }
  }
  if (!EVEN && s_replaced != kNoKey) {
    const Item again = item_again(a, a.first_item, C::kRows);
    for (int d = (threadIdx.x & 7) * 4; d < a.dim; d += 32)
      write_nonfinite<T>(a, again, threadIdx.x >> 3, s_replaced, d, d + 4);
  }
}

// ------------------------------------------------------------------ join
// One warp per row: the parts weighed by exp(lse_i - L), in their order.  Lane
// i holds the weight of part i; a part without keys has weight 0 and is not
// read (nothing was written there).
constexpr int kJoin = 8;
template <typename T>
__global__ void __launch_bounds__(128) attn_join_kernel(const float* part_o, const float* part_lse, int splits,
                                                        int64_t rows, int dim, T* out, float* lse) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  allow_next();
  wait_for_previous();  // for the parts
  if (row >= rows) return;
  part_lse += row * splits;
  const float first = lane < splits ? part_lse[lane] : -INFINITY;
  float top = first;
  for (int i = lane + 32; i < splits; i += 32) top = fmaxf(top, part_lse[i]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;  // a NaN part makes it NaN
  float acc[2][4] = {};
  for (int i0 = 0; i0 < splits; i0 += 32) {
    const float l = i0 == 0 ? first : i0 + lane < splits ? part_lse[i0 + lane] : -INFINITY;
    const float weight = ex2((l - base) * kLog2e);
    total += weight;
    const int n = min(32, splits - i0);
    const float* y = part_o + (i0 * rows + row) * dim + lane * 4;
    const int64_t step = rows * dim;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h * 128 >= dim) break;
      const bool mine = lane * 4 + h * 128 < dim;
      for (int j = 0; j < n; j += kJoin) {  // loads of kJoin parts in flight
        float4 x[kJoin];
        float f[kJoin];
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {
          f[i] = __shfl_sync(0xffffffffu, weight, (j + i) & 31);
          if (j + i >= n) f[i] = 0.0f;
          x[i] = mine && f[i] != 0.0f ? *reinterpret_cast<const float4*>(y + (j + i) * step + h * 128)
                                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kJoin; ++i)
          acc[h][0] += f[i] * x[i].x, acc[h][1] += f[i] * x[i].y, acc[h][2] += f[i] * x[i].z, acc[h][3] += f[i] * x[i].w;
      }
    }
  }
  total = warp_sum(total);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (lane * 4 + h * 128 < dim)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[row * dim + lane * 4 + h * 128 + i] = from_f32<T>(acc[h][i] * inv);
  if (lane == 0) lse[row] = total == 0.0f ? -INFINITY : base + logf(total);
}

// ------------------------------------------------------------------ host side
enum Kind { kKeys, kRows, kTensor };
struct Part {
  Kind kind = kKeys;
  int tiles = 0, splits = 0, chunk = 1;
};
struct Plan {
  Part prefix, own;
  int splits() const { return prefix.splits + own.splits; }
};

// One axis of keys for `sets` sets of `rows` query rows each: the kernel by
// the number of rows, and ranges of keys that give every SM a few CTAs but no
// CTA less than one block of keys.
Part plan_part(int64_t sets, int64_t rows, int64_t keys, int64_t dim, int dtype, bool tensor) {
  Part p;
  if (keys <= 0) return p;
  const bool f32 = dtype == KB_F32;
  // Up to a few row tiles the keys kernel reads the keys again for each (from
  // L2) and is still faster than a wider tile that stays half empty (8 key heads
  // x 128): fp32, 48 rows over 32000 keys 265 against 302 us (64: 342 against
  // 300); 16-bit on mma.sync, 32 rows over 8192 keys 24 against 32, 64 rows 33
  // against 35 (over 2048, 17 against 17).
  const bool few = rows <= (f32 ? 64 : tensor ? 16 : 48);
  // And where there is little to do, for it starts and ends sooner.  16-bit
  // against tcgen05, 8 heads x 128: 64 rows over 64 keys 7.7 against 13 us, over
  // 2048 17 against 19, over 8192 33 against 26; 512 rows over 256 keys 28
  // against 29, over 1024 40 against 34; one head, 32 rows over 4096 keys 12
  // against 15, over 32000 34 against 23.  fp32 against the rows kernel, 4 heads:
  // 96 rows over 2080 keys x 128 27 against 37, x 64 18 against 22; 128 rows over
  // 320 keys x 128 15 against 36, over 2080 39 against 37.
  const double each = (double)rows * dim * keys;
  const bool little = (f32 || tensor) && each <= (f32 ? 3e7 : 2e7) && 4.0 * sets * each < 1.2e9;
  p.kind = few || little ? kKeys : tensor ? kTensor : kRows;
  if (p.kind == kTensor) {
    // One CTA per SM, equal ranges of whole 128-key tiles: the number of
    // ranges that makes the last wave end first, a range's fixed cost (the
    // queries, the first scores, the way out) counted as kFixed tiles.
    constexpr int64_t kFixed = 3;
    p.tiles = (int)ceil_div(rows, (int64_t)(f32 ? kTc32Rows : tc_tile_rows(rows)));
    const int64_t items = p.tiles * sets, tiles = ceil_div(keys, 128), most = std::min<int64_t>(tiles, 64);
    int64_t best = 0;
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t each = ceil_div(tiles, s), n = ceil_div(tiles, each);
      const int64_t cost = ceil_div(items * n, (int64_t)sm_count()) * (each + kFixed);
      if (best == 0 || cost < best) best = cost, p.chunk = (int)each * 128, p.splits = (int)n;
    }
    return p;
  }
  const int tile = p.kind == kKeys ? 16 : 16 * (f32 ? rows_warps<float>() : rows_warps<__half>());
  p.tiles = (int)ceil_div(rows, tile);
  const int64_t block = 64, least = p.kind == kKeys ? block : 2 * block;
  const int64_t items = p.tiles * sets;
  const int64_t s = std::max<int64_t>(1, std::min(ceil_div((int64_t)4 * sm_count(), items), ceil_div(keys, least)));
  p.chunk = (int)(ceil_div(ceil_div(keys, s), block) * block);
  p.splits = (int)ceil_div(keys, p.chunk);
  return p;
}
Plan plan(int64_t batch, int64_t queries, int64_t heads_q, int64_t heads_kv, int64_t dim, int64_t prefix_keys,
          int64_t own_keys, int dtype, bool tensor) {
  const int64_t rows = queries * (heads_q / heads_kv);
  return {plan_part(heads_kv, batch * rows, prefix_keys, dim, dtype, tensor),
          plan_part(heads_kv * batch, rows, own_keys, dim, dtype, false)};
}
// At most 2^30 rows, and keys of a sequence.  One by one before their products, which
// have to fit 64 bits.
bool sizes_fit(int64_t batch, int64_t queries, int64_t heads_q, int64_t prefix_pages, int64_t width, int64_t page_size) {
  constexpr int64_t kMost = 0x3fffffff;
  return batch <= kMost && queries <= kMost && batch * queries <= kMost && heads_q <= kMost &&
         batch * queries * heads_q <= kMost && prefix_pages <= kMost && width <= kMost && page_size <= kMost &&
         std::max(prefix_pages, width) * page_size <= kMost;
}
// Parts, then (fp32 on the tensor cores) the prefix in halves.
size_t part_bytes(const Plan& p, int64_t rows, int64_t dim) {
  return p.splits() <= 1 ? 0 : (size_t)ceil_div(p.splits() * rows * (dim + 1), 4) * 16;
}

template <typename K>
int launch(K kern, int threads, size_t smem, AttnArgs a, int64_t first, int64_t items, uint64_t& attr_set,
           cudaStream_t stream) {
  if (items == 0) return KB_OK;
  int dev = 0;
  KB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(attr_set >> dev & 1)) {  // one bit per device ordinal
    KB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    if (dev < 64) attr_set |= 1ull << dev;
  }
  a.first_item = first;
  return launch_after(kern, dim3((unsigned)items), (unsigned)threads, smem, stream, a);
}
template <typename T, int DP, int NK>
int launch_rows(const AttnArgs& a, int64_t first, int64_t items, cudaStream_t stream) {
  static uint64_t attr_set = 0;
  using C = RowsCfg<T, DP, NK>;
  return launch(attn_rows_kernel<T, DP, NK>, C::kThreads, C::kSmem, a, first, items, attr_set, stream);
}
template <typename T, int DP, int NK, int STAGES, bool EVEN>
int launch_keys_as(const AttnArgs& a, int64_t first, int64_t items, cudaStream_t stream) {
  static uint64_t attr_set = 0;
  return launch(attn_keys_kernel<T, DP, NK, STAGES, EVEN>, 128, KeysCfg<T, DP, NK, STAGES>::kSmem, a, first, items,
                attr_set, stream);
}
template <typename T, int DP, int NK, int STAGES>
int launch_keys(const AttnArgs& a, int64_t first, int64_t items, cudaStream_t stream) {
  return first >= a.prefix_items && a.queries == 1 ? launch_keys_as<T, DP, NK, STAGES, true>(a, first, items, stream)
                                                   : launch_keys_as<T, DP, NK, STAGES, false>(a, first, items, stream);
}
template <typename T>
int launch_kind(Kind kind, const AttnArgs& a, int64_t first, int64_t items, cudaStream_t stream) {
  constexpr bool f32 = sizeof(T) == 4;
  if (kind == kKeys) {
    if (a.dim <= 64) return launch_keys<T, 64, 16, 2>(a, first, items, stream);
    if (a.dim <= 128) return launch_keys<T, 128, f32 ? 8 : 16, 2>(a, first, items, stream);
    return launch_keys<T, 256, f32 ? 8 : 16, 3>(a, first, items, stream);
  }
  if (a.dim <= 64) return launch_rows<T, 64, 64>(a, first, items, stream);
  if (a.dim <= 128) return launch_rows<T, 128, f32 ? 32 : 64>(a, first, items, stream);
  return launch_rows<T, 256, f32 ? 16 : 64>(a, first, items, stream);  // fp32: 200 KB with its 128 rows
}

}  // namespace
}  // namespace attn
}  // namespace lm
}  // namespace kb

extern "C" {

size_t kb_shared_prefix_attention_workspace_size(int64_t batch, int64_t queries, int64_t heads_q, int64_t heads_kv,
                                                 int64_t dim, int64_t prefix_pages, int64_t width,
                                                 int64_t page_size, int dtype) {
  using namespace kb::lm::attn;
  if (batch <= 0 || queries <= 0 || heads_q <= 0 || heads_kv <= 0 || dim <= 0 || page_size <= 0 || prefix_pages < 0 ||
      heads_q % heads_kv || !sizes_fit(batch, queries, heads_q, prefix_pages, width, page_size))
    return 0;
  const int64_t keys = prefix_pages * page_size;
  auto bytes = [&](bool tensor) {
    return part_bytes(plan(batch, queries, heads_q, heads_kv, dim, keys,
                           std::max<int64_t>(0, width - prefix_pages) * page_size, dtype, tensor),
                      batch * queries * heads_q, dim);
  };
  if (dtype == KB_F32) {
    const bool tensor = tc32_pays(batch * queries * (heads_q / heads_kv), heads_kv, dim, keys);
    return bytes(tensor) + (tensor ? tc32_bytes(heads_kv, dim, keys) : 0);
  }
  // strides decide whether the tensor-core kernel can take the prefix
  return std::max(bytes(false), bytes(true));
}

int kb_shared_prefix_attention(const void* q, const void* k_pages, const void* v_pages, const int32_t* prefix,
                               const int32_t* table, const int32_t* lens, void* out, float* lse, int64_t batch,
                               int64_t queries, int64_t heads_q, int64_t heads_kv, int64_t dim, int64_t prefix_pages,
                               int64_t width, int64_t pages, int64_t page_size, int64_t q_stride_seq,
                               int64_t q_stride_query, int64_t q_stride_head, int64_t k_stride_page,
                               int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_page,
                               int64_t v_stride_slot, int64_t v_stride_head, float scale, int dtype, void* workspace,
                               size_t workspace_bytes, kbStream stream) {
  const char* name = "kb_shared_prefix_attention";
  using namespace kb::lm;
  using namespace kb::lm::attn;
  KB_REQUIRE(batch >= 0 && queries >= 0 && heads_q >= 0 && heads_kv >= 0 && dim >= 0 && prefix_pages >= 0 &&
                 width >= 0 && pages >= 0 && page_size >= 1,
             KB_ERR_INVALID_ARG, "%s: negative size", name);
  KB_REQUIRE(dtype_size(dtype), KB_ERR_INVALID_ARG, "%s: unknown element type", name);
  if (batch == 0 || queries == 0 || heads_q == 0 || dim == 0) return KB_OK;
  KB_REQUIRE(sizes_fit(batch, queries, heads_q, prefix_pages, width, page_size), KB_ERR_UNSUPPORTED,
             "%s: too many rows or keys", name);
  const int64_t rows = batch * queries * heads_q;
  KB_REQUIRE(heads_kv >= 1 && heads_q % heads_kv == 0, KB_ERR_INVALID_ARG,
             "%s: %lld query heads do not divide into %lld key heads", name, (long long)heads_q, (long long)heads_kv);
  KB_REQUIRE(q && lens && out && lse, KB_ERR_INVALID_ARG, "%s: null pointer", name);
  const int64_t own_pages = std::max<int64_t>(0, width - prefix_pages);
  KB_REQUIRE((prefix_pages == 0 || prefix) && (own_pages == 0 || table), KB_ERR_INVALID_ARG, "%s: null table", name);
  KB_REQUIRE(prefix_pages + own_pages == 0 || (pages >= 1 && k_pages && v_pages), KB_ERR_INVALID_ARG,
             "%s: pages without a pool", name);
  const int e = dtype_size(dtype);
  KB_REQUIRE(dim <= 256 && dim * e % 16 == 0, KB_ERR_UNSUPPORTED,
             "%s: head dim %lld must be at most 256 and fill whole 16-byte vectors", name, (long long)dim);
  auto whole = [&](int64_t s) { return s * e % 16 == 0; };
  KB_REQUIRE(kb::aligned16(q) && kb::aligned16(k_pages) && kb::aligned16(v_pages) && kb::aligned16(out) &&
                 whole(q_stride_seq) && whole(q_stride_query) && whole(q_stride_head) && whole(k_stride_page) &&
                 whole(k_stride_slot) && whole(k_stride_head) && whole(v_stride_page) && whole(v_stride_slot) &&
                 whole(v_stride_head),
             KB_ERR_UNSUPPORTED, "%s: queries, pools and their strides must be multiples of 16 bytes", name);
  KB_REQUIRE(pages <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: too many pages", name);
  AttnArgs a{};
  a.q = q, a.k = k_pages, a.v = v_pages, a.out = out, a.lse = lse;
  a.prefix = prefix, a.table = table, a.lens = lens;
  a.batch = (int)batch, a.queries = (int)queries, a.heads_q = (int)heads_q, a.heads_kv = (int)heads_kv;
  a.group = (int)(heads_q / heads_kv), a.dim = (int)dim;
  a.prefix_pages = (int)prefix_pages, a.width = (int)width, a.pages = (int)pages, a.page_size = (int)page_size;
  a.page_shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    while ((int64_t)1 << ++a.page_shift < page_size) {
    }
  a.q_b = q_stride_seq, a.q_t = q_stride_query, a.q_h = q_stride_head;
  a.k_p = k_stride_page, a.k_s = k_stride_slot, a.k_h = k_stride_head;
  a.v_p = v_stride_page, a.v_s = v_stride_slot, a.v_h = v_stride_head;
  a.scale_log2 = scale * kLog2e;
  const int64_t keys = prefix_pages * page_size;
  const bool tensor = dtype == KB_F32 ? tc32_pays(batch * queries * a.group, heads_kv, dim, keys) : tc_fits(a, dtype);
  const Plan p = plan(batch, queries, heads_q, heads_kv, dim, keys, own_pages * page_size, dtype, tensor);
  a.splits = p.splits();
  a.prefix_tiles = p.prefix.tiles, a.prefix_splits = p.prefix.splits, a.prefix_chunk = p.prefix.chunk;
  a.own_tiles = p.own.tiles, a.own_splits = p.own.splits, a.own_chunk = p.own.chunk;
  a.prefix_items = (int64_t)p.prefix.tiles * p.prefix.splits * heads_kv;
  const int64_t items = a.prefix_items + (int64_t)p.own.tiles * p.own.splits * heads_kv * batch;
  KB_REQUIRE(items <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: too many work items", name);
  const bool halves = dtype == KB_F32 && p.prefix.kind == kTensor;
  void* scratch = nullptr;
  if (p.splits() > 1 || halves) {
    const size_t parts = part_bytes(p, rows, dim), need = parts + (halves ? tc32_bytes(heads_kv, dim, keys) : 0);
    KB_REQUIRE(workspace && workspace_bytes >= need, KB_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", name, need, workspace_bytes);
    KB_REQUIRE(kb::aligned16(workspace), KB_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name);
    if (p.splits() > 1) {
      a.part_o = static_cast<float*>(workspace);
      a.part_lse = a.part_o + (int64_t)p.splits() * rows * dim;
    }
    scratch = static_cast<char*>(workspace) + parts;
  }
  return with_dtype(dtype, [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    if (items) {
      if (p.prefix.kind == p.own.kind) {
        if (int st = launch_kind<T>(p.own.kind, a, 0, items, stream)) return st;
      } else {
        if (int st = halves                      ? tc32_launch(a, scratch, stream)
                     : p.prefix.kind == kTensor ? tc_launch(a, dtype, stream)
                                                : launch_kind<T>(p.prefix.kind, a, 0, a.prefix_items, stream))
          return st;
        if (int st = launch_kind<T>(p.own.kind, a, a.prefix_items, items - a.prefix_items, stream)) return st;
      }
      if (p.splits() == 1) return (int)KB_OK;
    }
    // also where there are no keys at all: zeros and -inf
    return launch_after(attn_join_kernel<T>, dim3((unsigned)kb::ceil_div(rows, 4)), 128u, 0, stream,
                        (const float*)a.part_o, (const float*)a.part_lse, p.splits(), rows, dim, static_cast<T*>(out),
                        lse);
  });
}

}  // extern "C"
