// lm_attention_tc32.cu — the shared prefix in fp32 on the fifth-generation
// tensor cores, with every operand as the sum of two fp16 values.
//
// x 2^e = hi + lo + r, hi = fp16(x 2^e), lo = fp16(x 2^e - hi): 22 bits of x, r
// below 2^-22 of it, where 2^e brings the largest magnitude of a query row, or of
// a key head's keys or values, to 2^13..2^14 (an element far below that largest
// keeps an absolute error of 2^-38 of it).  So neither another head nor another
// sequence's queries cost a result its bits.  Products: lo hi + hi lo + hi hi, exact in the tensor cores' fp32;
// lo lo is below fp32's resolution.  Three fp16 products cost less than the
// three of half the rate that TF32 halves would take, and 16-bit tiles fit
// shared memory.  The tensor cores' accumulation truncates, so the small cross
// terms go first, O is taken out after every key tile and summed with ordinary
// fp32 additions, and S is one chain of 24 steps of which 8 are large.
//
// Two launches before the kernel read the part of the prefix that some query
// sees: the largest magnitudes, then the halves of K and V into the workspace, [keys or values][hi, lo][head][key][64 or 128 columns],
// padded with zeros, from which TMA loads plain tiles.  They move 12 bytes per
// element where the products take 3 x 4 rows: they pay from a few dozen rows on.
//
// A CTA takes 128 query rows of one key head and a range of keys, in tiles of
// 128.  Roles (10 warps): warps 0-3 softmax (one thread per row), warps 4-7 the
// sum of O (one thread per row, in registers), warp 8 TMA (and a look at values
// that not all rows see), warp 9 products.
// S_{j+1} is issued before O_j = P_j V_j, into the other of two S buffers; P_j,
// hi and lo, takes S_j's 128 TMEM columns; O_j has two buffers.  TMEM: S 2 x
// 128, O 2 x 128.  Shared memory: Q, one K tile and one V tile, hi and lo, 64 KB
// each.
#include <float.h>

#include "lm_attention.cuh"
#include "lm_tc.cuh"

namespace kb {
namespace lm {
namespace attn {
namespace {

constexpr int kThreads = 320, kLoadWarp = 8, kMmaWarp = 9;
constexpr int kKeepBytes = 4 * kTile * 4;     // rescaling factors of four key tiles
constexpr int kSmemBytes = 6 * kTileBytes + kKeepBytes + 2 * kTile * 4 + 256 + 1024;
constexpr float kShift32 = 14.0f;             // weights are held 2^kShift32 high: their lo keeps its bits
constexpr int kLargest = 13;                  // log2 of what the largest magnitude becomes

// 2^e that brings magnitude `bits` (of a non-negative fp32) to 2^kLargest.
__device__ __forceinline__ int exponent_for(uint32_t bits) {
  return bits ? min(max(kLargest - ((int)(bits >> 23) - 127), -126), 126) : 0;
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// hi and lo of two values, packed
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const float a = x - f.x, b = y - f.y;  // exact; of a non-finite value 0, which says no more
  const __half2 l = __floats2half2_rn(isfinite(a) ? a : 0.0f, isfinite(b) ? b : 0.0f);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}

struct SplitArgs {
  AttnArgs a;
  uint32_t* largest;  // [2][heads_kv]: magnitudes of keys and values as bits
  __half* halves;     // [2][2][heads_kv][keys][cols]
  int keys, cols;     // padded
};

// The keys that some query sees, over the whole batch.
__device__ __forceinline__ int seen_keys(const AttnArgs& a) {
  __shared__ int s_top;
  if (threadIdx.x == 0) s_top = 0;
  __syncthreads();
  int top = 0;
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x) top = max(top, a.lens[b]);
  atomicMax(&s_top, top);
  __syncthreads();
  return min(s_top, a.prefix_pages * a.page_size);
}
// Four columns from column c of key j of head h (keys or values).
__device__ __forceinline__ float4 element4(const AttnArgs& a, bool values, int j, int h, int c) {
  const int pj = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
  const int64_t page = min(max(a.prefix[pj], 0), a.pages - 1), slot = j - pj * a.page_size;
  const float* x = values ? static_cast<const float*>(a.v) + page * a.v_p + slot * a.v_s + h * a.v_h
                          : static_cast<const float*>(a.k) + page * a.k_p + slot * a.k_s + h * a.k_h;
  return *reinterpret_cast<const float4*>(x + c);
}
__device__ __forceinline__ uint32_t magnitude(float4 x) {
  auto one = [](float v) {
    const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
  };
  return max(max(one(x.x), one(x.y)), max(one(x.z), one(x.w)));
}

// Grid of both: (blocks, key heads).
__global__ void __launch_bounds__(256) largest_kernel(SplitArgs s) {
  allow_next();
  const AttnArgs& a = s.a;
  const int seen = seen_keys(a), per_row = a.dim / 4, h = blockIdx.y;
  uint32_t top[2] = {};
  const int64_t n = (int64_t)seen * per_row;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int j = (int)(i / per_row), c = (int)(i - (int64_t)j * per_row) * 4;
    top[0] = max(top[0], magnitude(element4(a, false, j, h, c)));
    top[1] = max(top[1], magnitude(element4(a, true, j, h, c)));
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    top[kv] = __reduce_max_sync(0xffffffffu, top[kv]);
    if ((threadIdx.x & 31) == 0 && top[kv]) atomicMax(&s.largest[kv * a.heads_kv + h], top[kv]);
  }
}

__global__ void __launch_bounds__(256) halves_kernel(SplitArgs s) {
  allow_next();
  const AttnArgs& a = s.a;
  const int seen = seen_keys(a), per_row = s.cols / 4, h = blockIdx.y;
  wait_for_previous();
  const float scale[2] = {power2(exponent_for(s.largest[h])), power2(exponent_for(s.largest[a.heads_kv + h]))};
  const int64_t plane = (int64_t)a.heads_kv * s.keys * s.cols, n = (int64_t)s.keys * per_row;
#pragma unroll 2
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int j = (int)(i / per_row), c = (int)(i - (int64_t)j * per_row) * 4;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint2 hi = make_uint2(0, 0), lo = make_uint2(0, 0);
      if (j < seen && c < a.dim) {
        const float4 x = element4(a, kv, j, h, c);
        split2(x.x * scale[kv], x.y * scale[kv], hi.x, lo.x);
        split2(x.z * scale[kv], x.w * scale[kv], hi.y, lo.y);
      }
      __half* y = s.halves + 2 * kv * plane + ((int64_t)h * s.keys + j) * s.cols + c;
      *reinterpret_cast<uint2*>(y) = hi;
      *reinterpret_cast<uint2*>(y + plane) = lo;
    }
  }
}

__device__ __forceinline__ void tma_load3(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int col, int key, int plane) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(col), "r"(key), "r"(plane)
      : "memory");
}

template <int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
attn_prefix32_kernel(const __grid_constant__ CUtensorMap tm, const __grid_constant__ SplitArgs sp) {
  const AttnArgs& a = sp.a;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t *s_q = smem, *s_k = smem + 2 * kTileBytes, *s_v = smem + 4 * kTileBytes;  // hi, then lo
  float* s_keep = reinterpret_cast<float*>(smem + 6 * kTileBytes);                  // [4][rows]
  float* s_sum = s_keep + 4 * kTile;  // [2][rows]: first the largest magnitudes of a query's halves, at the end its sum
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_sum + 2 * kTile);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const uint32_t q_full = bar(0), k_full = bar(1), k_empty = bar(2), v_full = bar(3), v_empty = bar(4);
  auto s_full = [&](int j) { return bar(5 + (j & 1)); };
  // P and the rescaling factors of tile j: the softmax may be two tiles ahead of
  // the sum of O, which waits for these, but not four (S_{j+4} comes after
  // O_{j+2}, which comes after the sum has taken O_j)
  auto p_full = [&](int j) { return bar(7 + (j & 3)); };
  auto o_full = [&](int j) { return bar(11 + (j & 1)); };
  auto o_empty = [&](int j) { return bar(13 + (j & 1)); };
  const uint32_t v_landed = bar(15);  // a copy of values that are looked at before v_full
  const uint32_t written = bar(16);   // the rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_end = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_least = s_end + 1;
  __shared__ int s_replaced;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Item w = item_at(a, blockIdx.x, kTile);
  if (threadIdx.x == 0) {
    mbar_init(q_full, 2 * kTile);
    mbar_init(k_full, 1);
    mbar_init(k_empty, 1);
    mbar_init(v_full, 1);
    mbar_init(v_empty, 1);
    mbar_init(v_landed, 1);
    mbar_init(written, kTile);
    for (int j = 0; j < 2; ++j) {
      mbar_init(s_full(j), 1);
      mbar_init(p_full(j), kTile);
      mbar_init(p_full(j + 2), kTile);
      mbar_init(o_full(j), 1);
      mbar_init(o_empty(j), kTile);
    }
    *abort_flag = 0;
    *s_end = 0;
    *s_least = 0x7fffffff;
    s_replaced = kNoKey;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  __syncthreads();
  allow_next();
  const int row = threadIdx.x & (kTile - 1);
  int vis = 0;
  if (warp < 4) {
    if (row < w.rows) vis = visible(a, w.base + (w.row0 + row) / a.group);
    const int top = __reduce_max_sync(0xffffffffu, vis), low = __reduce_min_sync(0xffffffffu, vis > w.k0 ? vis : 0x7fffffff);
    if (lane == 0) atomicMax(s_end, top), atomicMin(s_least, low);
  }
  wait_for_previous();  // the halves and the magnitudes
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int end = min(w.k1, *s_end), least = *s_least;
  const int n = end > w.k0 ? (end - w.k0 + kTile - 1) / kTile : 0;
  // The first tile with values that not all rows of this CTA see, some, or only rows of others (they are in the halves,
  // too): warp 8 looks at them before they are used.
  const int look_from = max(least - w.k0, 0) / kTile;
  const int ek = exponent_for(sp.largest[w.h]), ev = exponent_for(sp.largest[a.heads_kv + w.h]);
  int eq = 0;  // of this thread's row
  const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16;
  auto s_col = [&](int j) { return tmem + (j & 1) * kTile; };
  auto o_col = [&](int j) { return tmem + 2 * kTile + (j & 1) * kTile; };

  if (warp < 8 && n > 0) {
    // ---------------- the queries' halves: warps 0-3 the first half of a row's columns, warps 4-7 the second
    const float* src = static_cast<const float*>(query_of(a, w, row < w.rows ? row : 0, 4));
    const int side = warp >> 2;
    float4 x[HALVES * 4][2];  // eight columns each
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HALVES * 4; ++i) {
      const int c = (side * HALVES * 4 + i) * 8;
      x[i][0] = x[i][1] = make_float4(0, 0, 0, 0);
      if (row < w.rows && c < a.dim) x[i][0] = *reinterpret_cast<const float4*>(src + c);
      if (row < w.rows && c + 4 < a.dim) x[i][1] = *reinterpret_cast<const float4*>(src + c + 4);
      top = max(top, max(magnitude(x[i][0]), magnitude(x[i][1])));
    }
    uint32_t* s_top = reinterpret_cast<uint32_t*>(s_sum);
    s_top[side * kTile + row] = top;
    asm volatile("bar.sync 1, 256;" ::: "memory");  // warps 0-7
    eq = exponent_for(max(top, s_top[(side ^ 1) * kTile + row]));
    const float scale = a.scale_log2 < 0.0f ? -power2(eq) : power2(eq);
#pragma unroll
    for (int k = 0; k < HALVES * 4; ++k) {
      const int i = side * HALVES * 4 + k;
      uint4 hi, lo;
      split2(x[k][0].x * scale, x[k][0].y * scale, hi.x, lo.x);
      split2(x[k][0].z * scale, x[k][0].w * scale, hi.y, lo.y);
      split2(x[k][1].x * scale, x[k][1].y * scale, hi.z, lo.z);
      split2(x[k][1].z * scale, x[k][1].w * scale, hi.w, lo.w);
      uint8_t* dst = s_q + (i >> 3) * kHalfBytes + row * 128 + (((i & 7) ^ (row & 7)) << 4);
      *reinterpret_cast<uint4*>(dst) = hi;
      *reinterpret_cast<uint4*>(dst + kTileBytes) = lo;
    }
    fence_proxy_async();
    mbar_arrive(q_full);
  }

  float m = -INFINITY, l = 0.0f;          // warps 0-3: the maximum in units of log2, and the sum
  float acc[HALVES * 64];                 // warps 4-7
  bool ok = true;
  if (warp == kLoadWarp) {
    // ---------------- K and V tiles, hi and lo
    bool alive = true;
    int issued = 0;
    for (int j = 0; j < n && alive; ++j) {
      for (int kv = 0; kv < 2 && alive; ++kv) {
        alive = warp_wait(kv ? v_empty : k_empty, (j & 1) ^ 1, abort_flag);
        if (!alive) break;
        const bool look = kv && j >= look_from;
        const uint32_t full = look ? v_landed : kv ? v_full : k_full;
        if (lane == 0) {
          mbar_expect_tx(full, 2 * HALVES * kHalfBytes);
          for (int part = 0; part < 2; ++part)
            for (int h = 0; h < HALVES; ++h)
              tma_load3(smem_u32(kv ? s_v : s_k) + part * kTileBytes + h * kHalfBytes, &tm, full, h * 64, w.k0 + j * kTile,
                        (2 * kv + part) * a.heads_kv + w.h);
        }
        __syncwarp();
        ++issued;
        if (!look) continue;
        alive = warp_wait(v_landed, (j - look_from) & 1, abort_flag);
        if (!alive) {
          drain(v_landed, (j - look_from) & 1);
          break;
        }
        bool any = false;
        for (int r = lane; r < kTile; r += 32)
          any |= replace_value_row<__half, HALVES>(smem_u32(s_v) + r * 128, false);  // lo is 0 where hi is not finite
        if (any) s_replaced = w.k0 + look_from * kTile;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full);
      }
    }
    // every issued copy must land before the CTA may exit
    if (lane == 0)
      for (int i = max(issued - 2, 0); i < issued; ++i)
        if (i % 2 == 0 || i / 2 < look_from) drain(i & 1 ? v_full : k_full, (i >> 1) & 1);
  } else if (warp == kMmaWarp) {
    // ---------------- products
    if (lane == 0 && n > 0) {
      constexpr uint32_t idesc_s = make_idesc<__half>(kTile, false), idesc_o = make_idesc<__half>(HALVES * 64, true);
      const uint64_t q_desc = make_desc(smem_u32(s_q), 16), k_desc = make_desc(smem_u32(s_k), 16),
                     v_desc = make_desc(smem_u32(s_v), kHalfBytes);
      auto scores = [&](int j) {
#pragma unroll
        for (int term = 0; term < 3; ++term) {  // lo hi, hi lo, hi hi
          const uint64_t q = advanced(q_desc, term == 0 ? kTileBytes : 0), k = advanced(k_desc, term == 1 ? kTileBytes : 0);
#pragma unroll
          for (int p = 0; p < HALVES * 4; ++p) {
            const uint32_t off = (p >> 2) * kHalfBytes + (p & 3) * 32;
            mma_ss(s_col(j), advanced(q, off), advanced(k, off), idesc_s, term > 0 || p > 0);
          }
        }
        mma_commit(s_full(j));
        mma_commit(k_empty);
      };
      bool alive = mbar_wait(q_full, 0, abort_flag) && mbar_wait(k_full, 0, abort_flag);
      if (alive) {
        tc_fence_after();
        scores(0);
      }
      for (int j = 0; j < n && alive; ++j) {
        if (j + 1 < n) {
          alive = mbar_wait(k_full, (j + 1) & 1, abort_flag);
          if (!alive) break;
          scores(j + 1);
        }
        alive = mbar_wait(v_full, j & 1, abort_flag) && mbar_wait(p_full(j), (j >> 2) & 1, abort_flag) &&
                mbar_wait(o_empty(j), ((j >> 1) & 1) ^ 1, abort_flag);
        if (!alive) break;
        tc_fence_after();
#pragma unroll
        for (int term = 0; term < 3; ++term) {
          const uint32_t p = s_col(j) + (term == 0 ? 64 : 0);
          const uint64_t v = advanced(v_desc, term == 1 ? kTileBytes : 0);
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            mma_ts(o_col(j), p + k * 8, advanced(v, k * 2048), idesc_o, term > 0 || k > 0);
        }
        mma_commit(o_full(j));
        mma_commit(v_empty);
      }
    }
  } else if (warp < 4) {
    // ---------------- softmax
    // powers of two, one after the other: their product may lie outside fp32, and infinity x 0 would be a NaN
    const float c = fminf(score_factor(a.scale_log2 * power2(-eq) * power2(-ek)), FLT_MAX);
    float ref = -INFINITY;  // the maximum as a score
    for (int j = 0; j < n; ++j) {
      ok = warp_wait(s_full(j), (j >> 1) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld(s_col(j) + lanes + i * 32, x + i * 32);
      tmem_ld_wait(x);
#pragma unroll
      for (int i = 1; i < 4; ++i) after_wait(x + i * 32);
      auto f = [&](int i) { return __uint_as_float(x[i]); };
      const int lim = min(vis, end) - (w.k0 + j * kTile);
      if (__any_sync(0xffffffffu, lim < kTile)) {
#pragma unroll
        for (int i = 0; i < kTile; ++i)
          if (i >= lim) x[i] = 0xff800000u;
      }
      float top[4] = {f(0), f(1), f(2), f(3)};
#pragma unroll
      for (int i = 4; i < kTile - 4; i += 8)
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = max3(top[k], f(i + k), f(i + k + 4));
#pragma unroll
      for (int k = 0; k < 4; ++k) top[k] = fmaxf(top[k], f(kTile - 4 + k));
      const float best = fmaxf(ref, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))), now = best * c;
      const bool none = now == -INFINITY, far = fabsf(now) >= kFar && !none;
      const float keep = ex2(far ? (ref - best) * c : m - (none ? 0.0f : now));
      ref = best, m = now;
      s_keep[(j & 3) * kTile + row] = keep;
      if (__any_sync(0xffffffffu, far)) {
        if (far) {
#pragma unroll
          for (int i = 0; i < kTile; ++i) x[i] = __float_as_uint((f(i) - ref) * c);
        }
      }
      const float by = far ? 1.0f : c, base = (far || none ? 0.0f : m) - kShift32;
      float sum[2] = {};
      // 32 keys at a time: hi over the first 64 columns of S, lo over the others (all of S is in registers)
#pragma unroll
      for (int i = 0; i < kTile; i += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float p0 = ex2(fmaf(f(i + k), by, -base)), p1 = ex2(fmaf(f(i + k + 1), by, -base));
          sum[0] += p0;
          sum[1] += p1;
          split2(p0, p1, hi[k >> 1], lo[k >> 1]);
        }
        tmem_st16(s_col(j) + lanes + i / 2, hi);
        tmem_st16(s_col(j) + lanes + 64 + i / 2, lo);
      }
      l = l * keep + (sum[0] + sum[1]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full(j));
    }
    s_sum[row] = l;  // the magnitudes there were read before the first S
  } else {
    // ---------------- the sum of O
#pragma unroll
    for (int i = 0; i < HALVES * 64; ++i) acc[i] = 0.0f;
    for (int j = 0; j < n; ++j) {
      ok = warp_wait(p_full(j), (j >> 2) & 1, abort_flag) && warp_wait(o_full(j), (j >> 1) & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const float keep = s_keep[(j & 3) * kTile + row];
#pragma unroll
      for (int i = 0; i < HALVES * 64; i += 32) {
        uint32_t y[32];
        tmem_ld(o_col(j) + lanes + i, y);
        tmem_ld_wait(y);
#pragma unroll
        for (int k = 0; k < 32; ++k) acc[i + k] = fmaf(acc[i + k], keep, __uint_as_float(y[k]));
      }
      tc_fence_before();
      mbar_arrive(o_empty(j));
    }
  }
  __syncthreads();  // every product is done, the sums are there
  if (warp < 4) {
    const bool none = l == 0.0f || n == 0;
    if (row < w.rows) {
      const int64_t at = row_index(a, w, row);
      const float lse = none ? -INFINITY : ((m == -INFINITY ? 0.0f : m) - kShift32) * kLn2 + logf(l);
      (a.part_o ? a.part_lse[at * a.splits + w.split] : a.lse[at]) = lse;
    }
  } else if (warp < 8) {
    // out through shared memory (the queries' room), 32 columns at a time, in whole pieces of rows
    const float sum = s_sum[row];
    const bool none = sum == 0.0f || n == 0;
    const float inv = none ? 0.0f : 1.0f / sum, back = power2(-ev);
    const int64_t at = row < w.rows ? row_index(a, w, row) : 0;
    const int64_t n_rows = (int64_t)a.batch * a.queries * a.heads_q;
    float* buf = reinterpret_cast<float*>(s_q) + (warp & 3) * 32 * 36;
    const int row0 = (warp & 3) * 32;
#pragma unroll
    for (int i = 0; i < HALVES * 64; i += 32) {
      if (i >= a.dim || !ok) break;
#pragma unroll
      for (int k = 0; k < 32; k += 4) {
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = none ? 0.0f : acc[i + k + e] * inv * back;
        *reinterpret_cast<float4*>(buf + lane * 36 + k) = make_float4(z[0], z[1], z[2], z[3]);
      }
      __syncwarp();
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const int q = p * 4 + (lane >> 3), col = i + (lane & 7) * 4;
        const float4 z = *reinterpret_cast<const float4*>(buf + q * 36 + (lane & 7) * 4);
        const int64_t at_row = __shfl_sync(0xffffffffu, at, q);
        if (row0 + q >= w.rows || col >= a.dim) continue;
        float* y = a.part_o ? a.part_o + ((int64_t)w.split * n_rows + at_row) * a.dim : static_cast<float*>(a.out) + at_row * a.dim;
        *reinterpret_cast<float4*>(y + col) = z;
      }
      __syncwarp();
    }
    mbar_arrive(written);
  } else if (warp == kLoadWarp && s_replaced != kNoKey && warp_wait(written, 0, abort_flag)) {
    for (int r = lane; r < w.rows; r += 32) write_nonfinite_row<float>(a, w, r, s_replaced);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int64_t padded_keys(int64_t keys) { return ceil_div(keys, kTile) * kTile; }

template <int HALVES>
int launch_as(const SplitArgs& s, cudaStream_t stream) {
  EncodeFn enc = encode_fn();
  KB_REQUIRE(enc != nullptr, KB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  CUtensorMap tm;
  cuuint64_t dims[3] = {(cuuint64_t)s.cols, (cuuint64_t)s.keys, (cuuint64_t)4 * s.a.heads_kv};
  cuuint64_t strides[2] = {(cuuint64_t)s.cols * 2, (cuuint64_t)s.cols * s.keys * 2};
  cuuint32_t box[3] = {64, kTile, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(&tm, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, s.halves, dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  KB_REQUIRE(r == CUDA_SUCCESS, KB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  static uint64_t attr_set = 0;  // one bit per device ordinal
  int dev = 0;
  KB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(attr_set >> dev & 1)) {
    KB_CUDA(cudaFuncSetAttribute(attn_prefix32_kernel<HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    if (dev < 64) attr_set |= 1ull << dev;
  }
  KB_CUDA(cudaMemsetAsync(s.largest, 0, 2 * s.a.heads_kv * sizeof(uint32_t), stream));
  const int64_t heads = s.a.heads_kv;
  const dim3 blocks((unsigned)std::min<int64_t>(ceil_div((int64_t)s.keys * s.cols / 4, 256),
                                                std::max<int64_t>(1, sm_count() * 8 / heads)),
                    (unsigned)heads);
  largest_kernel<<<blocks, 256, 0, stream>>>(s);
  if (int st = check_launch("kb_shared_prefix_attention")) return st;
  if (int st = launch_after(halves_kernel, blocks, 256u, 0, stream, s)) return st;
  return launch_after(attn_prefix32_kernel<HALVES>, dim3((unsigned)s.a.prefix_items), (unsigned)kThreads, kSmemBytes,
                      stream, tm, s);
}

}  // namespace

// Where the split pays, by the operations: against the kernel of mma.sync it
// took 74 against 65 us at 1.07e9 (256 rows x 8 heads x 1024 keys x 128), 66
// against 87 at 2.1e9, 162 against 267 at 8.6e9, 245 against 494 at 17e9 and 952
// against 3394 at 131e9 (calls with short continuations).  With magnitudes by row
// and head it takes 64, 136 and 191 us at the three in the middle, 739 at 137e9.
bool tc32_pays(int64_t rows, int64_t heads_kv, int64_t dim, int64_t keys) {
  return dim <= kTile && heads_kv <= 65535 && rows > 64 && keys > 0 && 4.0 * rows * heads_kv * dim * keys >= 1.2e9;
}
static size_t largest_bytes(int64_t heads_kv) { return (size_t)ceil_div(2 * heads_kv, 4) * 16; }
size_t tc32_bytes(int64_t heads_kv, int64_t dim, int64_t keys) {
  return largest_bytes(heads_kv) + (size_t)4 * heads_kv * padded_keys(keys) * (dim > 64 ? 128 : 64) * sizeof(__half);
}
int tc32_launch(const AttnArgs& a, void* scratch, cudaStream_t stream) {
  SplitArgs s{a, static_cast<uint32_t*>(scratch),
              reinterpret_cast<__half*>(static_cast<char*>(scratch) + largest_bytes(a.heads_kv)),
              (int)padded_keys((int64_t)a.prefix_pages * a.page_size), a.dim > 64 ? 128 : 64};
  return a.dim > 64 ? launch_as<2>(s, stream) : launch_as<1>(s, stream);
}
int tc32_read_fault(bool clear, int* value) { return read_fault(clear, value); }

}  // namespace attn
}  // namespace lm
}  // namespace kb
