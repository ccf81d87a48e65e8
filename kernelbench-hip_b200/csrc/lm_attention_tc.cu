// lm_attention_tc.cu — the shared prefix on the fifth-generation tensor cores:
// all query rows of one key head against the prefix's keys and values, in
// fp16 or bf16.
//
// A CTA takes up to two tiles of 128 query rows and a range of keys, in tiles
// of 128.  Per key tile j and row tile t:
//   S_t = Q_t K_j^T            tcgen05.mma, 128 x 128, accumulators in TMEM
//   P_t = exp2(S_t c - m)      one thread per row (tcgen05.ld), rounded to the
//                              values' 16 bits into TMEM over S_t (tcgen05.st):
//                              a product has operands of one type, and two
//                              halves of P would take two products.  Each
//                              weight is off by half a unit, out by that much
//                              of softmax |v|: bf16 0.0022 against 0.0017 of
//                              an output that is only rounded once
//   O_t += P_t V_j             tcgen05.mma with P from TMEM, O in TMEM
// c = scale log2(e).  m is a row's reference, not its exact maximum: it only
// moves when the maximum has grown past it by more than 2^kSlack, and then the
// row's O is scaled in TMEM (rare after the first tiles); l and O carry the
// same m, so it cancels in O / l.  l sums the unrounded exponentials in fp32.
// (kSlack 4 scaled some row of nearly every warp in the first ten key tiles of
// scores of deviation 2, a thousand cycles each; 8 scales almost none.)
//
// Roles (10 warps): warps 0-3 and 4-7 are the softmax of the two row tiles,
// warp 8 loads K and V tiles by TMA, one copy per page and 64 columns (the
// page table is the gather), and looks at those values that not all rows see
// (infinities and NaN among them: lm_attention.cuh), warp 9 issues the products in the order
//   O_0 += P_0 V_j, S_0 = Q_0 K_j+1, O_1 += P_1 V_j, S_1 = Q_1 K_j+1
// so that one row tile's products run during the other's softmax; O += P V
// begins with the first 64 keys while the others' exponentials are computed.
// The products of a thread are executed in order, so S_t(j + 1) may overwrite
// the P_t(j) that the product before it reads.
//
// TMEM (512 columns): S_0, S_1 (P_t in the first 64 columns of S_t), O_0, O_1.
// Shared memory: Q 64 KB, two stages of K and of V, 32 KB each, all in rows of
// 128 bytes with the 128-byte swizzle: K-major for Q and K, MN-major for V.
// Columns past the head size are zeros (TMA fills them), and so are V rows
// past the last key that any row of the CTA sees.
//
// Bound: 4 rows keys dim operations on the tensor cores, and as many cycles
// again of exponentials (16 per clock and SM against 128 x 128 x 128 products
// in 512 cycles), which overlap.  What it measured, by clocks read in a copy of
// this kernel: per key tile and row tile a softmax takes 2400 cycles (85 for the
// load, 320 for the maximum, 1800 for the exponentials, 170 for the store), O 520,
// S 820 (both operands from shared memory: 8 KB per 64 cycles of product), and
// this chain, not a unit, sets the pace.  256 samples x 32 heads x 128 over 32768
// keys, bf16: 0.167 ms from a cold cache, 820 TFLOP/s, half of a large library
// product's 1650.  Tried and slower: steps
// of 64 keys with two buffers for S (a product of 128 x 64 takes as long as one
// of 128 x 128), two threads per row (spills at 96 registers).
//
// Every wait is bounded: one that runs out raises the CTA's abort flag and the
// device's fault word, every role leaves, copies in flight are waited for
// (bounded), TMEM is freed; outputs are then invalid.
#include "lm_attention.cuh"
#include "lm_tc.cuh"

namespace kb {
namespace lm {
namespace attn {

namespace {

constexpr int kStages = 2;
constexpr int kThreads = 320;
constexpr int kLoadWarp = 8, kMmaWarp = 9;
constexpr int kSmemBytes = (2 + 2 * kStages) * kTileBytes + 256 + 1024;  // + barriers, alignment
constexpr float kSlack = 8.0f;                  // log2 of how far a maximum may pass the reference

template <typename T, int HALVES>
__global__ void __launch_bounds__(kThreads, 1)
attn_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                   const __grid_constant__ AttnArgs a, int row_tiles) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_k = smem + 2 * kTileBytes;
  uint8_t* s_v = s_k + kStages * kTileBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_v + kStages * kTileBytes);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const uint32_t q_full = bar(0);  // [2]
  auto k_full = [&](int s) { return bar(2 + s); };
  auto k_empty = [&](int s) { return bar(4 + s); };
  auto v_full = [&](int s) { return bar(6 + s); };
  auto v_empty = [&](int s) { return bar(8 + s); };
  auto s_full = [&](int t) { return bar(10 + t); };
  auto p_full = [&](int t, int half) { return bar(12 + 2 * t + half); };
  auto o_full = [&](int t) { return bar(16 + t); };
  const uint32_t v_landed = bar(18);  // a copy of values that are looked at before v_full
  const uint32_t written = bar(19);   // the rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_end = reinterpret_cast<int*>(tmem_slot + 2);
  int* s_least = s_end + 1;
  __shared__ int s_replaced;
  // first of all, so that no CTA holds TMEM while a launch before it has to take its own
  wait_for_previous();

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Item w = item_at(a, blockIdx.x, row_tiles * kTile);
  const int cols = row_tiles == 2 ? 512 : 256;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(q_full + 8 * t, kTile);
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t, 0), kTile);
      mbar_init(p_full(t, 1), kTile);
      mbar_init(o_full(t), 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    mbar_init(v_landed, 1);
    mbar_init(written, row_tiles * kTile);
    *abort_flag = 0;
    *s_end = 0;
    *s_least = 0x7fffffff;
    s_replaced = kNoKey;
    fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), cols);
    tmem_relinquish();
  }
  __syncthreads();
  allow_next();  // the sequences' own keys are read without a wait, and TMEM is taken
  // the keys that any row of this CTA sees
  const int t = warp >> 2, row = threadIdx.x & (kTile - 1);  // softmax warps: row tile, row in it
  const int r = t * kTile + row;
  int vis = 0;
  if (warp < 4 * row_tiles) {
    if (r < w.rows) vis = visible(a, w.base + (w.row0 + r) / a.group);
    const int top = __reduce_max_sync(0xffffffffu, vis), low = __reduce_min_sync(0xffffffffu, vis > w.k0 ? vis : 0x7fffffff);
    if (lane == 0) atomicMax(s_end, top), atomicMin(s_least, low);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int end = min(w.k1, *s_end), least = *s_least;
  const int n = end > w.k0 ? (end - w.k0 + kTile - 1) / kTile : 0;
  // The first tile with values that warp 8 looks at before they are used: some that only some rows see, or that none
  // does, in a page that is partly seen (they become zeros, for 0 x NaN).
  const int part_of_page = end < w.k0 + n * kTile && end % a.page_size != 0 ? n - 1 : n;
  const int look_from = min(part_of_page, least < end ? (uneven_from(w, least, kTile) - w.k0) / kTile : n);
  constexpr int halves = HALVES;  // of 64 columns; columns past dim are zeros
  const uint32_t o_col = row_tiles == 2 ? 256 : 128;

  if (warp == kLoadWarp) {
    // ---------------- K and V tiles: lane i copies page i of the tile
    const int slots = min(a.page_size, kTile), per_tile = kTile / slots;
    bool alive = true;
    int issued = 0;
    for (int j = 0; j < n && alive; ++j) {
      const int key0 = w.k0 + j * kTile, s = j % kStages;
      // past the prefix, or past what anyone sees: a page that is not there reads as zeros
      int page = a.pages, slot = 0;
      const int key = key0 + lane * slots;
      if (lane < per_tile && key < end) {
        page = min(max(w.pages[key / a.page_size], 0), a.pages - 1);
        slot = key % a.page_size;
      }
      const uint32_t parity = ((j / kStages) & 1) ^ 1;
      for (int kv = 0; kv < 2 && alive; ++kv) {
        const bool look = kv && j >= look_from;
        const uint32_t full = look ? v_landed : kv ? v_full(s) : k_full(s);
        if (!warp_wait(kv ? v_empty(s) : k_empty(s), parity, abort_flag)) {
          alive = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(full, halves * kHalfBytes);
        __syncwarp();
        if (lane < per_tile) {
          const uint32_t dst = smem_u32((kv ? s_v : s_k) + s * kTileBytes + lane * slots * 128);
          for (int h = 0; h < halves; ++h)
            tma_load(dst + h * kHalfBytes, kv ? &tm_v : &tm_k, full, h * 64, w.h, slot, page);
        }
        ++issued;
        if (!look) continue;
        alive = warp_wait(v_landed, (j - look_from) & 1, abort_flag);
        if (!alive) {
          drain(v_landed, (j - look_from) & 1);
          break;
        }
        bool any = false;
        for (int row = lane; row < kTile; row += 32)
          any |= replace_value_row<T, HALVES>(smem_u32(s_v) + s * kTileBytes + row * 128, key0 + row >= end);
        if (any) s_replaced = w.k0 + look_from * kTile;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full(s));
      }
    }
    // every issued copy must land before the CTA may exit
    if (lane == 0)
      for (int i = max(issued - 2 * kStages, 0); i < issued; ++i) {
        const int j = i / 2, s = j % kStages;
        if (i % 2 == 0 || j < look_from) drain(i & 1 ? v_full(s) : k_full(s), (j / kStages) & 1);
      }
    if (alive && s_replaced != kNoKey && warp_wait(written, 0, abort_flag))
      for (int i = lane; i < w.rows; i += 32) write_nonfinite_row<T>(a, w, i, s_replaced);
  } else if (warp == kMmaWarp) {
    // ---------------- products
    if (lane == 0 && n > 0) {
      constexpr int kDepth = HALVES * 4;
      constexpr uint32_t idesc_s = make_idesc<T>(kTile, false), idesc_o = make_idesc<T>(HALVES * 64, true);
      const uint64_t q_desc = make_desc(smem_u32(s_q), 16), k_desc = make_desc(smem_u32(s_k), 16),
                     v_desc = make_desc(smem_u32(s_v), kHalfBytes);
      auto scores = [&](int i, int s) {
        const uint64_t q = advanced(q_desc, i * kTileBytes), kd = advanced(k_desc, s * kTileBytes);
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
          const uint32_t off = (k >> 2) * kHalfBytes + (k & 3) * 32;
          mma_ss(tmem + i * kTile, advanced(q, off), advanced(kd, off), idesc_s, k > 0);
        }
        mma_commit(s_full(i));
      };
      bool alive = mbar_wait(k_full(0), 0, abort_flag);
      for (int i = 0; i < row_tiles && alive; ++i) {
        alive = mbar_wait(q_full + 8 * i, 0, abort_flag);
        if (!alive) break;
        tc_fence_after();
        scores(i, 0);
      }
      if (alive) mma_commit(k_empty(0));
      for (int j = 0; j < n && alive; ++j) {
        const int s = j % kStages, next = (j + 1) % kStages;
        const uint32_t parity = (j / kStages) & 1, next_parity = ((j + 1) / kStages) & 1;
        for (int i = 0; i < row_tiles && alive; ++i) {
          alive = i > 0 || mbar_wait(v_full(s), parity, abort_flag);
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // each half of P as soon as it is there
            alive = alive && mbar_wait(p_full(i, half), j & 1, abort_flag);
            if (!alive) break;
            tc_fence_after();
#pragma unroll
            for (int k = half * 4; k < half * 4 + 4; ++k)
              mma_ts(tmem + o_col + i * kTile, tmem + i * kTile + k * 8,
                     advanced(v_desc, s * kTileBytes + k * 2048), idesc_o, j > 0 || k > 0);
          }
          if (!alive) break;
          mma_commit(o_full(i));
          if (i == row_tiles - 1) mma_commit(v_empty(s));
          if (j + 1 < n) {
            alive = i > 0 || mbar_wait(k_full(next), next_parity, abort_flag);
            if (!alive) break;
            scores(i, next);
            if (i == row_tiles - 1) mma_commit(k_empty(next));
          }
        }
      }
    }
  } else if (t < row_tiles) {
    // ---------------- softmax: this thread's row
    const uint32_t lanes = (uint32_t)(warp & 3) * 32 << 16;
    const uint32_t s_addr = tmem + lanes + t * kTile, o_addr = tmem + lanes + o_col + t * kTile;
    const float c = score_factor(a.scale_log2);
    if (n > 0) {
      // the row of Q into the swizzled tile, all copies in flight at once
      const char* src = static_cast<const char*>(query_of(a, w, r < w.rows ? r : 0, 2));
      const uint32_t dst = smem_u32(s_q + t * kTileBytes + row * 128);
      auto at = [&](int i) { return dst + (i >> 3) * kHalfBytes + (((i & 7) ^ (row & 7)) << 4); };
#pragma unroll
      for (int i = 0; i < halves * 8; ++i) {
        const bool in = r < w.rows && i * 8 < a.dim;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at(i)), "l"(src + (in ? i * 16 : 0)),
                     "r"(in ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (a.scale_log2 < 0.0f) {  // scores are multiplied by |c|
        for (int i = 0; i < halves * 8; ++i) {
          uint32_t x[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                       : "r"(at(i)));
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at(i)), "r"(x[0] ^ 0x80008000u),
                       "r"(x[1] ^ 0x80008000u), "r"(x[2] ^ 0x80008000u), "r"(x[3] ^ 0x80008000u)
                       : "memory");
        }
      }
      fence_proxy_async();
      mbar_arrive(q_full + 8 * t);
    }
    float ref = -INFINITY, m = -INFINITY, l = 0.0f;  // the reference, as a score and in units of log2, and the sum
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = warp_wait(s_full(t), j & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t x[kTile];
#pragma unroll
      for (int i = 0; i < 4; ++i) tmem_ld(s_addr + i * 32, x + i * 32);
      tmem_ld_wait(x);
#pragma unroll
      for (int i = 1; i < 4; ++i) after_wait(x + i * 32);
      auto f = [&](int i) { return __uint_as_float(x[i]); };
      const int lim = min(vis, end) - (w.k0 + j * kTile);  // keys of this tile that the row sees
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
      const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), now = best * c;
      // move the reference where the maximum has outgrown it
      const bool move = now > m + kSlack;  // also from -inf; not for a NaN
      if (__any_sync(0xffffffffu, move)) {
        const float by = fmaxf(fabsf(m), fabsf(now)) < kFar ? m - now : (ref - best) * c;  // also from -inf
        const float keep = move ? ex2(by) : 1.0f;
        if (move) ref = best, m = now;
        l *= keep;
        if (j > 0) {
          ok = warp_wait(o_full(t), (j - 1) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int i = 0; i < a.dim; i += 32) {
            uint32_t y[32];
            tmem_ld(o_addr + i, y);
            tmem_ld_wait(y);
#pragma unroll
            for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * keep);
            tmem_st(o_addr + i, y);
          }
          tmem_st_wait();
        }
      }
      const bool far = fabsf(m) >= kFar && m != -INFINITY;
      if (__any_sync(0xffffffffu, far)) {
        if (far) {
#pragma unroll
          for (int i = 0; i < kTile; ++i) x[i] = __float_as_uint((f(i) - ref) * c);
        }
      }
      const float by = far ? 1.0f : c, base = (far || m == -INFINITY ? 0.0f : m) - kShift<T>;
      const uint64_t cc = pair(by, by), bb = pair(-base, -base);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = half * kTile / 2; i < (half + 1) * kTile / 2; i += 2) {
          float p0, p1;
          unpair(fma2(pair(f(i), f(i + 1)), cc, bb), p0, p1);
          p0 = ex2(p0);
          p1 = ex2(p1);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pair(p0, p1));
          x[i >> 1] = pack(p0, p1, (T*)nullptr);
        }
        tmem_st(s_addr + half * 32, x + half * 32);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full(t, half));
      }
      float l0, l1;
      unpair(add2(sum[0], sum[1]), l0, l1);
      l += l0 + l1;
    }
    if (ok && n > 0) ok = warp_wait(o_full(t), (n - 1) & 1, abort_flag);
    tc_fence_after();
    const bool none = l == 0.0f || n == 0;
    const int64_t at = r < w.rows ? row_index(a, w, r) : 0;
    const float base = m - kShift<T>, inv = none ? 0.0f : 1.0f / l;
    const float lse = none ? -INFINITY : (m == -INFINITY ? 0.0f : base) * kLn2 + logf(l);
    if (r < w.rows) (a.part_o ? a.part_lse[at * a.splits + w.split] : a.lse[at]) = lse;
    if (ok) {
      // Out through shared memory, 32 columns at a time, so that a warp writes
      // whole 128-byte pieces of rows (a thread's own row straight from its
      // registers took 5 us per CTA).  The row tile's Q, whose last product is
      // done, makes room: one buffer per warp, rows 144 bytes apart.
      const int64_t n_rows = (int64_t)a.batch * a.queries * a.heads_q;
      float* buf = reinterpret_cast<float*>(s_q + t * kTileBytes) + (warp & 3) * 32 * 36;
      const int row0 = t * kTile + (warp & 3) * 32;  // the warp's rows
#pragma unroll 1
      for (int i = 0; i < a.dim; i += 32) {
        uint32_t y[32];
        if (n > 0) {
          tmem_ld(o_addr + i, y);
          tmem_ld_wait(y);
        }
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          float z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) z[e] = none ? 0.0f : __uint_as_float(y[k + e]) * inv;
          *reinterpret_cast<float4*>(buf + lane * 36 + k) = make_float4(z[0], z[1], z[2], z[3]);
        }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const int q = p * 4 + (lane >> 3), col = i + (lane & 7) * 4;
          const float4 z = *reinterpret_cast<const float4*>(buf + q * 36 + (lane & 7) * 4);
          const int64_t at_row = __shfl_sync(0xffffffffu, at, q);
          if (row0 + q >= w.rows || col >= a.dim) continue;
          if (a.part_o) {  // a part without keys is not read: its zeros do no harm
            *reinterpret_cast<float4*>(a.part_o + ((int64_t)w.split * n_rows + at_row) * a.dim + col) = z;
          } else {
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at_row * a.dim + col) =
                make_uint2(pack(z.x, z.y, (T*)nullptr), pack(z.z, z.w, (T*)nullptr));
          }
        }
        __syncwarp();
      }
    }
    mbar_arrive(written);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ------------------------------------------------------------------ host side
// Pool of pages as {column, head, slot, page}; a box is one head's 64 columns
// of a page's slots (at most 128), in 128-byte rows with the 128-byte swizzle.
int make_map(CUtensorMap* tm, const void* base, const AttnArgs& a, int dtype, int64_t page, int64_t slot, int64_t head) {
  EncodeFn enc = encode_fn();
  KB_REQUIRE(enc != nullptr, KB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.heads_kv, (cuuint64_t)a.page_size, (cuuint64_t)a.pages};
  cuuint64_t strides[3] = {(cuuint64_t)head * 2, (cuuint64_t)slot * 2, (cuuint64_t)page * 2};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)std::min(a.page_size, kTile), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(tm, dtype == KB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  KB_REQUIRE(r == CUDA_SUCCESS, KB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return KB_OK;
}

template <typename T, int HALVES>
int launch_as(const AttnArgs& a, int dtype, int row_tiles, cudaStream_t stream) {
  CUtensorMap tk, tv;
  if (int st = make_map(&tk, a.k, a, dtype, a.k_p, a.k_s, a.k_h)) return st;
  if (int st = make_map(&tv, a.v, a, dtype, a.v_p, a.v_s, a.v_h)) return st;
  static uint64_t attr_set = 0;  // one bit per device ordinal
  int dev = 0;
  KB_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(attr_set >> dev & 1)) {
    KB_CUDA(cudaFuncSetAttribute(attn_prefix_kernel<T, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    if (dev < 64) attr_set |= 1ull << dev;
  }
  return launch_after(attn_prefix_kernel<T, HALVES>, dim3((unsigned)a.prefix_items), (unsigned)kThreads, kSmemBytes,
                      stream, tk, tv, a, row_tiles);
}

}  // namespace

int tc_tile_rows(int64_t rows) { return rows <= kTile ? kTile : 2 * kTile; }

bool tc_fits(const AttnArgs& a, int dtype) {
  // a page is a whole part of a 128-key tile, of at least one swizzle group, or whole tiles
  const bool pages = (kTile % a.page_size == 0 && a.page_size >= 8) || a.page_size % kTile == 0;
  auto stride = [](int64_t s) { return s > 0 && s * 2 < ((int64_t)1 << 40); };
  return dtype != KB_F32 && a.dim <= kTile && a.prefix_pages > 0 && pages && stride(a.k_p) && stride(a.k_s) &&
         stride(a.k_h) && stride(a.v_p) && stride(a.v_s) && stride(a.v_h);
}

int tc_launch(const AttnArgs& a, int dtype, cudaStream_t stream) {
  const int row_tiles = tc_tile_rows((int64_t)a.batch * a.queries * a.group) / kTile;
  if (a.dim <= 64)
    return dtype == KB_F16 ? launch_as<__half, 1>(a, dtype, row_tiles, stream)
                           : launch_as<__nv_bfloat16, 1>(a, dtype, row_tiles, stream);
  return dtype == KB_F16 ? launch_as<__half, 2>(a, dtype, row_tiles, stream)
                         : launch_as<__nv_bfloat16, 2>(a, dtype, row_tiles, stream);
}

int tc_read_fault(bool clear, int* value) { return read_fault(clear, value); }

}  // namespace attn
}  // namespace lm
}  // namespace kb
