// lm_rope.cu — RMS norm of every query and key head with the position
// rotation in the same pass, and its backward pass.
//
//   y = x r w,   r = 1 / sqrt(mean(x^2) + eps)       (one head vector of `dim`)
//   z = Rot(y):  for each pair (a, b) of the first `rotary` elements, with
//                c, s from row `position` of the tables,
//                z_a = a c - b s,  z_b = b c + a s;  the rest is unchanged
// Pairs are (i, i + rotary / 2), or (2 i, 2 i + 1) when interleaved.
//
// Backward, from dz: dy = Rot^T(dz) (the rotation by the opposite angle),
//   xh = x r,  dw = sum over heads and tokens of dy xh,
//   dx = r (dy w - xh mean(dy w xh)).
// r is computed again from x (one multiply-add per element) instead of being
// kept from the forward pass.
//
// Statistics and products are fp32; outputs are rounded once.  dw is summed
// in fp64 over warps and CTAs in a fixed order, so it does not depend on
// timing.  A position outside the table gives NaN in the rotated elements.
//
// Both passes are bound by HBM (2 and 3 times the heads' bytes), so the work
// is laid out to need no second look at an element and few shuffles: L lanes
// hold one head vector, each lane four pairs (a, b), both elements of a pair
// in the same lane.  With the half-split pairs that is four elements of the
// first half and the four that they turn with, two 8-byte (16-bit types) or
// 16-byte loads; interleaved, eight elements in a row.  The norm's sum is
// log2(L) shuffles, the rotation none.  A warp takes kBatch x 32 / L heads of
// one token, all loads issued before the first use, so cos and sin are read
// once per token and warp.  16384 tokens x 40 heads x 128, bf16, on a B200:
// forward 67 us (5.0 TB/s of the 6.6 that a plain copy reaches), backward with
// both weights' gradients 108 us (4.7 TB/s), where instruction issue is next.
#include "lm_common.cuh"

namespace kb {
namespace lm {
namespace {

constexpr int kMaxDim = 512;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;

struct RopeArgs {
  const void* x[2];   // q, k: [tokens, heads, dim], strides below, dim contiguous
  const void* dz[2];  // backward: gradients of the outputs, contiguous
  const void* w[2];   // [dim] or null
  void* out[2];       // forward: z; backward: dx; contiguous
  const float* cos_t;  // [table_rows, rotary / 2]
  const float* sin_t;
  const void* pos;
  int64_t tokens, table_rows;
  int64_t stride_t[2], stride_h[2];
  int heads[2];
  int dim, rotary, interleaved, pos64, weight32, table_vec;
  float eps, inv_dim;
  int unit_heads;
  uint32_t units_q, units_token;  // units of the queries, and in all, of one token
  double* partial;  // backward: [grid][2][dim]
};

__device__ __forceinline__ int64_t position(const RopeArgs& a, int64_t t) {
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
}

// The pair that element e < rotary belongs to, its partner, and whether e is
// the pair's first element.
__device__ __forceinline__ void pair_of(int e, int rotary, int interleaved, int& i, int& partner, bool& first) {
  const int half = rotary >> 1;
  if (interleaved) {
    i = e >> 1;
    first = (e & 1) == 0;
    partner = e ^ 1;
  } else {
    first = e < half;
    i = first ? e : e - half;
    partner = first ? e + half : e - half;
  }
}

template <typename W>
__device__ __forceinline__ float weight_at(const void* w, int e) {
  return w ? to_f32(static_cast<const W*>(w)[e]) : 1.0f;
}

constexpr int kVecDim = 256;   // heads up to here stay in registers
constexpr int kVecThreads = 128, kVecWarps = kVecThreads / 32;
constexpr int64_t kMaxUnits = 1ll << 31;
constexpr int kFlush = 128;    // terms of a sum for dw in fp32 before it moves to fp64

// Four elements as they lie in memory, 8 or 16 bytes.
template <typename T>
struct Raw4 {
  uint2 v;
  __device__ void set(int i, T x) { reinterpret_cast<T*>(&v)[i] = x; }
};
template <>
struct Raw4<float> {
  float4 v;
  __device__ void set(int i, float x) { reinterpret_cast<float*>(&v)[i] = x; }
};
__device__ __forceinline__ void unpack(const Raw4<float>& r, float (&x)[4]) {
  x[0] = r.v.x, x[1] = r.v.y, x[2] = r.v.z, x[3] = r.v.w;
}
__device__ __forceinline__ void unpack(const Raw4<__half>& r, float (&x)[4]) {
  const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&r.v.x));
  const float2 hi = __half22float2(*reinterpret_cast<const __half2*>(&r.v.y));
  x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
}
__device__ __forceinline__ void unpack(const Raw4<__nv_bfloat16>& r, float (&x)[4]) {
  x[0] = __uint_as_float(r.v.x << 16), x[1] = __uint_as_float(r.v.x & 0xffff0000u);
  x[2] = __uint_as_float(r.v.y << 16), x[3] = __uint_as_float(r.v.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__half* p, const float (&v)[4]) {
  const __half2 lo = __floats2half2_rn(v[0], v[1]), hi = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
// A lane's part of a head vector, unconverted (loads in flight hold few registers).
template <typename T>
struct Raw8 {
  Raw4<T> a, b;
};

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// How a lane's pairs lie in memory: two vectors of four whose elements turn
// with each other; eight elements in a row, each turning with its neighbour;
// or element by element, for any size and alignment.
enum Layout { kHalves, kNeighbours, kAny };

// The four pairs of lane `l` of a head vector: pair p = 4 l + j turns when
// p < rotary / 2.
template <int LAYOUT>
struct Pairs {
  int first, half, dim, off_a, off_b, interleaved;
  bool on;  // this lane holds elements of the head
  __device__ Pairs(const RopeArgs& a, int l) {
    first = 4 * l;
    half = a.rotary >> 1;
    dim = a.dim;
    interleaved = a.interleaved;
    on = 8 * l < dim;
    off_a = LAYOUT == kNeighbours ? 8 * l : first < half ? first : a.rotary + 2 * (first - half);
    off_b = LAYOUT == kNeighbours ? 8 * l + 4 : first < half ? first + half : off_a + 4;
  }
  // the elements of pair p; b is dim or more where there is none
  __device__ int ea(int p) const { return interleaved ? 2 * p : p < half ? p : 2 * p; }
  __device__ int eb(int p) const { return interleaved ? 2 * p + 1 : p < half ? p + half : 2 * p + 1; }
  __device__ bool turns(int j) const {  // with kHalves a lane turns all its pairs or none
    return LAYOUT == kHalves ? first < half : first + j < half;
  }
  template <typename T>
  __device__ void fetch(const T* x, Raw8<T>& r) const {
    if (LAYOUT != kAny) {
      r.a = *reinterpret_cast<const Raw4<T>*>(x + off_a);
      r.b = *reinterpret_cast<const Raw4<T>*>(x + off_b);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = ea(first + j), k = eb(first + j);
        r.a.set(j, i < dim ? x[i] : from_f32<T>(0.0f));
        r.b.set(j, k < dim ? x[k] : from_f32<T>(0.0f));
      }
    }
  }
  template <typename T>
  __device__ void get(const Raw8<T>& r, float (&a)[4], float (&b)[4]) const {
    unpack(r.a, a);
    unpack(r.b, b);
    if (LAYOUT == kNeighbours) {
      const float t0 = a[1], t1 = a[3];
      a[1] = a[2], a[2] = b[0], a[3] = b[2];
      b[0] = t0, b[2] = b[1], b[1] = t1;
    }
  }
  // the same in pairs of fp32: (a0, a1), (a2, a3)
  template <typename T>
  __device__ void get(const Raw8<T>& r, uint64_t (&a)[2], uint64_t (&b)[2]) const {
    float x[4], y[4];
    get(r, x, y);
    a[0] = pair(x[0], x[1]), a[1] = pair(x[2], x[3]), b[0] = pair(y[0], y[1]), b[1] = pair(y[2], y[3]);
  }
  template <typename T>
  __device__ void store(T* x, const uint64_t (&a)[2], const uint64_t (&b)[2]) const {
    float u[4], v[4];
    unpair(a[0], u[0], u[1]), unpair(a[1], u[2], u[3]), unpair(b[0], v[0], v[1]), unpair(b[1], v[2], v[3]);
    store(x, u, v);
  }
  // (u, v) = (a uc + b us, b vc + a vs); a pair that does not turn takes no product with its partner, which may
  // be infinite
  __device__ void turned(const uint64_t (&a)[2], const uint64_t (&b)[2], const uint64_t (&uc)[2], const uint64_t (&us)[2],
                         const uint64_t (&vc)[2], const uint64_t (&vs)[2], uint64_t (&u)[2], uint64_t (&v)[2]) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) u[i] = mul2(a[i], uc[i]), v[i] = mul2(b[i], vc[i]);
    if (turns(3)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) u[i] = fma2(b[i], us[i], u[i]), v[i] = fma2(a[i], vs[i], v[i]);
    } else if (turns(0)) {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        if (!turns(j)) continue;
        float x[2], y[2], p[2], q[2], s[2], t[2];
        unpair(u[j >> 1], x[0], x[1]), unpair(v[j >> 1], y[0], y[1]);
        unpair(a[j >> 1], p[0], p[1]), unpair(b[j >> 1], q[0], q[1]);
        unpair(us[j >> 1], s[0], s[1]), unpair(vs[j >> 1], t[0], t[1]);
        x[j & 1] += q[j & 1] * s[j & 1];
        y[j & 1] += p[j & 1] * t[j & 1];
        u[j >> 1] = pair(x[0], x[1]), v[j >> 1] = pair(y[0], y[1]);
      }
    }
  }
  template <typename T>
  __device__ void store(T* x, float (&a)[4], float (&b)[4]) const {
    if (LAYOUT == kNeighbours) {
      const float lo[4] = {a[0], b[0], a[1], b[1]}, hi[4] = {a[2], b[2], a[3], b[3]};
      store4(x + off_a, lo);
      store4(x + off_b, hi);
    } else if (LAYOUT == kHalves) {
      store4(x + off_a, a);
      store4(x + off_b, b);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = ea(first + j), k = eb(first + j);
        if (i < dim) x[i] = from_f32<T>(a[j]);
        if (k < dim) x[k] = from_f32<T>(b[j]);
      }
    }
  }
  // cos and sin of the four pairs at token t; 1 and 0 where a pair does not turn
  __device__ void table(const RopeArgs& a, int64_t t, float (&c)[4], float (&s)[4]) const {
    const int64_t p = position(a, t);
    const bool inside = p >= 0 && p < a.table_rows;
    const float nan = __int_as_float(0x7fc00000);
    const float *ct = a.cos_t + (inside ? p : 0) * half + first, *st = a.sin_t + (inside ? p : 0) * half + first;
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = 1.0f, s[j] = 0.0f;
    if (!inside) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (turns(j)) c[j] = s[j] = nan;
    } else if (a.table_vec) {  // rows of whole vectors: a lane turns all its pairs or none
      if (first < half) {
        unpack(*reinterpret_cast<const Raw4<float>*>(ct), c);
        unpack(*reinterpret_cast<const Raw4<float>*>(st), s);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (turns(j)) c[j] = ct[j], s[j] = st[j];
    }
  }
  template <typename T>
  __device__ void weights(const void* w, int w32, float (&a)[4], float (&b)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = b[j] = 1.0f;
    if (!w || !on) return;
    if (w32) {
      Raw8<float> r;
      fetch(static_cast<const float*>(w), r);
      get(r, a, b);
    } else {
      Raw8<T> r;
      fetch(static_cast<const T*>(w), r);
      get(r, a, b);
    }
  }
  // the element that slot i holds: a[i], then b[i - 4]
  __device__ int element(int i) const {
    const int j = i & 3;
    if (LAYOUT == kHalves) return (i < 4 ? off_a : off_b) + j;
    return i < 4 ? ea(first + j) : eb(first + j);
  }
};

// A unit of work: a.unit_heads heads of one token, of its queries or keys.
template <typename T, int L, int LAYOUT>
__global__ void __launch_bounds__(kVecThreads, 8) rope_forward(RopeArgs a, uint32_t units) {
  constexpr int kGroups = 32 / L, kBatch = sizeof(T) == 2 ? 4 : 2;
  allow_next();
  wait_for_previous();
  const uint32_t id = blockIdx.x * kVecWarps + (threadIdx.x >> 5);
  if (id >= units) return;
  const int lane = threadIdx.x & 31, group = lane / L;
  const Pairs<LAYOUT> pr(a, lane % L);
  const uint32_t t = id / a.units_token, i = id - t * a.units_token;
  const int which = i >= a.units_q;
  const int heads = a.heads[which];
  const int64_t stride = a.stride_h[which];
  int h = (int)(which ? i - a.units_q : i) * a.unit_heads + group;
  const int last = min(h - group + a.unit_heads, heads);
  const T* x = static_cast<const T*>(a.x[which]) + (int64_t)t * a.stride_t[which];
  T* z = static_cast<T*>(a.out[which]) + (int64_t)t * heads * a.dim;
  // z_a = r (x_a aa + x_b ab), z_b = r (x_b bb + x_a ba): the weights times cos and sin
  uint64_t aa[2], ab[2], bb[2], ba[2];
  bool ready = false;
  for (; h - group < last; h += kBatch * kGroups) {
    Raw8<T> xr[kBatch] = {};
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (h + k * kGroups < last && pr.on) pr.fetch(x + (h + k * kGroups) * stride, xr[k]);
    if (!ready) {  // while the first heads are on their way
      float c[4], s[4], wa[4], wb[4];
      pr.table(a, t, c, s);
      pr.template weights<T>(a.w[which], a.weight32, wa, wb);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint64_t ci = pair(c[2 * i], c[2 * i + 1]), si = pair(s[2 * i], s[2 * i + 1]);
        const uint64_t wai = pair(wa[2 * i], wa[2 * i + 1]), wbi = pair(wb[2 * i], wb[2 * i + 1]);
        aa[i] = mul2(wai, ci), ab[i] = mul2(mul2(wbi, si), pair(-1.0f, -1.0f));
        bb[i] = mul2(wbi, ci), ba[i] = mul2(wai, si);
      }
      ready = true;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int at = h + k * kGroups;
      if (at - group >= last) break;
      uint64_t xa[2], xb[2], za[2], zb[2];
      pr.get(xr[k], xa, xb);
      float s0, s1;
      unpair(fma2(xa[0], xa[0], fma2(xa[1], xa[1], fma2(xb[0], xb[0], mul2(xb[1], xb[1])))), s0, s1);
      const float r = rsqrtf(group_sum<L>(s0 + s1) * a.inv_dim + a.eps);
      pr.turned(xa, xb, aa, ab, bb, ba, za, zb);
      const uint64_t rr = pair(r, r);
#pragma unroll
      for (int i = 0; i < 2; ++i) za[i] = mul2(za[i], rr), zb[i] = mul2(zb[i], rr);
      if (at < last && pr.on) pr.store(z + at * a.dim, za, zb);
    }
  }
}

// Persistent: warps walk the units of the queries, then those of the keys,
// with their sums for dw in registers, moved to fp64 in shared memory often
// enough that no fp32 sum runs over more than kFlush terms.
template <typename T, int L, int LAYOUT>
__global__ void __launch_bounds__(kVecThreads, 4) rope_backward(RopeArgs a) {
  constexpr int kGroups = 32 / L, kBatch = 2;
  __shared__ double acc[kVecWarps][16][32];  // [warp][which * 8 + a0..3 b0..3][lane]
  allow_next();
  wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / L;
  const Pairs<LAYOUT> pr(a, lane % L);
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[warp][i][lane] = 0.0;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int heads = a.heads[which];
    const int64_t stride = a.stride_h[which];
    const uint32_t per_token = which ? a.units_token - a.units_q : a.units_q;
    const uint32_t units = (uint32_t)a.tokens * per_token;
    uint64_t wa[2], wb[2], ga[2] = {}, gb[2] = {};
    {
      float u[4], v[4];
      pr.template weights<T>(a.w[which], a.weight32, u, v);
#pragma unroll
      for (int i = 0; i < 2; ++i) wa[i] = pair(u[2 * i], u[2 * i + 1]), wb[i] = pair(v[2 * i], v[2 * i + 1]);
    }
    int terms = 0;
    auto flush = [&] {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float u[2], v[2];
        unpair(ga[i], u[0], u[1]), unpair(gb[i], v[0], v[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[warp][which * 8 + 2 * i + j][lane] += (double)u[j];
          acc[warp][which * 8 + 4 + 2 * i + j][lane] += (double)v[j];
        }
        ga[i] = gb[i] = 0;
      }
      terms = 0;
    };
    for (uint32_t id = blockIdx.x * kVecWarps + warp; id < units; id += gridDim.x * kVecWarps) {
      const uint32_t t = id / per_token;
      int h = (int)(id - t * per_token) * a.unit_heads + group;
      const int last = min(h - group + a.unit_heads, heads);
      const T* x = static_cast<const T*>(a.x[which]) + (int64_t)t * a.stride_t[which];
      const T* dz = static_cast<const T*>(a.dz[which]) + (int64_t)t * heads * a.dim;
      T* dx = static_cast<T*>(a.out[which]) + (int64_t)t * heads * a.dim;
      uint64_t cc[2], sn[2], ns[2];
      Raw8<T> xr[kBatch] = {}, dr[kBatch] = {};
      auto fetch = [&](int k, int at) {
        if (at < last && pr.on) {
          pr.fetch(x + at * stride, xr[k]);
          pr.fetch(dz + at * a.dim, dr[k]);
        }
      };
#pragma unroll
      for (int k = 0; k < kBatch; ++k) fetch(k, h + k * kGroups);
      {
        float c[4], s[4];
        pr.table(a, t, c, s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          cc[i] = pair(c[2 * i], c[2 * i + 1]), sn[i] = pair(s[2 * i], s[2 * i + 1]);
          ns[i] = pair(-s[2 * i], -s[2 * i + 1]);
        }
      }
      for (; h - group < last; h += kBatch * kGroups) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int at = h + k * kGroups;
          if (at - group >= last) break;
          uint64_t xa[2], xb[2], da[2], db[2], ya[2], yb[2], ta[2], tb[2];
          pr.get(xr[k], xa, xb);
          pr.get(dr[k], da, db);
          fetch(k, at + kBatch * kGroups);  // the head that takes this one's place
          pr.turned(da, db, cc, sn, cc, ns, ya, yb);  // dy
#pragma unroll
          for (int i = 0; i < 2; ++i) ta[i] = mul2(ya[i], xa[i]), tb[i] = mul2(yb[i], xb[i]);
          float ss, dot, s1, d1;
          unpair(fma2(xa[0], xa[0], fma2(xa[1], xa[1], fma2(xb[0], xb[0], mul2(xb[1], xb[1])))), ss, s1);
          unpair(fma2(ta[0], wa[0], fma2(ta[1], wa[1], fma2(tb[0], wb[0], mul2(tb[1], wb[1])))), dot, d1);
          ss += s1;
          dot += d1;
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) {
            ss += __shfl_xor_sync(0xffffffffu, ss, o);
            dot += __shfl_xor_sync(0xffffffffu, dot, o);
          }
          const float r = rsqrtf(ss * a.inv_dim + a.eps);
          const float m = -(r * dot * a.inv_dim * r);  // - r mean(dy w xh)
          const bool mine = at < last && pr.on;
          const float rg = mine ? r : 0.0f;
          const uint64_t rr = pair(r, r), mm = pair(m, m), rrg = pair(rg, rg);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ga[i] = fma2(ta[i], rrg, ga[i]);
            gb[i] = fma2(tb[i], rrg, gb[i]);
            ya[i] = mul2(rr, fma2(xa[i], mm, mul2(ya[i], wa[i])));
            yb[i] = mul2(rr, fma2(xb[i], mm, mul2(yb[i], wb[i])));
          }
          if (mine) pr.store(dx + at * a.dim, ya, yb);
        }
        if (++terms == kFlush / kBatch) flush();
      }
    }
    flush();
  }
  __syncthreads();
  // element e of weight `which`: over warps and groups of lanes, in order
  for (int i = threadIdx.x; i < 16 * L; i += kVecThreads) {
    const int slot = i / L, of = i % L;
    double sum = 0.0;
    for (int w = 0; w < kVecWarps; ++w)
      for (int g = 0; g < kGroups; ++g) sum += acc[w][slot][g * L + of];
    const int e = Pairs<LAYOUT>(a, of).element(slot & 7);
    if (e < a.dim) a.partial[(int64_t)blockIdx.x * 2 * a.dim + (slot >> 3) * a.dim + e] = sum;
  }
}

// Heads larger than kVecDim: one warp per (token, head), the vector staged in
// shared memory.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rope_forward_any(RopeArgs a) {
  extern __shared__ float smem[];
  allow_next();
  wait_for_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* y = smem + warp * a.dim;
  const int total_heads = a.heads[0] + a.heads[1];
  const int64_t items = a.tokens * total_heads;
  const float nan = __int_as_float(0x7fc00000);
  for (int64_t it = (int64_t)blockIdx.x * kWarps + warp; it < items; it += (int64_t)gridDim.x * kWarps) {
    const int64_t t = it / total_heads;
    int h = (int)(it - t * total_heads);
    const int which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const T* x = static_cast<const T*>(a.x[which]) + t * a.stride_t[which] + h * a.stride_h[which];
    T* z = static_cast<T*>(a.out[which]) + (t * a.heads[which] + h) * a.dim;
    float ss = 0.0f;
    for (int e = lane; e < a.dim; e += 32) {
      const float v = to_f32(x[e]);
      y[e] = v;
      ss += v * v;
    }
    const float r = rsqrtf(warp_sum(ss) / (float)a.dim + a.eps);
    for (int e = lane; e < a.dim; e += 32) y[e] *= r * weight_at<W>(a.w[which], e);
    __syncwarp();
    const int64_t p = position(a, t);
    const bool inside = p >= 0 && p < a.table_rows;
    const int64_t row = inside ? p * (a.rotary >> 1) : 0;
    for (int e = lane; e < a.dim; e += 32) {
      float v = y[e];
      if (e < a.rotary) {
        int i, partner;
        bool first;
        pair_of(e, a.rotary, a.interleaved, i, partner, first);
        const float c = inside ? a.cos_t[row + i] : nan, s = inside ? a.sin_t[row + i] : nan;
        v = first ? v * c - y[partner] * s : v * c + y[partner] * s;
      }
      z[e] = from_f32<T>(v);
    }
    __syncwarp();
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rope_backward_any(RopeArgs a) {
  extern __shared__ double dsmem[];
  allow_next();
  wait_for_previous();
  // per warp: dw of both weights (fp64), then dy
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double* acc = dsmem + (int64_t)warp * 2 * a.dim;
  float* dy = reinterpret_cast<float*>(dsmem + (int64_t)kWarps * 2 * a.dim) + warp * a.dim;
  for (int e = lane; e < 2 * a.dim; e += 32) acc[e] = 0.0;
  const int total_heads = a.heads[0] + a.heads[1];
  const int64_t items = a.tokens * total_heads;
  const float nan = __int_as_float(0x7fc00000);
  for (int64_t it = (int64_t)blockIdx.x * kWarps + warp; it < items; it += (int64_t)gridDim.x * kWarps) {
    const int64_t t = it / total_heads;
    int h = (int)(it - t * total_heads);
    const int which = h >= a.heads[0];
    if (which) h -= a.heads[0];
    const T* x = static_cast<const T*>(a.x[which]) + t * a.stride_t[which] + h * a.stride_h[which];
    const int64_t at = (t * a.heads[which] + h) * a.dim;
    const T* dz = static_cast<const T*>(a.dz[which]) + at;
    T* dx = static_cast<T*>(a.out[which]) + at;
    float ss = 0.0f;
    for (int e = lane; e < a.dim; e += 32) {
      const float v = to_f32(x[e]);
      ss += v * v;
    }
    const float r = rsqrtf(warp_sum(ss) / (float)a.dim + a.eps);
    const int64_t p = position(a, t);
    const bool inside = p >= 0 && p < a.table_rows;
    const int64_t row = inside ? p * (a.rotary >> 1) : 0;
    float dot = 0.0f;
    for (int e = lane; e < a.dim; e += 32) {
      float g = to_f32(dz[e]);
      if (e < a.rotary) {
        int i, partner;
        bool first;
        pair_of(e, a.rotary, a.interleaved, i, partner, first);
        const float c = inside ? a.cos_t[row + i] : nan, s = inside ? a.sin_t[row + i] : nan;
        const float o = to_f32(dz[partner]);
        g = first ? g * c + o * s : g * c - o * s;
      }
      const float xh = to_f32(x[e]) * r;
      acc[which * a.dim + e] += (double)(g * xh);
      g *= weight_at<W>(a.w[which], e);
      dy[e] = g;
      dot += g * xh;
    }
    const float mean = warp_sum(dot) / (float)a.dim;
    for (int e = lane; e < a.dim; e += 32) {
      const float xh = to_f32(x[e]) * r;
      dx[e] = from_f32<T>(r * (dy[e] - xh * mean));
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * a.dim; e += kThreads) {
    double s = 0.0;
    for (int w = 0; w < kWarps; ++w) s += dsmem[(int64_t)w * 2 * a.dim + e];
    a.partial[(int64_t)blockIdx.x * 2 * a.dim + e] = s;
  }
}

// dw[e] = the sum of the CTAs' partials, in an order that the sizes fix.
template <typename W>
__global__ void __launch_bounds__(1024) rope_weight_grads(const double* partial, int parts, int dim, W* dqw, W* dkw) {
  __shared__ double red[128][9];
  const int col = threadIdx.x & 7, row = threadIdx.x >> 3;  // 8 columns of the partials x 128 of their rows
  const int e = blockIdx.x * 8 + col;
  allow_next();
  wait_for_previous();  // for the partials
  double s = 0.0;
  if (e < 2 * dim)
#pragma unroll 8
    for (int i = row; i < parts; i += 128) s += partial[(int64_t)i * 2 * dim + e];
  red[row][col] = s;
  __syncthreads();
  if (row < 16) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += red[row + 16 * i][col];
    red[row][col] = s;
  }
  __syncthreads();
  if (row || e >= 2 * dim) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += red[i][col];
  W* out = e < dim ? dqw : dkw;
  if (out) out[e < dim ? e : e - dim] = from_f32<W>((float)s);
}

int backward_grid(int64_t tokens, int heads) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(tokens * heads, kWarps), (int64_t)sm_count() * 4));
}

// Lanes per head: the power of two that holds dim / 8 of them.
int lanes_for(int64_t dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }
// Fills in the layout of the register kernels; returns the units of work.  A
// unit takes up to 4 * `most` heads per group of lanes (cos, sin and weights
// are prepared once for them), fewer while that leaves SMs without work.
int64_t lay_out(RopeArgs& a, int most) {
  const int step = 32 / lanes_for(a.dim) * 4;
  auto units = [&](int64_t heads) { return ceil_div(a.heads[0], heads) + ceil_div(a.heads[1], heads); };
  a.unit_heads = step * most;
  while (a.unit_heads > step && a.tokens * units(a.unit_heads) < (int64_t)sm_count() * 64) a.unit_heads /= 2;
  a.units_q = (uint32_t)ceil_div(a.heads[0], a.unit_heads);
  a.units_token = (uint32_t)units(a.unit_heads);
  a.inv_dim = 1.0f / (float)a.dim;
  a.table_vec = a.rotary % 8 == 0 && aligned16(a.cos_t) && aligned16(a.sin_t);
  return a.tokens * a.units_token;
}
// Whether a lane's elements can be read as vectors of four.
bool vector_ok(const RopeArgs& a, int e, bool backward) {
  auto whole = [&](const void* p) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % (4 * e) == 0; };
  if (a.dim % 8 || (!a.interleaved && a.rotary % 8)) return false;
  for (int i = 0; i < 2; ++i) {
    if (a.stride_t[i] % 4 || a.stride_h[i] % 4 || !whole(a.x[i]) || !whole(a.out[i]) || !aligned16(a.w[i])) return false;
    if (backward && !whole(a.dz[i])) return false;
  }
  return true;
}
// f(lanes per head, layout): both as types that hold a constant
template <typename F>
int with_layout(const RopeArgs& a, bool vec, F f) {
  auto lanes = [&](auto layout) {
    const int l = lanes_for(a.dim);
    if (l == 8) return f(std::integral_constant<int, 8>{}, layout);
    if (l == 16) return f(std::integral_constant<int, 16>{}, layout);
    return f(std::integral_constant<int, 32>{}, layout);
  };
  if (!vec) return lanes(std::integral_constant<int, kAny>{});
  if (a.interleaved) return lanes(std::integral_constant<int, kNeighbours>{});
  return lanes(std::integral_constant<int, kHalves>{});
}

int check_shape(const char* name, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t dim, int64_t rotary,
                int64_t table_rows, int dtype, int weight_dtype) {
  KB_REQUIRE(tokens >= 0 && heads_q >= 0 && heads_kv >= 0 && table_rows >= 0, KB_ERR_INVALID_ARG,
             "%s: negative size", name);
  KB_REQUIRE(dtype_size(dtype) && dtype_size(weight_dtype), KB_ERR_INVALID_ARG, "%s: unknown element type", name);
  KB_REQUIRE(dim >= 1 && dim <= kMaxDim, KB_ERR_UNSUPPORTED, "%s: head dim %lld not in 1..%d", name, (long long)dim,
             kMaxDim);
  KB_REQUIRE(rotary >= 0 && rotary <= dim && rotary % 2 == 0, KB_ERR_INVALID_ARG,
             "%s: rotary size %lld must be even and at most %lld", name, (long long)rotary, (long long)dim);
  // one by one before their sums and products, which have to fit 64 bits
  KB_REQUIRE(heads_q <= 65535 && heads_kv <= 65535 && heads_q + heads_kv <= 65535, KB_ERR_UNSUPPORTED,
             "%s: too many heads", name);
  KB_REQUIRE(tokens <= kMaxUnits, KB_ERR_UNSUPPORTED, "%s: too many tokens", name);
  return KB_OK;
}

// f(element type, weight type)
template <typename F>
int with_types(int dtype, int weight_dtype, F f) {
  return with_dtype(dtype, [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    if (weight_dtype == KB_F32) return f(x, static_cast<float*>(nullptr));
    return f(x, static_cast<T*>(nullptr));
  });
}

}  // namespace
}  // namespace lm
}  // namespace kb

extern "C" {

int kb_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight, const float* cos_table,
                    const float* sin_table, const void* positions, void* q_out, void* k_out, int64_t tokens,
                    int64_t heads_q, int64_t heads_kv, int64_t dim, int64_t rotary, int64_t table_rows,
                    int64_t q_stride_token, int64_t q_stride_head, int64_t k_stride_token, int64_t k_stride_head,
                    int dtype, int weight_dtype, int positions_64, int interleaved, float eps, kbStream stream) {
  const char* name = "kb_qk_norm_rope";
  using namespace kb::lm;
  if (int st = check_shape(name, tokens, heads_q, heads_kv, dim, rotary, table_rows, dtype, weight_dtype)) return st;
  KB_REQUIRE(weight_dtype == KB_F32 || weight_dtype == dtype, KB_ERR_INVALID_ARG,
             "%s: weights must be fp32 or of the inputs' type", name);
  if (tokens == 0 || heads_q + heads_kv == 0) return KB_OK;
  KB_REQUIRE((heads_q == 0 || (q && q_out)) && (heads_kv == 0 || (k && k_out)) && positions, KB_ERR_INVALID_ARG,
             "%s: null pointer", name);
  KB_REQUIRE(rotary == 0 || table_rows == 0 || (cos_table && sin_table), KB_ERR_INVALID_ARG, "%s: null table", name);
  RopeArgs a{};
  a.x[0] = q, a.x[1] = k, a.w[0] = q_weight, a.w[1] = k_weight, a.out[0] = q_out, a.out[1] = k_out;
  a.cos_t = cos_table, a.sin_t = sin_table, a.pos = positions;
  a.tokens = tokens, a.table_rows = table_rows;
  a.stride_t[0] = q_stride_token, a.stride_t[1] = k_stride_token;
  a.stride_h[0] = q_stride_head, a.stride_h[1] = k_stride_head;
  a.heads[0] = (int)heads_q, a.heads[1] = (int)heads_kv;
  a.dim = (int)dim, a.rotary = (int)rotary, a.interleaved = interleaved, a.pos64 = positions_64, a.eps = eps;
  a.weight32 = weight_dtype == KB_F32;
  if (dim <= kVecDim) {
    // 16-bit, 16384 x 40 x 128: 66 us with 2, 68 with 4, 70 with 1; fp32, half the tokens: 57, 60, 55
    const int64_t units = lay_out(a, dtype == KB_F32 ? 1 : 2), blocks = kb::ceil_div(units, kVecWarps);
    KB_REQUIRE(units <= kMaxUnits, KB_ERR_UNSUPPORTED, "%s: too many tokens", name);
    return with_dtype(dtype, [&](auto* x) {
      using T = std::remove_pointer_t<decltype(x)>;
      return with_layout(a, vector_ok(a, sizeof(T), false), [&](auto l, auto v) {
        return launch_after(rope_forward<T, decltype(l)::value, decltype(v)::value>, dim3((unsigned)blocks),
                            (unsigned)kVecThreads, 0, stream, a, units);
      });
    });
  }
  const int64_t items = tokens * (heads_q + heads_kv);
  const unsigned grid = (unsigned)std::min<int64_t>(kb::ceil_div(items, kWarps), (int64_t)kb::sm_count() * 16);
  return with_types(dtype, weight_dtype, [&](auto* x, auto* w) {
    using T = std::remove_pointer_t<decltype(x)>;
    using W = std::remove_pointer_t<decltype(w)>;
    return launch_after(rope_forward_any<T, W>, dim3(grid), (unsigned)kThreads, kWarps * dim * sizeof(float), stream, a);
  });
}

size_t kb_qk_norm_rope_backward_workspace_size(int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t dim) {
  if (tokens <= 0 || dim <= 0 || heads_q + heads_kv <= 0) return 0;
  return (size_t)kb::sm_count() * 4 * 2 * dim * sizeof(double);
}

int kb_qk_norm_rope_backward(const void* dq_out, const void* dk_out, const void* q, const void* k,
                             const void* q_weight, const void* k_weight, const float* cos_table,
                             const float* sin_table, const void* positions, void* dq, void* dk, void* dq_weight,
                             void* dk_weight, int64_t tokens, int64_t heads_q, int64_t heads_kv, int64_t dim,
                             int64_t rotary, int64_t table_rows, int64_t q_stride_token, int64_t q_stride_head,
                             int64_t k_stride_token, int64_t k_stride_head, int dtype, int weight_dtype,
                             int positions_64, int interleaved, float eps, void* workspace, size_t workspace_bytes,
                             kbStream stream) {
  const char* name = "kb_qk_norm_rope_backward";
  using namespace kb::lm;
  if (int st = check_shape(name, tokens, heads_q, heads_kv, dim, rotary, table_rows, dtype, weight_dtype)) return st;
  KB_REQUIRE(weight_dtype == KB_F32 || weight_dtype == dtype, KB_ERR_INVALID_ARG,
             "%s: weights must be fp32 or of the inputs' type", name);
  const bool any = tokens > 0 && heads_q + heads_kv > 0;
  int grid = 0;
  double* partial = nullptr;
  if (any) {
    KB_REQUIRE((heads_q == 0 || (q && dq && dq_out)) && (heads_kv == 0 || (k && dk && dk_out)) && positions,
               KB_ERR_INVALID_ARG, "%s: null pointer", name);
    KB_REQUIRE(rotary == 0 || table_rows == 0 || (cos_table && sin_table), KB_ERR_INVALID_ARG, "%s: null table", name);
    grid = backward_grid(tokens, (int)(heads_q + heads_kv));
    const size_t need = (size_t)grid * 2 * dim * sizeof(double);
    KB_REQUIRE(workspace && workspace_bytes >= need, KB_ERR_WORKSPACE,
               "%s: workspace of %zu bytes needed, %zu given", name, need, workspace_bytes);
    KB_REQUIRE(kb::aligned16(workspace), KB_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", name);
    partial = static_cast<double*>(workspace);
  }
  RopeArgs a{};
  a.x[0] = q, a.x[1] = k, a.dz[0] = dq_out, a.dz[1] = dk_out, a.w[0] = q_weight, a.w[1] = k_weight;
  a.out[0] = dq, a.out[1] = dk, a.cos_t = cos_table, a.sin_t = sin_table, a.pos = positions;
  a.tokens = tokens, a.table_rows = table_rows;
  a.stride_t[0] = q_stride_token, a.stride_t[1] = k_stride_token;
  a.stride_h[0] = q_stride_head, a.stride_h[1] = k_stride_head;
  a.heads[0] = (int)heads_q, a.heads[1] = (int)heads_kv;
  a.dim = (int)dim, a.rotary = (int)rotary, a.interleaved = interleaved, a.pos64 = positions_64, a.eps = eps;
  a.weight32 = weight_dtype == KB_F32;
  a.partial = partial;
  return with_types(dtype, weight_dtype, [&](auto* x, auto* w) {
    using T = std::remove_pointer_t<decltype(x)>;
    using W = std::remove_pointer_t<decltype(w)>;
    if (any && dim <= kVecDim) {
      const int64_t units = lay_out(a, dtype == KB_F32 ? 1 : 4);  // as above: 112 us with 4, 118 with 1; fp32 99, 92
      KB_REQUIRE(units <= kMaxUnits, KB_ERR_UNSUPPORTED, "%s: too many tokens", name);
      grid = (int)std::min<int64_t>(kb::ceil_div(units, kVecWarps), (int64_t)kb::sm_count() * 4);  // four per SM
      if (int st = with_layout(a, vector_ok(a, sizeof(T), true), [&](auto l, auto v) {
            return launch_after(rope_backward<T, decltype(l)::value, decltype(v)::value>, dim3((unsigned)grid),
                                (unsigned)kVecThreads, 0, stream, a);
          }))
        return st;
    } else if (any) {
      const size_t smem = (size_t)kWarps * dim * (2 * sizeof(double) + sizeof(float));
      if (int st = launch_after(rope_backward_any<T, W>, dim3((unsigned)grid), (unsigned)kThreads, smem, stream, a))
        return st;
    }
    if (!dq_weight && !dk_weight) return (int)KB_OK;
    return launch_after(rope_weight_grads<W>, dim3((unsigned)kb::ceil_div(2 * dim, 8)), 1024u, 0, stream,
                        (const double*)partial, grid, dim, static_cast<W*>(dq_weight), static_cast<W*>(dk_weight));
  });
}

}  // extern "C"
