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
// in fp64 per warp, then over warps and CTAs in a fixed order, so it does not
// depend on timing.  A position outside the table gives NaN in the rotated
// elements.
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
  int dim, rotary, interleaved, pos64;
  float eps;
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

// One warp per (token, head), the vector staged in shared memory: any dim up
// to kMaxDim, any rotary size, any alignment and strides.
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads) rope_forward_any(RopeArgs a) {
  extern __shared__ float smem[];
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

// dw[e] = the sum of the CTAs' partials in their order.
template <typename W>
__global__ void rope_weight_grads(const double* __restrict__ partial, int parts, int dim, W* __restrict__ dqw,
                                  W* __restrict__ dkw) {
  __shared__ double red[8][33];
  const int lane = threadIdx.x, row = threadIdx.y;  // 32 x 8: a column of the partials per lane
  const int e = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (e < 2 * dim)
    for (int i = row; i < parts; i += 8) s += partial[(int64_t)i * 2 * dim + e];
  red[row][lane] = s;
  __syncthreads();
  if (row || e >= 2 * dim) return;
  for (int i = 1; i < 8; ++i) s += red[i][lane];
  W* out = e < dim ? dqw : dkw;
  if (out) out[e < dim ? e : e - dim] = from_f32<W>((float)s);
}

int backward_grid(int64_t tokens, int heads) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(tokens * heads, kWarps), (int64_t)sm_count() * 4));
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
  KB_REQUIRE(heads_q + heads_kv <= 65535, KB_ERR_UNSUPPORTED, "%s: too many heads", name);
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
  const int64_t items = tokens * (heads_q + heads_kv);
  const unsigned grid = (unsigned)std::min<int64_t>(kb::ceil_div(items, kWarps), (int64_t)kb::sm_count() * 16);
  return with_types(dtype, weight_dtype, [&](auto* x, auto* w) {
    using T = std::remove_pointer_t<decltype(x)>;
    using W = std::remove_pointer_t<decltype(w)>;
    rope_forward_any<T, W><<<grid, kThreads, kWarps * dim * sizeof(float), stream>>>(a);
    return kb::check_launch(name);
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
  a.partial = partial;
  return with_types(dtype, weight_dtype, [&](auto* x, auto* w) {
    using T = std::remove_pointer_t<decltype(x)>;
    using W = std::remove_pointer_t<decltype(w)>;
    if (any) {
      const size_t smem = (size_t)kWarps * dim * (2 * sizeof(double) + sizeof(float));
      rope_backward_any<T, W><<<grid, kThreads, smem, stream>>>(a);
      if (int st = kb::check_launch(name)) return st;
    }
    if (!dq_weight && !dk_weight) return (int)KB_OK;
    rope_weight_grads<W><<<(unsigned)kb::ceil_div(2 * dim, 32), dim3(32, 8), 0, stream>>>(
        partial, grid, (int)dim, static_cast<W*>(dq_weight), static_cast<W*>(dk_weight));
    return kb::check_launch(name);
  });
}

}  // extern "C"
