// lm_logits.cu — penalties for repeated tokens, biases and grammar masks on
// the logits of a batch, in one pass.
//
// For row b and token v with logit l, c = how often v stands in the row's
// output history, seen = v stands in its prompt or output history:
//   l1 = seen ? (l > 0 ? l / repetition : l * repetition) : l
//   l2 = l1 - frequency c - (c > 0 ? presence : 0)
//   l3 = l2 + bias(v)                       (the last listing of v counts)
//   out = mask bit v set ? l3 : -inf
// in fp32, rounded once.  Ids outside [0, vocab) (padding) are ignored.
//
// A CTA owns a chunk of one row's vocabulary and keeps one 32-bit word per
// token of it in shared memory: the count, a bit for the prompt and the
// index of the bias.  Histories are scattered into the words with integer
// atomics, whose order does not change the result.
#include "lm_common.cuh"

namespace kb {
namespace lm {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;                      // tokens per CTA: 32 KB of words
constexpr int kCountBits = 20, kBiasShift = 21;   // count | prompt bit | bias index + 1
constexpr uint32_t kCountMask = (1u << kCountBits) - 1, kPromptBit = 1u << kCountBits;
constexpr int64_t kMaxOutput = kCountMask, kMaxBias = (1 << (32 - kBiasShift)) - 1;

struct LogitsArgs {
  const void* logits;
  void* out;
  const void *prompt, *output, *bias_ids;
  const float *repetition, *presence, *frequency, *bias_values;
  const uint32_t* mask;
  int64_t vocab, stride, n_prompt, n_output, n_bias, mask_stride;
  int ids64;
};

__device__ __forceinline__ int64_t id_at(const void* ids, int64_t i, int ids64) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

template <typename T>
__global__ void __launch_bounds__(kThreads) penalize_kernel(LogitsArgs a) {
  __shared__ uint32_t word[kChunk];
  const int64_t row = blockIdx.y, first = (int64_t)blockIdx.x * kChunk;
  const int n = (int)min((int64_t)kChunk, a.vocab - first);
  for (int i = threadIdx.x; i < n; i += kThreads) word[i] = 0;
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.n_bias; i += kThreads) {
    const int64_t v = id_at(a.bias_ids, row * a.n_bias + i, a.ids64) - first;
    if (v >= 0 && v < n) atomicMax(&word[v], (uint32_t)(i + 1) << kBiasShift);
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < a.n_prompt; i += kThreads) {
    const int64_t v = id_at(a.prompt, row * a.n_prompt + i, a.ids64) - first;
    if (v >= 0 && v < n) atomicOr(&word[v], kPromptBit);
  }
  for (int64_t i = threadIdx.x; i < a.n_output; i += kThreads) {
    const int64_t v = id_at(a.output, row * a.n_output + i, a.ids64) - first;
    if (v >= 0 && v < n) atomicAdd(&word[v], 1u);
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[row] : 1.0f;
  const float pres = a.presence ? a.presence[row] : 0.0f;
  const float freq = a.frequency ? a.frequency[row] : 0.0f;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride + first;
  T* y = static_cast<T*>(a.out) + row * a.vocab + first;
  const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float l = to_f32(x[i]);
    const uint32_t w = word[i];
    if (w & (kCountMask | kPromptBit)) {
      l = l > 0.0f ? l / rep : l * rep;
      const uint32_t c = w & kCountMask;
      if (c) l = l - freq * (float)c - pres;
    }
    if (w >> kBiasShift) l += a.bias_values[row * a.n_bias + (w >> kBiasShift) - 1];
    if (mask && !(mask[(first + i) >> 5] >> ((first + i) & 31) & 1)) l = -INFINITY;
    y[i] = from_f32<T>(l);
  }
}

}  // namespace
}  // namespace lm
}  // namespace kb

extern "C" {

int kb_penalize_logits(const void* logits, void* out, const void* prompt, const void* output,
                       const float* repetition, const float* presence, const float* frequency, const void* bias_ids,
                       const float* bias_values, const void* mask, int64_t rows, int64_t vocab, int64_t row_stride,
                       int64_t prompt_len, int64_t output_len, int64_t bias_len, int64_t mask_stride, int dtype,
                       int ids_64, kbStream stream) {
  const char* name = "kb_penalize_logits";
  using namespace kb::lm;
  KB_REQUIRE(rows >= 0 && vocab >= 0 && prompt_len >= 0 && output_len >= 0 && bias_len >= 0, KB_ERR_INVALID_ARG,
             "%s: negative size", name);
  KB_REQUIRE(dtype_size(dtype), KB_ERR_INVALID_ARG, "%s: unknown element type", name);
  if (rows == 0 || vocab == 0) return KB_OK;
  KB_REQUIRE(logits && out, KB_ERR_INVALID_ARG, "%s: null pointer", name);
  KB_REQUIRE(row_stride >= vocab || rows == 1, KB_ERR_INVALID_ARG, "%s: row stride smaller than the vocabulary", name);
  KB_REQUIRE((!prompt_len || prompt) && (!output_len || output) && (!bias_len || (bias_ids && bias_values)),
             KB_ERR_INVALID_ARG, "%s: null history or bias", name);
  KB_REQUIRE(output_len <= kMaxOutput, KB_ERR_UNSUPPORTED, "%s: output history longer than %lld", name,
             (long long)kMaxOutput);
  KB_REQUIRE(bias_len <= kMaxBias, KB_ERR_UNSUPPORTED, "%s: more than %lld biases a row", name, (long long)kMaxBias);
  KB_REQUIRE(rows <= 65535, KB_ERR_UNSUPPORTED, "%s: more than 65535 rows", name);
  KB_REQUIRE(kb::ceil_div(vocab, kChunk) <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: vocabulary too large", name);
  LogitsArgs a{logits, out, prompt, output, bias_ids, repetition, presence, frequency, bias_values,
               static_cast<const uint32_t*>(mask), vocab, row_stride, prompt_len, output_len, bias_len, mask_stride,
               ids_64};
  const dim3 grid((unsigned)kb::ceil_div(vocab, kChunk), (unsigned)rows);
  return with_dtype(dtype, [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    penalize_kernel<T><<<grid, kThreads, 0, stream>>>(a);
    return kb::check_launch(name);
  });
}

}  // extern "C"
