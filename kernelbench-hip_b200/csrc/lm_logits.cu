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
// Bound by HBM (logits in, logits out); the histories are small, but finding
// out which tokens they hold takes a chain of latencies.  Two ways:
//
// Large batches: two launches.  The first only copies and masks, at the speed
// of HBM.  The second, one CTA per row, gathers the row's ids into a hash
// table in shared memory (one 32-bit word per token: the output count, a bit
// for the prompt, the index of the bias), as soon as it finds room beside the
// first launch's CTAs (programmatic dependent launch; mostly as those leave),
// waits for them, and writes the tokens that change.
//
// Small batches and histories too long for the table: one launch.  A CTA takes
// a slice of one row's vocabulary with one word per token of it in shared
// memory, reads the row's whole histories, scatters the ids of its slice into
// the words and lists the tokens that have one, copies and masks the slice,
// and writes the listed tokens again.
//
// Either way words are changed by integer atomics only, whose order does not
// change the result.
//
// 256 x 131072 bf16 with 3000 ids and 300 biases a row and a mask, on a B200:
// 43 us, of which the copy takes 20 (142 MB; 7.1 TB/s, where a plain copy of larger
// buffers measures 6.6: part of what it writes is still in L2 as it ends); one launch
// of slices took 63, and a cluster of CTAs per row that shared the histories out and
// scattered them over distributed shared memory 112.
#include "lm_common.cuh"

namespace kb {
namespace lm {
namespace {

constexpr int kThreads = 512, kCopyThreads = 256, kRowThreads = 1024;
constexpr int kFlight = 4;        // vectors in flight per thread
constexpr int kTouched = 4;       // changed tokens in flight per thread
constexpr int kIds = 3;           // ids of each history in flight per thread at first
constexpr int kMinSlice = 2048;   // tokens of a CTA's slice
constexpr int kMaxSlice = 16384;  // 96 KB of words and list: two CTAs per SM
constexpr uint32_t kNoKey = 0xffffffffu;
constexpr int kMaxTable = 16384;          // slots: 128 KB of keys and words
constexpr int64_t kLargeBytes = 8 << 20;  // logits from which two launches pay
constexpr int kCountBits = 20, kBiasShift = 21;   // count | prompt bit | bias index + 1
constexpr uint32_t kCountMask = (1u << kCountBits) - 1, kPromptBit = 1u << kCountBits;
constexpr int64_t kMaxPrompt = 1ll << 40;  // sums and places of ids fit 64 bits
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


// One row of a list of ids; -1 past its end.
struct List {
  const void* ids;
  int64_t from, n;
  int ids64;
  __device__ List(const void* p, int64_t row, int64_t count, int is64) : ids(p), from(row * count), n(count), ids64(is64) {}
  __device__ int64_t at(int64_t i) const { return i < n ? id_at(ids, from + i, ids64) : -1; }
};

struct RowTerms {
  float rep, pres, freq;
  const float* bias;
};
__device__ __forceinline__ float penalized(float l, uint32_t w, const RowTerms& t) {
  if (w & (kCountMask | kPromptBit)) {
    l = l > 0.0f ? l / t.rep : l * t.rep;
    const uint32_t c = w & kCountMask;
    if (c) l = l - t.freq * (float)c - t.pres;
  }
  if (w >> kBiasShift) l += t.bias[(w >> kBiasShift) - 1];
  return l;
}
// Bits i .. i + count - 1 of a bitmap, and others; the word after is read only where they reach it.
__device__ __forceinline__ uint32_t bits_at(const uint32_t* map, int64_t i, int count) {
  const uint32_t lo = map[i >> 5], hi = (i & 31) + count > 32 ? map[(i >> 5) + 1] : 0u;
  return __funnelshift_r(lo, hi, (uint32_t)i & 31);
}

// One slice of a row, n tokens from `first` on, copied or masked in vectors by
// NT threads: fetch() starts the first loads, finish() does the rest.
template <typename T, int NT>
struct Slice {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  T* y;
  const uint32_t* mask;
  int64_t first;
  int n, head;
  uint32_t vecs;
  union Vec {
    uint4 v;
    T t[kVec];
  } u[kFlight];

  __device__ Slice(const LogitsArgs& a, int64_t row, int64_t from, int count) : first(from), n(count) {
    x = static_cast<const T*>(a.logits) + row * a.stride + first;
    y = static_cast<T*>(a.out) + row * a.vocab + first;
    mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const uintptr_t px = reinterpret_cast<uintptr_t>(x), py = reinterpret_cast<uintptr_t>(y);
    // vectors after the first `head` tokens, where both are aligned alike
    head = ((px ^ py) & 15) == 0 ? min(n, (int)((16 - (px & 15)) & 15) / (int)sizeof(T)) : n;
    vecs = (uint32_t)(n - head) / kVec;
  }
  __device__ bool masked(int i) const { return mask && !(mask[(first + i) >> 5] >> ((first + i) & 31) & 1); }
  __device__ void fetch(uint32_t i0) {
#pragma unroll
    for (int f = 0; f < kFlight; ++f)
      if (i0 + f * NT < vecs) u[f].v = __ldcs(reinterpret_cast<const uint4*>(x + head + (i0 + f * NT) * kVec));
  }
  __device__ void one(int i) { y[i] = masked(i) ? from_f32<T>(-INFINITY) : x[i]; }
  __device__ void finish() {
    for (int i = threadIdx.x; i < head; i += NT) one(i);
    for (int i = head + vecs * kVec + threadIdx.x; i < n; i += NT) one(i);
    for (uint32_t i0 = threadIdx.x; i0 < vecs; i0 += kFlight * NT) {
      if (i0 != threadIdx.x) fetch(i0);
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        if (i0 + f * NT >= vecs) break;
        const int j = head + (i0 + f * NT) * kVec;
        if (mask) {
          const uint32_t allowed = bits_at(mask, first + j, kVec);
#pragma unroll
          for (int k = 0; k < kVec; ++k)
            if (!(allowed >> k & 1)) u[f].t[k] = from_f32<T>(-INFINITY);
        }
        __stcs(reinterpret_cast<uint4*>(y + j), u[f].v);
      }
    }
  }
};

__device__ __forceinline__ RowTerms terms_of(const LogitsArgs& a, int64_t row) {
  return {a.repetition ? a.repetition[row] : 1.0f, a.presence ? a.presence[row] : 0.0f,
          a.frequency ? a.frequency[row] : 0.0f, a.bias_values + row * a.n_bias};
}

// ------------------------------------------------------------------ large batches
// Grid: (slices of kCopySlice tokens, rows).
template <typename T>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(LogitsArgs a) {
  constexpr int kSlice = kCopyThreads * kFlight * 16 / sizeof(T);
  wait_for_previous();
  allow_next();  // after the wait: the next launch reads the histories before its own
  const int64_t first = (int64_t)blockIdx.x * kSlice;
  Slice<T, kCopyThreads> slice(a, blockIdx.y, first, (int)min((int64_t)kSlice, a.vocab - first));
  slice.fetch(threadIdx.x);
  slice.finish();
}

// The word of token v in the table of `size` slots (a power of two, more than
// there are ids), by linear probing.
__device__ __forceinline__ uint32_t* slot_of(uint32_t* keys, uint32_t* words, uint32_t size, uint32_t v) {
  uint32_t i = (v * 2654435761u) >> 7 & (size - 1);  // multiplicative hashing by 2^32 / golden ratio
  for (uint32_t tries = 0; tries < size; ++tries, i = (i + 1) & (size - 1)) {
    const uint32_t old = atomicCAS(&keys[i], kNoKey, v);
    if (old == kNoKey || old == v) break;
  }
  return &words[i];
}

// One CTA per row; dynamic shared memory: keys and words, `size` of each.
// Loads are issued in batches before any is used: a thread's time here is
// the number of times that it waits for memory.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) touched_kernel(LogitsArgs a, uint32_t size) {
  extern __shared__ __align__(16) uint32_t table[];
  uint32_t *keys = table, *words = table + size;
  allow_next();
  const int64_t row = blockIdx.x;
  const List bias(a.bias_ids, row, a.n_bias, a.ids64), prompt(a.prompt, row, a.n_prompt, a.ids64),
      output(a.output, row, a.n_output, a.ids64);
  auto load = [&](const List& list, int64_t i0, uint32_t (&v)[kIds]) {
#pragma unroll
    for (int k = 0; k < kIds; ++k) {
      const int64_t id = list.at(i0 + k * kRowThreads);
      v[k] = id >= 0 && id < a.vocab ? (uint32_t)id : kNoKey;
    }
  };
  auto scatter = [&](const List& list, uint32_t (&v)[kIds], auto f) {
    for (int64_t i0 = threadIdx.x; i0 < list.n; i0 += kIds * kRowThreads) {
      if (i0 != threadIdx.x) load(list, i0, v);
#pragma unroll
      for (int k = 0; k < kIds; ++k)
        if (v[k] != kNoKey) f(slot_of(keys, words, size, v[k]), i0 + k * kRowThreads);
    }
  };
  uint32_t bias_ids[kIds], prompt_ids[kIds], output_ids[kIds];
  load(bias, threadIdx.x, bias_ids);
  load(prompt, threadIdx.x, prompt_ids);
  load(output, threadIdx.x, output_ids);
  const RowTerms terms = terms_of(a, row);
  for (uint32_t i = threadIdx.x; i < size; i += kRowThreads) keys[i] = kNoKey, words[i] = 0;
  __syncthreads();
  if (a.n_bias) {
    scatter(bias, bias_ids, [](uint32_t* p, int64_t i) { atomicMax(p, (uint32_t)(i + 1) << kBiasShift); });
    __syncthreads();  // the maxima of the bias indices, before the lower bits fill
  }
  scatter(prompt, prompt_ids, [](uint32_t* p, int64_t) { atomicOr(p, kPromptBit); });
  scatter(output, output_ids, [](uint32_t* p, int64_t) { atomicAdd(p, 1u); });
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  T* y = static_cast<T*>(a.out) + row * a.vocab;
  const uint32_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
  __syncthreads();
  // The new values need nothing of the copy (where out is logits, it stores
  // these unchanged): they take the words' place, and only their way out waits.
  for (uint32_t i0 = threadIdx.x; i0 < size; i0 += kTouched * kRowThreads) {
    uint32_t v[kTouched];
    T l[kTouched];
    bool allowed[kTouched];
#pragma unroll
    for (int k = 0; k < kTouched; ++k) {
      const uint32_t i = i0 + k * kRowThreads;
      v[k] = i < size ? keys[i] : kNoKey;
      allowed[k] = v[k] != kNoKey && (!mask || (mask[v[k] >> 5] >> (v[k] & 31) & 1));
      l[k] = v[k] != kNoKey ? x[v[k]] : from_f32<T>(0.0f);
    }
#pragma unroll
    for (int k = 0; k < kTouched; ++k) {
      const uint32_t i = i0 + k * kRowThreads;
      if (allowed[k])
        words[i] = __float_as_uint(penalized(to_f32(l[k]), words[i], terms));
      else if (v[k] != kNoKey)
        keys[i] = kNoKey;
    }
  }
  wait_for_previous();  // until the copy is done
  for (uint32_t i = threadIdx.x; i < size; i += kRowThreads)  // the thread's own slots: no barrier
    if (keys[i] != kNoKey) y[keys[i]] = from_f32<T>(__uint_as_float(words[i]));
}

// ------------------------------------------------------------------ small batches, long histories
// Grid: (slices, rows); `slice` tokens, a multiple of 32.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) penalize_kernel(LogitsArgs a, int slice_size) {
  extern __shared__ __align__(16) uint32_t word[];  // [slice_size], then the list of tokens that have one
  uint16_t* list = reinterpret_cast<uint16_t*>(word + slice_size);
  __shared__ uint32_t listed;
  allow_next();
  wait_for_previous();
  const int64_t row = blockIdx.y, first = (int64_t)blockIdx.x * slice_size;
  const int n = (int)min((int64_t)slice_size, a.vocab - first);
  Slice<T, kThreads> slice(a, row, first, n);
  slice.fetch(threadIdx.x);  // on their way while the histories are read
  const RowTerms terms = terms_of(a, row);
  // the first ids of each list, too
  const List bias(a.bias_ids, row, a.n_bias, a.ids64), prompt(a.prompt, row, a.n_prompt, a.ids64),
      output(a.output, row, a.n_output, a.ids64);
  const int64_t bias_id = bias.at(threadIdx.x);
  int64_t prompt_ids[kIds], output_ids[kIds];
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    prompt_ids[k] = prompt.at(threadIdx.x + k * kThreads);
    output_ids[k] = output.at(threadIdx.x + k * kThreads);
  }
  for (int i = threadIdx.x * 4; i < slice_size; i += kThreads * 4)
    *reinterpret_cast<uint4*>(word + i) = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  auto scatter = [&](int64_t id, auto f) {
    const int64_t v = id - first;
    if (v >= 0 && v < n && f(&word[v]) == 0) list[atomicAdd(&listed, 1u)] = (uint16_t)v;
  };
  if (a.n_bias) {
    scatter(bias_id, [&](uint32_t* p) { return atomicMax(p, (uint32_t)(threadIdx.x + 1) << kBiasShift); });
    for (int64_t i = threadIdx.x + kThreads; i < a.n_bias; i += kThreads)
      scatter(bias.at(i), [&](uint32_t* p) { return atomicMax(p, (uint32_t)(i + 1) << kBiasShift); });
    __syncthreads();  // the maxima of the bias indices, before the lower bits fill
  }
  auto seen = [](uint32_t* p) { return atomicOr(p, kPromptBit); };
  auto made = [](uint32_t* p) { return atomicAdd(p, 1u); };
#pragma unroll
  for (int k = 0; k < kIds; ++k) {
    scatter(prompt_ids[k], seen);
    scatter(output_ids[k], made);
  }
#pragma unroll 4
  for (int64_t i = threadIdx.x + kIds * kThreads; i < a.n_prompt; i += kThreads) scatter(prompt.at(i), seen);
#pragma unroll 4
  for (int64_t i = threadIdx.x + kIds * kThreads; i < a.n_output; i += kThreads) scatter(output.at(i), made);
  slice.finish();
  __syncthreads();  // the list is whole, the slice is written
  for (uint32_t k = threadIdx.x; k < listed; k += kThreads) {
    const int i = list[k];
    // where out is logits, the value has been stored unchanged
    if (!slice.masked(i)) slice.y[i] = from_f32<T>(penalized(to_f32(slice.x[i]), word[i], terms));
  }
}

// Sets a kernel's limit of dynamic shared memory, once per device.
int allow_smem(const void* kernel, int bytes, uint64_t& done) {
  int dev = 0;
  KB_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && (done >> dev & 1)) return KB_OK;
  KB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done |= 1ull << dev;
  return KB_OK;
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
  KB_REQUIRE(prompt_len <= kMaxPrompt, KB_ERR_UNSUPPORTED, "%s: prompt history too long", name);
  KB_REQUIRE(rows <= 65535, KB_ERR_UNSUPPORTED, "%s: more than 65535 rows", name);
  KB_REQUIRE(vocab <= 0x7fffffff, KB_ERR_UNSUPPORTED, "%s: vocabulary too large", name);
  LogitsArgs a{logits, out, prompt, output, bias_ids, repetition, presence, frequency, bias_values,
               static_cast<const uint32_t*>(mask), vocab, row_stride, prompt_len, output_len, bias_len, mask_stride,
               ids_64};
  const int64_t ids = prompt_len + output_len + bias_len;
  return with_dtype(dtype, [&](auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    if (ids == 0 || (ids <= kMaxTable / 2 && rows * vocab * (int64_t)sizeof(T) >= kLargeBytes)) {
      constexpr int kSlice = kCopyThreads * kFlight * 16 / sizeof(T);
      const dim3 grid((unsigned)kb::ceil_div(vocab, kSlice), (unsigned)rows);
      if (int st = launch_after(copy_kernel<T>, grid, (unsigned)kCopyThreads, 0, stream, a)) return st;
      if (ids == 0) return (int)KB_OK;
      static uint64_t done = 0;
      if (int st = allow_smem((const void*)touched_kernel<T>, kMaxTable * 8, done)) return st;
      uint32_t size = 32;
      while (size < 2 * ids) size *= 2;
      return launch_after(touched_kernel<T>, dim3((unsigned)rows), (unsigned)kRowThreads, size * 8, stream, a, size);
    }
    // Slices: as large as shared memory allows (the histories are read once
    // for each), smaller while that leaves SMs without work.
    int slice = kMaxSlice;
    while (slice > kMinSlice && rows * kb::ceil_div(vocab, slice) < 2 * kb::sm_count()) slice /= 2;
    static uint64_t done = 0;
    if (int st = allow_smem((const void*)penalize_kernel<T>, kMaxSlice * 6, done)) return st;
    const dim3 grid((unsigned)kb::ceil_div(vocab, slice), (unsigned)rows);
    return launch_after(penalize_kernel<T>, grid, (unsigned)kThreads, (size_t)slice * 6, stream, a, slice);
  });
}

}  // extern "C"
