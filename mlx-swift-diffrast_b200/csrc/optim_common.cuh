// optim_common.cuh — what the many-tensor optimizer kernels share: element
// types, the split of a list of tensors into chunks, and the gradient norm's
// partial sums.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <utility>

#include "common.cuh"

namespace dr {

constexpr int kOptThreads = 256;
constexpr int kOptVec = 8;                          // consecutive elements of one thread
constexpr int kOptChunk = kOptThreads * kOptVec;    // elements a block handles at once

// Elements of one thread, widened to float.  The 16-bit types widen exactly.
template <typename T>
__device__ __forceinline__ float widen(T x);
template <>
__device__ __forceinline__ float widen(float x) { return x; }
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// Rounding to nearest even: parameters and gradients are what a user stores in
// 16 bits; everything in between stays in float.
template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

// kOptVec consecutive elements as they lie in memory, at an address that is a
// multiple of their size: one access of 16 or 32 bytes.
template <typename T>
struct Words {
  static constexpr int kCount = kOptVec * sizeof(T) / 16;
  static_assert(kCount == 1 || kCount == 2, "16 or 32 bytes");
  uint4 w[kCount];
};

template <typename T>
__device__ __forceinline__ Words<T> load_words(const T* p) {
  Words<T> x;
  if constexpr (Words<T>::kCount == 2)
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(x.w[0].x), "=r"(x.w[0].y), "=r"(x.w[0].z), "=r"(x.w[0].w), "=r"(x.w[1].x), "=r"(x.w[1].y),
                   "=r"(x.w[1].z), "=r"(x.w[1].w)
                 : "l"(p)
                 : "memory");
  else
    x.w[0] = *reinterpret_cast<const uint4*>(p);
  return x;
}

template <typename T>
__device__ __forceinline__ void widen_words(const Words<T>& words, float (&x)[kOptVec]) {
  const T* e = reinterpret_cast<const T*>(words.w);
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) x[i] = widen(e[i]);
}

template <typename T>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[kOptVec]) {
  widen_words(load_words(p), x);
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[kOptVec]) {
  Words<T> words;
  T* e = reinterpret_cast<T*>(words.w);
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) e[i] = narrow<T>(x[i]);
  if constexpr (Words<T>::kCount == 2)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(words.w[0].x),
                 "r"(words.w[0].y), "r"(words.w[0].z), "r"(words.w[0].w), "r"(words.w[1].x), "r"(words.w[1].y),
                 "r"(words.w[1].z), "r"(words.w[1].w)
                 : "memory");
  else
    *reinterpret_cast<uint4*>(p) = words.w[0];
}

template <typename T>
__host__ __device__ __forceinline__ bool vector_aligned(const T* p) {
  return (uintptr_t)p % (kOptVec * sizeof(T)) == 0;
}

// load_words at any address of T's alignment.
template <typename T>
__device__ __forceinline__ Words<T> gather_words(const T* p) {
  Words<T> x;
  T* e = reinterpret_cast<T*>(x.w);
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) e[i] = p[i];
  return x;
}

// `valid` (0 .. kOptVec) elements at any address of T's alignment; the others are 0.
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int valid, float (&x)[kOptVec]) {
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) x[i] = i < valid ? widen(p[i]) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store_some(T* p, int valid, const float (&x)[kOptVec]) {
#pragma unroll
  for (int i = 0; i < kOptVec; ++i)
    if (i < valid) p[i] = narrow<T>(x[i]);
}

// A list holds fewer chunks than an int does (4e12 elements), checked at the entries.
constexpr int64_t kOptMostElements = (int64_t)INT32_MAX * kOptChunk;
inline int64_t opt_chunks(int64_t n) { return (n + kOptChunk - 1) / kOptChunk; }

// The tensor of a list that chunk c belongs to: the last whose first chunk is
// <= c.  Tensors without elements are not in the list, so it is the one.
__device__ __forceinline__ int tensor_of(const unsigned* first, int count, unsigned c) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A block takes chunks b, b + gridDim, ... in rounds of one to a warp: each
// warp looks one chunk of the next round up and leaves what it found in shared
// memory.  The list lies in the parameter bank, where each tensor's row is a
// miss at its first use on a multiprocessor; eight warps wait for eight of them
// at once.  Three rounds are kept: one being looked up, one in use, and one that
// a slower warp may still be in.
constexpr int kOptWarps = kOptThreads / 32;
constexpr int kRounds = 3;

// Sum over the block in a fixed order; every thread gets it.
template <int THREADS = kOptThreads>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s_warp[THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();  // s_warp may still be read from an earlier call
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) s += s_warp[i];
  return s;
}

// The norm that `count` partial sums of squares give: the same value in every
// block that asks, whatever its place.
template <int THREADS = kOptThreads>
__device__ __forceinline__ double norm_of(const double* part, int count) {
  // Added in the same order whatever the block's size: by the first kOptThreads threads.
  double s = 0.0;
  if (threadIdx.x < kOptThreads)
    for (int i = threadIdx.x; i < count; i += kOptThreads) s += part[i];
  return sqrt(block_sum<THREADS>(s));
}

// min(1, max_norm / (norm + 1e-6)); a NaN stays one.
__device__ __forceinline__ float clip_factor(double norm, double max_norm) {
  const double c = max_norm / (norm + 1e-6);
  return c >= 1.0 ? 1.0f : (float)c;
}

// Launches `kernel`, which calls after_previous(), while the launch before it on
// the stream is still running.
template <typename... Params, typename... Args>
inline cudaError_t launch_early(cudaStream_t stream, unsigned blocks, int threads, void (*kernel)(Params...),
                                Args&&... args) {
  cudaLaunchAttribute early = {};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3((unsigned)threads);
  config.stream = stream;
  config.attrs = &early;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}
// In a kernel that the next one on the stream may overlap: it may start.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// In a kernel launched early: what the launch before it wrote is there.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

bool valid_type(int type);
// Launches the partial sums of squares of a list; *parts of them lie in `work`.
// With `norm`, for a list of one round of one block: it forms the norm itself,
// and with max_norm > 0 clips the gradients by it.
dr_status grad_norm_parts(dr_ctx* ctx, const dr_grad_tensor* grads, int count, double* work, int* parts, float* norm,
                          double max_norm);
// *norm = the norm that the partial sums give.
dr_status grad_norm_finish(dr_ctx* ctx, const double* work, int parts, float* norm);

}  // namespace dr
