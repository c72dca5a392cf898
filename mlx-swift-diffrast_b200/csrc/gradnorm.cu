// gradnorm.cu — the 2-norm of a list of gradients, and clipping by it.
//
//   norm = sqrt(sum_i g_i^2),   g_i <- g_i min(1, max_norm / (norm + 1e-6))
//
// Squares are formed and added in double: the square of any float is exact
// there, so no gradient overflows or vanishes before the norm does.  A block
// leaves one partial sum; whoever needs the norm adds the partial sums in
// their order (norm_of), so no atomic's order shows in the result.  Bound by
// memory: the 127 MB of the million-triangle soup's gradients take 22 us on the
// device (5.7 TB/s, 20 of them the pass itself), 24.6 with their launches; the
// double arithmetic costs 0.3 of them.  Clipping reads them again, from L2 where
// they fit it.
#include "optim_common.cuh"

namespace dr {

bool valid_type(int type) { return type == DR_F32 || type == DR_BF16 || type == DR_F16; }

namespace {

struct GradEntry {
  void* data;
  int64_t n;
  int type;
};

// A launch carries its list as a parameter, which a captured graph keeps: no
// table in device memory that a replay would have to find unchanged.  The block
// comes in three sizes: the host copies all of it at each launch, and 28 KB of
// it cost 2 us where 2 KB cost next to nothing (the norm of two small tensors,
// 13.5 us with the small block at the time, took 15.7 with the large one).
template <int CAP>
struct GradTable {
  GradEntry t[CAP];
  unsigned first[CAP];  // each tensor's first chunk
  int count;
  unsigned chunks;
};
constexpr int kSmall = 64, kMedium = 250, kLarge = 1000;
static_assert(sizeof(GradTable<kLarge>) + 64 <= 32764, "kernel parameters");

// Partial sums per launch at most, whatever the device.
constexpr int kMaxParts = 2048;

// A chunk: where it begins, how many elements of its tensor it holds.
struct GradSlot {
  char* data;
  int valid, type;
};

template <int CAP>
__device__ __forceinline__ void look_up(const GradTable<CAP>& tab, unsigned c, GradSlot& slot) {
  if (c >= tab.chunks) return;
  const int i = tensor_of(tab.first, tab.count, c);
  const GradEntry& e = tab.t[i];
  const int64_t at = (int64_t)(c - tab.first[i]) * kOptChunk;
  if (threadIdx.x % 32 == 0)
    slot = {(char*)e.data + at * (e.type == DR_F32 ? 4 : 2), (int)min((int64_t)kOptChunk, e.n - at), e.type};
}

// One thread's elements of a chunk, of any type, as they lie in memory.
struct Fetched {
  Words<float> w;  // a 16-bit type's elements are in the first half
  int type;        // -1: nothing here, or summed already
};

template <typename T>
__device__ __forceinline__ double squares(const float (&x)[kOptVec]) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) s = __fma_rn((double)x[i], (double)x[i], s);
  return s;
}

template <typename T>
__device__ __forceinline__ double squares_of(const T* p, int valid) {
  float x[kOptVec];
  load_some(p, valid, x);
  return squares<T>(x);
}

// Fetches the thread's elements of a chunk, or, where they are not whole, adds
// their squares to s.
__device__ __forceinline__ void fetch(const GradSlot& e, Fetched& x, double& s) {
  const int bytes = e.type == DR_F32 ? 4 : 2, valid = e.valid - (int)threadIdx.x * kOptVec;
  const char* p = e.data + threadIdx.x * kOptVec * bytes;
  x.type = -1;
  if (valid >= kOptVec && ((uintptr_t)p & (kOptVec * bytes - 1)) == 0) {
    x.type = e.type;
    if (e.type == DR_F32) x.w = load_words((const float*)p);
    else x.w.w[0] = load_words((const __half*)p).w[0];
  } else if (valid > 0) {
    if (e.type == DR_F32) s += squares_of((const float*)p, valid);
    else if (e.type == DR_BF16) s += squares_of((const __nv_bfloat16*)p, valid);
    else s += squares_of((const __half*)p, valid);
  }
}

template <typename T>
__device__ __forceinline__ double squares_of(const Fetched& x) {
  Words<T> w;
#pragma unroll
  for (int i = 0; i < Words<T>::kCount; ++i) w.w[i] = x.w.w[i];
  float f[kOptVec];
  widen_words(w, f);
  return squares<T>(f);
}

template <typename T>
__device__ __forceinline__ void scale_vec(const GradSlot& e, float f) {
  const int valid = min(kOptVec, e.valid - (int)threadIdx.x * kOptVec);
  if (valid <= 0) return;
  float x[kOptVec];
  T* p = (T*)e.data + threadIdx.x * kOptVec;
  const bool whole = valid == kOptVec && vector_aligned(p);
  if (whole) load_vec(p, x);
  else load_some(p, valid, x);
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) x[i] = __fmul_rn(x[i], f);
  if (whole) store_vec(p, x);
  else store_some(p, valid, x);
}

__device__ __forceinline__ void scale_chunk(const GradSlot& e, float f) {
  if (e.type == DR_F32) scale_vec<float>(e, f);
  else if (e.type == DR_BF16) scale_vec<__nv_bfloat16>(e, f);
  else scale_vec<__half>(e, f);
}

// A thread's loads of kAhead chunks are under way together: 22.4 us for the soup
// with four; 25 with two (and twice the blocks), 31 with eight.
constexpr int kAhead = 4;
static_assert(kOptWarps % kAhead == 0, "rounds of whole batches");

template <int CAP>
__global__ void __launch_bounds__(kOptThreads) k_grad_norm_parts(const __grid_constant__ GradTable<CAP> tab,
                                                                 double* __restrict__ part,
                                                                 float* __restrict__ norm, double max_norm) {
  __shared__ GradSlot s_slots[kRounds][kOptWarps];
  const unsigned warp = threadIdx.x / 32;
  double s = 0.0;
  unsigned c = blockIdx.x;
  look_up(tab, c + warp * gridDim.x, s_slots[0][warp]);
  __syncthreads();
  for (int round = 0; c < tab.chunks; round = round + 1 == kRounds ? 0 : round + 1) {
#pragma unroll 1
    for (int b = 0; b < kOptWarps && c < tab.chunks; b += kAhead) {
      Fetched x[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        x[a].type = -1;
        if (c < tab.chunks) fetch(s_slots[round][b + a], x[a], s);
        c += gridDim.x;
      }
      if (b == 0)
        look_up(tab, c + (kOptWarps - kAhead + warp) * gridDim.x, s_slots[round + 1 == kRounds ? 0 : round + 1][warp]);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        if (x[a].type == DR_F32) s += squares_of<float>(x[a]);
        else if (x[a].type == DR_BF16) s += squares_of<__nv_bfloat16>(x[a]);
        else if (x[a].type == DR_F16) s += squares_of<__half>(x[a]);
      }
    }
    __syncthreads();
  }
  let_next_start();
  s = block_sum(s);
  if (!norm) {
    if (threadIdx.x == 0) part[blockIdx.x] = s;
    return;
  }
  // The only block of the only launch: the list is one round, whose slots are still there.
  s = sqrt(s);
  if (threadIdx.x == 0) *norm = (float)s;
  const float f = max_norm > 0.0 ? clip_factor(s, max_norm) : 1.0f;
  if (f == 1.0f) return;
  for (unsigned b = 0; b < tab.chunks; ++b) scale_chunk(s_slots[0][b], f);
}

// `part` of the two kernels below is written by the launch before them while
// they are resident already: a plain pointer, so that its loads are ordinary
// (coherent) ones, which the wait's memory clobber holds behind it.
__global__ void __launch_bounds__(kOptThreads) k_grad_norm_finish(const double* part, int count, float* norm) {
  after_previous();
  const double s = norm_of(part, count);
  if (threadIdx.x == 0) *norm = (float)s;
}

template <int CAP>
__global__ void __launch_bounds__(kOptThreads) k_clip_scale(const __grid_constant__ GradTable<CAP> tab,
                                                            const double* part, int parts, double max_norm,
                                                            float* norm) {
  __shared__ GradSlot s_slots[kRounds][kOptWarps];
  const unsigned warp = threadIdx.x / 32;
  unsigned c = blockIdx.x;
  look_up(tab, c + warp * gridDim.x, s_slots[0][warp]);
  after_previous();
  const double s = norm_of(part, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
  const float f = clip_factor(s, max_norm);
  if (f == 1.0f) return;
  __syncthreads();
  for (int round = 0; c < tab.chunks; round = round + 1 == kRounds ? 0 : round + 1) {
    look_up(tab, c + (kOptWarps + warp) * gridDim.x, s_slots[round + 1 == kRounds ? 0 : round + 1][warp]);
#pragma unroll 1
    for (int b = 0; b < kOptWarps && c < tab.chunks; ++b, c += gridDim.x) scale_chunk(s_slots[round][b], f);
    __syncthreads();
  }
}

// Blocks of a launch at most: enough to fill the device, and few enough that
// adding their partial sums costs little.
unsigned most_blocks(const dr_ctx* ctx) { return (unsigned)std::min(kMaxParts, ctx->num_sms * 4); }

dr_status check_list(dr_ctx* ctx, const dr_grad_tensor* g, int count, const char* what) {
  DR_REQUIRE(ctx, count >= 0 && (count == 0 || g), "%s: null list or count < 0", what);
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    DR_REQUIRE(ctx, g[i].n >= 0 && (g[i].n == 0 || g[i].data), "%s: tensor %d has a null pointer or n < 0", what, i);
    DR_REQUIRE(ctx, valid_type(g[i].type), "%s: tensor %d has an unknown type %d", what, i, g[i].type);
    DR_REQUIRE(ctx, g[i].n < kOptMostElements && (chunks += opt_chunks(g[i].n)) < INT32_MAX, "%s: too many elements", what);
    DR_REQUIRE(ctx, (uintptr_t)g[i].data % (g[i].type == DR_F32 ? 4 : 2) == 0, "%s: tensor %d is misaligned", what, i);
  }
  return DR_OK;
}

// A list whose norm one block forms, and by which it scales it, in one launch.
bool is_small(const dr_grad_tensor* g, int count) {
  static_assert(DR_GRAD_NORM_SMALL_COUNT == kSmall && DR_GRAD_NORM_SMALL_ELEMENTS == kOptWarps * kOptChunk, "as stated");
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) chunks += opt_chunks(g[i].n);
  return chunks <= kOptWarps && count <= kSmall;
}

// The next launch's part of a list, from *i on: at most CAP tensors with elements.
template <int CAP>
void fill(const dr_grad_tensor* g, int count, int* i, GradTable<CAP>* tab) {
  int64_t chunks = 0;
  tab->count = 0;
  for (; *i < count && tab->count < CAP; ++*i) {
    const dr_grad_tensor& t = g[*i];
    if (t.n == 0) continue;
    tab->first[tab->count] = (unsigned)chunks;
    tab->t[tab->count++] = {t.data, t.n, t.type};
    chunks += opt_chunks(t.n);
  }
  tab->chunks = (unsigned)chunks;
}

template <int CAP>
dr_status launch_parts(dr_ctx* ctx, const dr_grad_tensor* g, int count, double* work, int* parts, float* norm,
                       double max_norm) {
  for (int i = 0; i < count;) {
    GradTable<CAP> tab;
    fill(g, count, &i, &tab);
    if (tab.count == 0) break;
    const unsigned blocks = norm ? 1 : std::min(tab.chunks, most_blocks(ctx));
    DR_TB(ctx);
    k_grad_norm_parts<CAP><<<blocks, kOptThreads, 0, ctx->stream>>>(tab, norm ? nullptr : work + *parts, norm,
                                                                       max_norm);
    DR_LAUNCHED(ctx, "grad_norm_parts");
    *parts += (int)blocks;
  }
  return DR_OK;
}

template <int CAP>
dr_status launch_scale(dr_ctx* ctx, const dr_grad_tensor* g, int count, const double* work, int parts,
                       double max_norm, float* norm) {
  bool first = true;  // the launch behind the norm's
  for (int i = 0; i < count;) {
    GradTable<CAP> tab;
    fill(g, count, &i, &tab);
    if (tab.count == 0) break;
    const unsigned blocks = std::min(tab.chunks, 2 * most_blocks(ctx));
    DR_TB(ctx);
    if (first)
      DR_CUDA(ctx, launch_early(ctx->stream, blocks, kOptThreads, k_clip_scale<CAP>, tab, work, parts, max_norm, norm), "clip_scale");
    else
      k_clip_scale<CAP><<<blocks, kOptThreads, 0, ctx->stream>>>(tab, work, parts, max_norm, norm);
    first = false;
    DR_LAUNCHED(ctx, "clip_scale");
  }
  return DR_OK;
}

}  // namespace

dr_status grad_norm_finish(dr_ctx* ctx, const double* work, int parts, float* norm) {
  DR_TB(ctx);
  DR_CUDA(ctx, launch_early(ctx->stream, 1, kOptThreads, k_grad_norm_finish, work, parts, norm), "grad_norm_finish");
  DR_LAUNCHED(ctx, "grad_norm_finish");
  return DR_OK;
}

dr_status grad_norm_parts(dr_ctx* ctx, const dr_grad_tensor* grads, int count, double* work, int* parts,
                          float* norm, double max_norm) {
  *parts = 0;
  return count <= kSmall    ? launch_parts<kSmall>(ctx, grads, count, work, parts, norm, max_norm)
         : count <= kMedium ? launch_parts<kMedium>(ctx, grads, count, work, parts, norm, max_norm)
                            : launch_parts<kLarge>(ctx, grads, count, work, parts, norm, max_norm);
}

}  // namespace dr

using namespace dr;

extern "C" {

size_t dr_grad_norm_work_bytes(const dr_ctx* ctx, int count) {
  if (!ctx || count < 0) return 0;
  return sizeof(double) * (size_t)kMaxParts * (size_t)(count / kLarge + 1);
}

dr_status dr_grad_norm(dr_ctx* ctx, const dr_grad_tensor* grads, int count, float* norm, void* work) {
  DR_ENTER(ctx);
  DR_REQUIRE(ctx, norm && (uintptr_t)norm % 4 == 0, "grad_norm: a 4-byte aligned norm is required");
  dr_status st = check_list(ctx, grads, count, "grad_norm");
  if (st != DR_OK) return st;
  const bool small = is_small(grads, count);
  DR_REQUIRE(ctx, small || (work && ((uintptr_t)work & 7) == 0), "grad_norm: an 8-byte aligned work is required");
  int parts = 0;
  if ((st = grad_norm_parts(ctx, grads, count, (double*)work, &parts, small ? norm : nullptr, 0.0)) != DR_OK) return st;
  return small && parts ? DR_OK : grad_norm_finish(ctx, (const double*)work, parts, norm);
}

dr_status dr_clip_grad_norm(dr_ctx* ctx, const dr_grad_tensor* grads, int count, double max_norm, float* norm,
                            void* work) {
  DR_ENTER(ctx);
  DR_REQUIRE(ctx, norm && (uintptr_t)norm % 4 == 0, "clip_grad_norm: a 4-byte aligned norm is required");
  DR_REQUIRE(ctx, max_norm > 0.0 && max_norm < 1e300, "clip_grad_norm: max_norm must be positive and finite");
  dr_status st = check_list(ctx, grads, count, "clip_grad_norm");
  if (st != DR_OK) return st;
  const bool small = is_small(grads, count);
  DR_REQUIRE(ctx, small || (work && ((uintptr_t)work & 7) == 0), "clip_grad_norm: an 8-byte aligned work is required");
  int parts = 0;
  if ((st = grad_norm_parts(ctx, grads, count, (double*)work, &parts, small ? norm : nullptr, max_norm)) != DR_OK)
    return st;
  if (small && parts) return DR_OK;
  if (parts == 0) return grad_norm_finish(ctx, (const double*)work, 0, norm);  // nothing to scale
  const double* part = (const double*)work;
  return count <= kSmall    ? launch_scale<kSmall>(ctx, grads, count, part, parts, max_norm, norm)
         : count <= kMedium ? launch_scale<kMedium>(ctx, grads, count, part, parts, max_norm, norm)
                            : launch_scale<kLarge>(ctx, grads, count, part, parts, max_norm, norm);
}

}  // extern "C"
