// gradnorm.cu — the 2-norm of a list of gradients, and clipping by it.
//
//   norm = sqrt(sum_i g_i^2),   g_i <- g_i min(1, max_norm / (norm + 1e-6))
//
// Squares are formed and added in double: the square of any float is exact
// there, so no gradient overflows or vanishes before the norm does.  A block
// leaves one partial sum; whoever needs the norm adds the partial sums in
// their order (norm_of), so no atomic's order shows in the result.
#include "optim_common.cuh"

namespace dr {

bool valid_type(int type) { return type == DR_F32 || type == DR_BF16 || type == DR_F16; }

namespace {

struct GradEntry {
  void* data;
  int64_t n;
  unsigned first_chunk;
  int type;
};

// A launch carries its list as a parameter, which a captured graph keeps: no
// table in device memory that a replay would have to find unchanged.  Small
// lists use a small parameter block.
template <int CAP>
struct GradTable {
  GradEntry t[CAP];
  int count;
  unsigned chunks;
};
constexpr int kSmall = 64, kLarge = 1280;
static_assert(sizeof(GradTable<kLarge>) + 64 <= 32764, "kernel parameters");

// Partial sums per launch at most, whatever the device.
constexpr int kMaxParts = 2048;

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* base, int64_t n, int64_t at) {
  float x[kOptVec];
  const T* p = base + at;
  if (at + kOptVec <= n && ((uintptr_t)p & 15) == 0) load_vec(p, x);
  else load_some(p, (int)max((int64_t)0, min((int64_t)kOptVec, n - at)), x);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) s = __fma_rn((double)x[i], (double)x[i], s);
  return s;
}

template <int CAP>
__global__ void __launch_bounds__(kOptThreads) k_grad_norm_parts(const __grid_constant__ GradTable<CAP> tab,
                                                                 double* __restrict__ part) {
  double s = 0.0;
  for (unsigned c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const GradEntry& e = tab.t[tensor_of(tab.t, tab.count, c)];
    const int64_t at = (int64_t)(c - e.first_chunk) * kOptChunk + threadIdx.x * kOptVec;
    if (e.type == DR_F32) s += chunk_squares((const float*)e.data, e.n, at);
    else if (e.type == DR_BF16) s += chunk_squares((const __nv_bfloat16*)e.data, e.n, at);
    else s += chunk_squares((const __half*)e.data, e.n, at);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(kOptThreads) k_grad_norm_finish(const double* __restrict__ part, int count,
                                                                  float* __restrict__ norm) {
  const double s = norm_of(part, count);
  if (threadIdx.x == 0) *norm = (float)s;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(T* base, int64_t n, int64_t at, float c) {
  float x[kOptVec];
  T* p = base + at;
  const bool whole = at + kOptVec <= n && ((uintptr_t)p & 15) == 0;
  const int valid = (int)max((int64_t)0, min((int64_t)kOptVec, n - at));
  if (whole) load_vec(p, x);
  else load_some(p, valid, x);
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) x[i] = __fmul_rn(x[i], c);
  if (whole) store_vec(p, x);
  else store_some(p, valid, x);
}

template <int CAP>
__global__ void __launch_bounds__(kOptThreads) k_clip_scale(const __grid_constant__ GradTable<CAP> tab,
                                                            const double* __restrict__ part, int parts,
                                                            double max_norm, float* __restrict__ norm) {
  const double s = norm_of(part, parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)s;
  const float f = clip_factor(s, max_norm);
  if (f == 1.0f) return;
  for (unsigned c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const GradEntry& e = tab.t[tensor_of(tab.t, tab.count, c)];
    const int64_t at = (int64_t)(c - e.first_chunk) * kOptChunk + threadIdx.x * kOptVec;
    if (e.type == DR_F32) chunk_scale((float*)e.data, e.n, at, f);
    else if (e.type == DR_BF16) chunk_scale((__nv_bfloat16*)e.data, e.n, at, f);
    else chunk_scale((__half*)e.data, e.n, at, f);
  }
}

// Blocks of a launch over `chunks`: enough to fill the device, and few enough
// that adding their partial sums costs little.
unsigned list_blocks(const dr_ctx* ctx, unsigned chunks) {
  return std::max(1u, std::min(chunks, (unsigned)std::min(kMaxParts, ctx->num_sms * 8)));
}

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

// The next launch's part of a list, from *i on: at most CAP tensors with elements.
template <int CAP>
void fill(const dr_grad_tensor* g, int count, int* i, GradTable<CAP>* tab) {
  int64_t chunks = 0;
  tab->count = 0;
  for (; *i < count && tab->count < CAP; ++*i) {
    const dr_grad_tensor& t = g[*i];
    if (t.n == 0) continue;
    tab->t[tab->count++] = {t.data, t.n, (unsigned)chunks, t.type};
    chunks += opt_chunks(t.n);
  }
  tab->chunks = (unsigned)chunks;
}

template <int CAP>
dr_status launch_parts(dr_ctx* ctx, const dr_grad_tensor* g, int count, double* work, int* parts) {
  for (int i = 0; i < count;) {
    GradTable<CAP> tab;
    fill(g, count, &i, &tab);
    if (tab.count == 0) break;
    const unsigned blocks = list_blocks(ctx, tab.chunks);
    DR_TB(ctx);
    k_grad_norm_parts<CAP><<<blocks, kOptThreads, 0, ctx->stream>>>(tab, work + *parts);
    DR_LAUNCHED(ctx, "grad_norm_parts");
    *parts += (int)blocks;
  }
  return DR_OK;
}

template <int CAP>
dr_status launch_scale(dr_ctx* ctx, const dr_grad_tensor* g, int count, const double* work, int parts,
                       double max_norm, float* norm) {
  for (int i = 0; i < count;) {
    GradTable<CAP> tab;
    fill(g, count, &i, &tab);
    if (tab.count == 0) break;
    DR_TB(ctx);
    k_clip_scale<CAP><<<list_blocks(ctx, tab.chunks), kOptThreads, 0, ctx->stream>>>(tab, work, parts, max_norm, norm);
    DR_LAUNCHED(ctx, "clip_scale");
  }
  return DR_OK;
}

}  // namespace

dr_status grad_norm_finish(dr_ctx* ctx, const double* work, int parts, float* norm) {
  DR_TB(ctx);
  k_grad_norm_finish<<<1, kOptThreads, 0, ctx->stream>>>(work, parts, norm);
  DR_LAUNCHED(ctx, "grad_norm_finish");
  return DR_OK;
}

dr_status grad_norm_parts(dr_ctx* ctx, const dr_grad_tensor* grads, int count, double* work, int* parts) {
  *parts = 0;
  return count <= kSmall ? launch_parts<kSmall>(ctx, grads, count, work, parts)
                         : launch_parts<kLarge>(ctx, grads, count, work, parts);
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
  DR_REQUIRE(ctx, norm && work && ((uintptr_t)work & 7) == 0, "grad_norm: norm and an 8-byte aligned work are required");
  dr_status st = check_list(ctx, grads, count, "grad_norm");
  if (st != DR_OK) return st;
  int parts = 0;
  if ((st = grad_norm_parts(ctx, grads, count, (double*)work, &parts)) != DR_OK) return st;
  return grad_norm_finish(ctx, (const double*)work, parts, norm);
}

dr_status dr_clip_grad_norm(dr_ctx* ctx, const dr_grad_tensor* grads, int count, double max_norm, float* norm,
                            void* work) {
  DR_ENTER(ctx);
  DR_REQUIRE(ctx, norm && work && ((uintptr_t)work & 7) == 0,
             "clip_grad_norm: norm and an 8-byte aligned work are required");
  DR_REQUIRE(ctx, max_norm > 0.0 && max_norm < 1e300, "clip_grad_norm: max_norm must be positive and finite");
  dr_status st = check_list(ctx, grads, count, "clip_grad_norm");
  if (st != DR_OK) return st;
  int parts = 0;
  if ((st = grad_norm_parts(ctx, grads, count, (double*)work, &parts)) != DR_OK) return st;
  if (parts == 0) return grad_norm_finish(ctx, (const double*)work, 0, norm);  // nothing to scale
  return count <= kSmall ? launch_scale<kSmall>(ctx, grads, count, (const double*)work, parts, max_norm, norm)
                         : launch_scale<kLarge>(ctx, grads, count, (const double*)work, parts, max_norm, norm);
}

}  // extern "C"
