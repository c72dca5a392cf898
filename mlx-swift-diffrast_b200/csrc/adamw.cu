// adamw.cu — the AdamW step over many tensors, with states in 32 or in 8 bits.
//
//   g = coef grad;  m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every operation on elements is a separate IEEE round-to-nearest step in
// float, so moments, states and (32-bit states) parameters are the same bit for
// bit as an unfused evaluation; with 8-bit states the parameter's quotient is a
// product with the hardware's reciprocal.  The factors in t are formed in double
// on the device from each tensor's clock (t, b1^t, b2^t), which the step itself
// advances: nothing in a captured step is fixed to the t of its capture.
//
// 32-bit states are bound by memory: 28 bytes an element in fp32, 1150 to 1180 us
// for sixteen 2048^2x4 textures (268 M elements, 7.5 GB), 6.4 to 6.5 TB/s.  8-bit
// states move 16 (fp32) or 10 bytes (16-bit types) and are bound by issue: 355
// instructions for a block of 256 elements, most of them the exact roundings, the
// root, the random bits and the codes; the same textures in fp16 take 475 us on the
// device, 5.7 TB/s, and up to 555 in a long run, at the power limit.
#include <new>
#include <type_traits>

#include "optim_common.cuh"

namespace dr {
namespace {

struct AdamEntry {
  void* param;
  const void* grad;
  float* master;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int64_t n;
  double lr_ratio, weight_decay;
  uint32_t seed;
  int aligned;  // kVectors: weights, gradient and 32-bit states may be accessed in vectors; kCodes: 8-bit states
};

constexpr int kVectors = 1, kCodes = 2;

// beta1, beta2, what they leave of 1, and 1.
struct Betas {
  float b1, b2, one_m_b1, one_m_b2, one;
};

struct AdamHyper {
  double lr, beta1, beta2, max_norm;
  const float* lr_device;
  float eps;
  const double* part;  // partial sums of the norm's squares; nullptr without clipping
  int parts;
  float* norm;
  uint32_t* ticket;
  Betas betas;
};

// The list is a kernel parameter, in two sizes as gradnorm.cu's: when the second
// was brought in, a step of two tensors took 8.2 us with the small block and 11
// with the large one (now 7.9 with the small one, 5.8 on the device).
template <int CAP>
struct AdamTable {
  AdamEntry t[CAP];
  double* clock[CAP];   // apart from the rows: the last block reads them all (1.6 us less for 30 tensors and more)
  unsigned first[CAP];  // each tensor's first chunk
  AdamHyper h;
  int count;
  unsigned chunks;
};
constexpr int kSmall = 32, kLarge = 300;
static_assert(sizeof(AdamTable<kSmall>) <= 4096 && sizeof(AdamTable<kLarge>) <= 32764, "kernel parameters");

// What a step's elements share: for tensor e at its step t.
struct AdamFactors {
  float decay;     // 1 - lr wd
  float step;      // lr / (1 - b1^t)
  float inv_sqrt;  // 1 / sqrt(1 - b2^t)
  uint32_t key;    // of the random bits
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  // Two rounds of xor-shift and multiplication by an odd number (the first 32
  // bits behind the point of sqrt 2 and sqrt 3): each input bit flips each
  // output bit with probability 0.500 +- 0.004.
  x = (x ^ (x >> 16)) * 0x6A09E667u;
  x = (x ^ (x >> 15)) * 0xBB67AE85u;
  return x ^ (x >> 16);
}

__device__ __forceinline__ AdamFactors factors_of(const AdamEntry& e, const double* clock, const AdamHyper& h) {
  const double t = clock[0] + 1.0, b1t = clock[1] * h.beta1, b2t = clock[2] * h.beta2;
  const double lr = (h.lr_device ? (double)*h.lr_device : h.lr) * e.lr_ratio;
  AdamFactors f;
  f.decay = (float)(1.0 - lr * e.weight_decay);
  f.step = (float)(lr / (1.0 - b1t));
  f.inv_sqrt = (float)rsqrt(1.0 - b2t);
  f.key = mix(mix((uint32_t)(long long)t) ^ e.seed);
  return f;
}

// 8-bit states: a warp holds a block of 256 elements, eight to a lane.
constexpr int kStateBlock = 256;
static_assert(kStateBlock == 32 * kOptVec, "one block of states to a warp");

// An 8-bit step's block has 16 warps, and its chunk kBlocks8 blocks of states for
// each, one in each part of kPart8 elements.
constexpr int kThreads8 = 512, kWarps8 = kThreads8 / 32;
constexpr int kBlocks8 = 2;
constexpr int kPart8 = kThreads8 * kOptVec, kChunk8 = kPart8 * kBlocks8;

// A chunk: its tensor's factors, and where it begins.
struct AdamSlot {
  AdamFactors f;
  const void* weights;  // that are read: the master's where there are some
  void* param;
  const void* grad;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  uint32_t block;  // of states, from the tensor's first on
  int valid;       // elements
  int aligned;
  int tensor;
};

// Chunk c into `slot`; `before`: what this warp looked up last (or nullptr).
template <typename P, typename G, bool MASTER, int BITS, int CAP>
__device__ __forceinline__ void look_up(const AdamTable<CAP>& tab, unsigned c, AdamSlot& slot,
                                        const AdamSlot* before) {
  if (c >= tab.chunks) return;
  const int i = tensor_of(tab.first, tab.count, c);
  const AdamEntry& e = tab.t[i];
  constexpr int kChunk = BITS == 32 ? kOptChunk : kChunk8;
  const int64_t at = (int64_t)(c - tab.first[i]) * kChunk;
  AdamFactors f;
  if (before && before->tensor == i) f = before->f;
  else f = factors_of(e, tab.clock[i], tab.h);
  if (threadIdx.x % 32 != 0) return;
  constexpr int kState = BITS == 32 ? 4 : 1;
  slot.f = f;
  slot.tensor = i;
  slot.weights = MASTER ? (const void*)(e.master + at) : (const P*)e.param + at;
  slot.param = (P*)e.param + at;
  slot.grad = (const G*)e.grad + at;
  slot.m = (char*)e.m + at * kState;
  slot.v = (char*)e.v + at * kState;
  slot.block = (uint32_t)(at / kStateBlock);
  if (BITS == 8) {
    slot.m_scale = e.m_scale + at / kStateBlock;
    slot.v_scale = e.v_scale + at / kStateBlock;
  }
  slot.valid = (int)min((int64_t)kChunk, e.n - at);
  slot.aligned = e.aligned;
}

__device__ __forceinline__ float next_m(const Betas& b, float m, float g) {
  return __fadd_rn(__fmul_rn(m, b.b1), __fmul_rn(g, b.one_m_b1));
}
__device__ __forceinline__ float next_v(const Betas& b, float v, float g) {
  return __fadd_rn(__fmul_rn(v, b.b2), __fmul_rn(__fmul_rn(g, g), b.one_m_b2));
}
__device__ __forceinline__ float next_p(const AdamFactors& f, float eps, float p, float m, float r) {
  const float denom = __fadd_rn(__fmul_rn(r, f.inv_sqrt), eps);
  return __fsub_rn(__fmul_rn(p, f.decay), __fdiv_rn(__fmul_rn(m, f.step), denom));
}

// One thread's kOptVec elements, loaded and stored whole where they are inside
// the tensor and every pointer is aligned, else one by one.
template <typename T>
__device__ __forceinline__ void load_n(const T* p, bool whole, int valid, float (&x)[kOptVec]) {
  if (whole) load_vec(p, x);
  else load_some(p, valid, x);
}
template <typename T>
__device__ __forceinline__ void store_n(T* p, bool whole, int valid, const float (&x)[kOptVec]) {
  if (whole) store_vec(p, x);
  else store_some(p, valid, x);
}

// 32-bit states: one thread's elements of a chunk.
template <typename P, typename G, bool MASTER>
__device__ __forceinline__ void update32(const AdamSlot& e, const Betas& b, float eps, float coef) {
  const unsigned at = threadIdx.x * kOptVec;
  const int valid = min(kOptVec, e.valid - (int)at);
  if (valid <= 0) return;
  P* p = (P*)e.param + at;
  const G* g = (const G*)e.grad + at;
  float* w = (float*)e.weights + at;
  float *m = (float*)e.m + at, *v = (float*)e.v + at;
  const bool whole = e.aligned && valid == kOptVec;
  float xp[kOptVec], xg[kOptVec], xm[kOptVec], xv[kOptVec];
  if (MASTER) load_n(w, whole, valid, xp);
  else load_n(p, whole, valid, xp);
  load_n(g, whole, valid, xg);
  load_n(m, whole, valid, xm);
  load_n(v, whole, valid, xv);
  const AdamFactors f = e.f;
#pragma unroll
  for (int i = 0; i < kOptVec; ++i) {
    const float gi = __fmul_rn(xg[i], coef);
    xm[i] = next_m(b, xm[i], gi);
    xv[i] = next_v(b, xv[i], gi);
    xp[i] = next_p(f, eps, xp[i], xm[i], __fsqrt_rn(xv[i]));
  }
  store_n(m, whole, valid, xm);
  store_n(v, whole, valid, xv);
  if (MASTER) store_n(w, whole, valid, xp);
  store_n(p, whole, valid, xp);
}

constexpr float kMaxCode = 448.0f;  // e4m3's largest

__device__ __forceinline__ void codes_to_float(uint2 c, float (&x)[kOptVec]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned short two = (unsigned short)((i < 2 ? c.x : c.y) >> (16 * (i & 1)));
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));  // exact
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint2 float_to_codes(const float (&x)[kOptVec]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned short lo, hi;  // saturating at +-448, to nearest even; a pair's first element in the low byte
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * i + 1]), "f"(x[4 * i]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * i + 3]), "f"(x[4 * i + 2]));
    w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// Two floats in a register pair: one instruction for both, each rounded as
// the single one is (fp16 textures: 547 us with them, 594 with single ones).
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float x, float y) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two both(float x) { return two(x, x); }
__device__ __forceinline__ float2 apart(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// The hardware's approximations, within one or two units in the last place.
__device__ __forceinline__ float rsqrt_fast(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float x, float y, float z) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// -sqrt(v), rounded to nearest, of nv = -v: with y = 1/sqrt(v) nearly, t = -v y
// is nearly -sqrt(v), t^2 - v its exact residual (one fused operation), and
// (t^2 - v) y / 2 what it is off by (Newton's step for t^2 = v; Markstein's
// argument for why its rounding is the right one).  Equal to the correctly
// rounded root for every float of the exponents from 2^-97 to 2^103; below 2^-100
// the residual loses bits, and v below 2^-126 counts as (nearly) 0.
__device__ __forceinline__ Two neg_sqrt(Two nv) {
  const float2 x = apart(nv);
  const Two y = two(rsqrt_fast(fmaxf(fabsf(x.x), 0x1p-126f)), rsqrt_fast(fmaxf(fabsf(x.y), 0x1p-126f)));
  const Two t = nv * y;
  return fma2(fma2(t, t, nv), y * both(0.5f), t);
}

// Scale of a block from its largest magnitude, and the factor 448 / (largest),
// rounded to nearest, that takes values to codes.  Below 2^-100 a block is zero; a
// value that is not finite makes it NaN.
__device__ __forceinline__ void scale_of(float top, float& scale, float& inv) {
  // The quotient by a reciprocal and its residual, as for the root; all times 2^-20, for the reciprocal of a large one.
  const float t = __fmul_rn(fmaxf(top, 0x1p-100f), 0x1p-20f), k = -kMaxCode * 0x1p-20f;
  const float y = rcp_fast(-t), q = __fmul_rn(k, y);
  inv = __fmaf_rn(__fmaf_rn(q, t, k), y, q);
  scale = __fmaf_rn(top, 1.0f / kMaxCode, __fsub_rn(top, top));  // top - top: 0, or NaN for what is not finite
  if (top < 0x1p-100f) scale = inv = 0.0f;
}

// The code of a value, given its negative (or +0) and z = 2^-120 (value / scale):
// e4m3's grid is that of z's bits above the lowest 20, its small evenly spaced
// values lying where float's are.  The low bits and the random ones (16 of them
// and half of their last one's worth) carry into the last kept bit with the
// probability of z's distance from the lower neighbour.  What is not 0 becomes
// code 1 at least; the largest, within two of z's last units of 448's, cannot be
// carried above 0x7E by less than 2^20 - 7.  The code is in the highest byte,
// the others are what is cut off.  HALF: which 16 bits of `word`.
template <int HALF>
__device__ __forceinline__ uint32_t round_stochastic(float z, float neg, uint32_t word) {
  // Signed: a z of -0 counts as less than 0.
  const uint32_t w = (uint32_t)max(__float_as_int(z), (int)min(__float_as_uint(neg), 1u << 20));
  // 2^4 (16 bits16 + 8): bytes 0x80, bits16's low and high one, 0.
  return (w << 4) + __byte_perm(word, 0x80u, HALF ? 0x5324 : 0x5104);
}
// The highest bytes of four words.
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

constexpr uint32_t kGolden = 0x9E3779B9u;

// One thread's elements of a block of states as they lie in memory.  W: the type
// of the weights that are read, the master's where there are some.
template <typename W, typename G>
struct Fetched {
  Words<W> w;
  Words<G> g;
  uint2 m, r;
  float m_scale, r_scale;
};

template <typename W, typename G>
__device__ __forceinline__ void fetch(const AdamSlot& e, int part, Fetched<W, G>& x) {
  const unsigned at = part * kPart8 + threadIdx.x * kOptVec, block = part * kWarps8 + threadIdx.x / 32;
  if (e.aligned & kVectors) {
    x.w = load_words((const W*)e.weights + at);
    x.g = load_words((const G*)e.grad + at);
  } else {
    x.w = gather_words((const W*)e.weights + at);
    x.g = gather_words((const G*)e.grad + at);
  }
  x.m = *reinterpret_cast<const uint2*>((const uint8_t*)e.m + at);
  x.r = *reinterpret_cast<const uint2*>((const uint8_t*)e.v + at);
  x.m_scale = e.m_scale[block];
  x.r_scale = e.v_scale[block];
}

// NB blocks of states of a chunk, from part `first` on, one thread's elements of
// each; fetched before where WHOLE.  All lanes of a warp, which hold one block
// of each part, come here with the same WHOLE.
template <bool WHOLE, int NB, typename P, typename G, bool MASTER, typename F>
__device__ __forceinline__ void update8(const AdamSlot& e, const Betas& b, float eps, float coef, const F* in,
                                        int first) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  float xm[NB][kOptVec], xr[NB][kOptVec];
  float m_top[NB], r_top[NB];
  const Two kc = both(coef);
  const Two kb1 = both(b.b1), kg1 = both(b.one_m_b1), nb2 = both(-b.b2), ng2 = both(-b.one_m_b2);
  // A sum of two products is a fused operation with a 1 that the compiler does
  // not know: it would make a packed product and sum one, with one rounding.
  const Two one = both(b.one);
  const Two ki = both(-e.f.inv_sqrt), ke = both(eps), ks = both(-e.f.step), kd = both(e.f.decay);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const unsigned at = (first + n) * kPart8 + threadIdx.x * kOptVec;
    const int valid = WHOLE ? kOptVec : max(0, min(kOptVec, e.valid - (int)at));
    P* p = (P*)e.param + at;
    float* w = (float*)e.weights + at;
    float xp[kOptVec], xg[kOptVec];
    uint2 cm = make_uint2(0, 0), cr = make_uint2(0, 0);
    float m_scale, r_scale;
    if (WHOLE) {
      widen_words(in[n].w, xp);
      widen_words(in[n].g, xg);
      cm = in[n].m;
      cr = in[n].r;
      m_scale = in[n].m_scale;
      r_scale = in[n].r_scale;
    } else {
      const uint8_t *m = (const uint8_t*)e.m + at, *v = (const uint8_t*)e.v + at;
      if (MASTER) load_some(w, valid, xp);
      else load_some(p, valid, xp);
      load_some((const G*)e.grad + at, valid, xg);
#pragma unroll
      for (int i = 0; i < kOptVec; ++i) {
        if (i < valid) {
          (i < 4 ? cm.x : cm.y) |= (uint32_t)m[i] << (8 * (i & 3));
          (i < 4 ? cr.x : cr.y) |= (uint32_t)v[i] << (8 * (i & 3));
        }
      }
      m_scale = e.m_scale[(first + n) * kWarps8 + warp];
      r_scale = e.v_scale[(first + n) * kWarps8 + warp];
    }
    codes_to_float(cm, xm[n]);
    codes_to_float(cr, xr[n]);
    const Two sm = both(m_scale), sr = both(r_scale);
    m_top[n] = r_top[n] = 0.0f;
#pragma unroll
    for (int i = 0; i < kOptVec; i += 2) {
      const Two gi = two(xg[i], xg[i + 1]) * kc;
      const Two mi = fma2(two(xm[n][i], xm[n][i + 1]) * sm * kb1, one, gi * kg1);
      const Two r = two(xr[n][i], xr[n][i + 1]) * sr;
      const Two nr = neg_sqrt(fma2(r * r * nb2, one, gi * gi * ng2));  // -v, and -sqrt(v) from here on
      const float2 d = apart(fma2(nr, ki, ke));
      const float2 np = apart(fma2(mi * ks, two(rcp_fast(d.x), rcp_fast(d.y)), two(xp[i], xp[i + 1]) * kd));
      const float2 m2 = apart(mi), r2 = apart(nr);
      xp[i] = np.x;
      xp[i + 1] = np.y;
      // Behind the tensor's end there is nothing: a block of NaN must not reach its scale from there.
      xm[n][i] = WHOLE || i < valid ? m2.x : 0.0f;
      xm[n][i + 1] = WHOLE || i + 1 < valid ? m2.y : 0.0f;
      xr[n][i] = WHOLE || i < valid ? r2.x : 0.0f;
      xr[n][i + 1] = WHOLE || i + 1 < valid ? r2.y : 0.0f;
      m_top[n] = max_nan(m_top[n], fabsf(xm[n][i]), fabsf(xm[n][i + 1]));
      r_top[n] = max_nan(r_top[n], fabsf(xr[n][i]), fabsf(xr[n][i + 1]));
    }
    if (WHOLE && (e.aligned & kVectors)) {
      if (MASTER) store_vec(w, xp);
      store_vec(p, xp);
    } else {
      if (MASTER) store_some(w, valid, xp);
      store_some(p, valid, xp);
    }
  }
  // The scales of the 2 NB blocks of moments, each formed in eight lanes.
  static_assert(2 * NB <= 4, "eight lanes to a block");
  float top = 0.0f, scale, inv;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    // Magnitudes order as their bits do, NaN above infinity.
    const float m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m_top[n])));
    const float r = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r_top[n])));
    if (lane / 16 == n) top = lane & 8 ? r : m;
  }
  scale_of(top, scale, inv);
  if (lane % 8 == 0 && lane < 16 * NB)
    ((lane & 8) ? e.v_scale : e.m_scale)[(first + lane / 16) * kWarps8 + warp] = scale;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const unsigned at = (first + n) * kPart8 + threadIdx.x * kOptVec, block = (first + n) * kWarps8 + warp;
    uint8_t *m = (uint8_t*)e.m + at, *v = (uint8_t*)e.v + at;
    const float m_inv = __shfl_sync(0xffffffffu, inv, 16 * n), r_inv = __shfl_sync(0xffffffffu, inv, 16 * n + 8);
    const uint32_t key = mix(e.f.key + e.block + block) + (uint32_t)lane * (kOptVec / 2 * kGolden);
    const Two im = both(m_inv), ir = both(-r_inv), grid = both(0x1p-120f);
    uint32_t code[kOptVec];
#pragma unroll
    for (int i = 0; i < kOptVec; i += 2) {
      const float2 qm = apart(two(xm[n][i], xm[n][i + 1]) * im);
      const float2 qr = apart(two(xr[n][i], xr[n][i + 1]) * ir * grid);
      const uint32_t word = mix(key + i / 2 * kGolden);
      code[i] = round_stochastic<0>(qr.x, xr[n][i], word);
      code[i + 1] = round_stochastic<1>(qr.y, xr[n][i + 1], word);
      xm[n][i] = qm.x;
      xm[n][i + 1] = qm.y;
    }
    const uint2 cm = float_to_codes(xm[n]);
    const uint2 cr =
        make_uint2(top_bytes(code[0], code[1], code[2], code[3]), top_bytes(code[4], code[5], code[6], code[7]));
    if (WHOLE) {
      *reinterpret_cast<uint2*>(m) = cm;
      *reinterpret_cast<uint2*>(v) = cr;
    } else {
      const int valid = max(0, min(kOptVec, e.valid - (int)at));
#pragma unroll
      for (int i = 0; i < kOptVec; ++i) {
        if (i < valid) {
          m[i] = (uint8_t)((i < 4 ? cm.x : cm.y) >> (8 * (i & 3)));
          v[i] = (uint8_t)((i < 4 ? cr.x : cr.y) >> (8 * (i & 3)));
        }
      }
    }
  }
}

// The clipping factor, which every block of a step forms for itself.  False
// where the step is to change nothing.
template <int THREADS>
__device__ __forceinline__ bool begin_step(const AdamHyper& h, float& coef) {
  coef = 1.0f;
  if (!h.part) return true;
  after_previous();
  const double norm = norm_of<THREADS>(h.part, h.parts);
  if (blockIdx.x == 0 && threadIdx.x == 0) *h.norm = (float)norm;
  coef = clip_factor(norm, h.max_norm);
  return isfinite((float)norm);  // by the norm that the caller sees; the same in every block
}

// One more to *count, and what it was.  Released and acquired: the reads that a
// block did before its barrier are behind it for whoever draws a later number.
__device__ __forceinline__ uint32_t draw(uint32_t* count) {
  uint32_t was;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(was) : "l"(count) : "memory");
  return was;
}

// The last block to come here has every other block's reads of the clocks
// behind it: it advances them, and leaves the ticket as it found it.
template <int CAP>
__device__ __forceinline__ void end_step(const AdamTable<CAP>& tab) {
  const AdamHyper& h = tab.h;
  __shared__ bool s_last;
  __syncthreads();
  if (threadIdx.x == 0) s_last = gridDim.x == 1 || draw(h.ticket) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  for (int i = threadIdx.x; i < tab.count; i += blockDim.x) {
    double* k = tab.clock[i];
    k[0] += 1.0;
    k[1] *= h.beta1;
    k[2] *= h.beta2;
  }
  if (threadIdx.x == 0 && gridDim.x > 1) *h.ticket = 0;
}

// A chunk of 2048 elements at a time, four blocks to a multiprocessor, whose
// waits hide each other.  More and shorter-lived blocks stream one large list
// slightly faster (64 to a multiprocessor: 1140 us for the sixteen textures) but
// start dearly on lists of many tensors (120 bf16 tensors with master weights:
// 110 us; 127 with 64).  Fetching the next chunk during the arithmetic takes the
// registers of two of the four blocks (1560 us).
template <typename P, typename G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kOptThreads) k_adamw(const __grid_constant__ AdamTable<CAP> tab) {
  __shared__ AdamSlot s_slots[kRounds][kOptWarps];
  const unsigned warp = threadIdx.x / 32;
  unsigned c = blockIdx.x;
  look_up<P, G, MASTER, 32>(tab, c + warp * gridDim.x, s_slots[0][warp], nullptr);
  float coef;
  if (!begin_step<kOptThreads>(tab.h, coef)) return;
  __syncthreads();
  for (int round = 0; c < tab.chunks; round = round + 1 == kRounds ? 0 : round + 1) {
    look_up<P, G, MASTER, 32>(tab, c + (kOptWarps + warp) * gridDim.x,
                              s_slots[round + 1 == kRounds ? 0 : round + 1][warp], &s_slots[round][warp]);
#pragma unroll 1
    for (int b = 0; b < kOptWarps && c < tab.chunks; ++b, c += gridDim.x)
      update32<P, G, MASTER>(s_slots[round][b], tab.h.betas, tab.h.eps, coef);
    __syncthreads();
  }
  end_step(tab);
}

// The arithmetic takes about as long as the memory: a thread's next elements
// are on their way while it computes.  One wave of one block of 16 warps to a
// multiprocessor, two blocks of states to a warp: their instructions interleave
// and share constants and addresses.  Sixteen textures in fp16: 475 us on the
// device (520 to 555 in a long run, where the power limit holds the clock down); with
// two blocks of 8 warps 500 (565), which start 0.3 us faster on small lists; with
// one block of states to a warp and three blocks 547; the same with the next
// elements on their way through shared memory, by asynchronous or bulk copies,
// 528 and 667 (64 registers, in which the packed constants do not stay).
template <typename P, typename G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads8, 1) k_adamw8(const __grid_constant__ AdamTable<CAP> tab) {
  using W = typename std::conditional<MASTER, float, P>::type;
  __shared__ AdamSlot s_slots[kRounds][kWarps8];
  const int warp = threadIdx.x / 32;
  const auto whole_in = [&](const AdamSlot& e) {
    return (e.aligned & kCodes) && (kBlocks8 - 1) * kPart8 + (warp + 1) * kStateBlock <= e.valid;
  };
  const auto fetch_all = [&](const AdamSlot& e, Fetched<W, G>* x) {
#pragma unroll
    for (int n = 0; n < kBlocks8; ++n) fetch(e, n, x[n]);
  };
  unsigned c = blockIdx.x;
  look_up<P, G, MASTER, 8>(tab, c + warp * gridDim.x, s_slots[0][warp], nullptr);
  float coef;
  if (!begin_step<kThreads8>(tab.h, coef)) return;
  __syncthreads();
  const AdamSlot* slot = &s_slots[0][0];
  bool whole = whole_in(*slot);
  Fetched<W, G> here[kBlocks8], next[kBlocks8];
  if (whole) fetch_all(*slot, here);
  for (int round = 0, following = 1, b = 0;;) {
    const AdamSlot* const this_slot = slot;
    const bool this_whole = whole;
    c += gridDim.x;
    if (++b == kWarps8) {
      b = 0;
      round = following;
      if (++following == kRounds) following = 0;
      __syncthreads();  // the round was looked up
    }
    if (c < tab.chunks) {
      slot = &s_slots[round][b];
      whole = whole_in(*slot);
      if (whole) fetch_all(*slot, next);
    }
    if (b == 1)  // the next round, whose chunk 0 is kWarps8 - 1 ahead
      look_up<P, G, MASTER, 8>(tab, c + (kWarps8 - 1 + warp) * gridDim.x, s_slots[following][warp],
                               &s_slots[round][warp]);
    if (this_whole) {
      update8<true, kBlocks8, P, G, MASTER>(*this_slot, tab.h.betas, tab.h.eps, coef, here, 0);
    } else {
#pragma unroll 1
      for (int n = 0; n < kBlocks8; ++n) {  // a tensor's end, or its pointers are not aligned
        const int left = this_slot->valid - n * kPart8 - warp * kStateBlock;
        if (left >= kStateBlock && (this_slot->aligned & kCodes)) {
          Fetched<W, G> one;
          fetch(*this_slot, n, one);
          update8<true, 1, P, G, MASTER>(*this_slot, tab.h.betas, tab.h.eps, coef, &one, n);
        } else if (left > 0) {
          update8<false, 1, P, G, MASTER, Fetched<W, G>>(*this_slot, tab.h.betas, tab.h.eps, coef, nullptr, n);
        }
      }
    }
    if (c >= tab.chunks) break;
#pragma unroll
    for (int n = 0; n < kBlocks8; ++n) here[n] = next[n];
  }
  end_step(tab);
}

// One launch for the tensors of one combination of types, CAP at a time.
template <typename P, typename G, bool MASTER, int BITS, int CAP>
dr_status launch(dr_ctx* ctx, const dr_adamw_tensor* t, int count, const AdamHyper& h, int pt, int gt, bool* early) {
  for (int i = 0; i < count;) {
    AdamTable<CAP> tab;
    int64_t chunks = 0;
    tab.count = 0;
    tab.h = h;
    for (; i < count && tab.count < CAP; ++i) {
      const dr_adamw_tensor& x = t[i];
      if (x.n == 0 || x.param_type != pt || x.grad_type != gt || (x.master != nullptr) != MASTER) continue;
      AdamEntry& e = tab.t[tab.count];
      e = {x.param, x.grad, x.master, x.m, x.v, x.m_scale, x.v_scale, x.n, x.lr_ratio, x.weight_decay, x.seed, 0};
      if (vector_aligned((const P*)x.param) && vector_aligned((const G*)x.grad) &&
          (!MASTER || vector_aligned(x.master)) &&
          (BITS == 8 || (vector_aligned((const float*)x.m) && vector_aligned((const float*)x.v))))
        e.aligned |= kVectors;
      if (BITS == 8 && (((uintptr_t)x.m | (uintptr_t)x.v) & 7) == 0) e.aligned |= kCodes;
      tab.clock[tab.count] = x.clock;
      tab.first[tab.count++] = (unsigned)chunks;
      chunks += BITS == 32 ? opt_chunks(x.n) : (x.n + kChunk8 - 1) / kChunk8;
    }
    if (tab.count == 0) break;
    tab.chunks = (unsigned)chunks;
    // Behind the norm's launch: while it is still running.
    const auto start = [&](void (*kernel)(AdamTable<CAP>), unsigned blocks, int threads) {
      if (*early) {
        *early = false;
        return launch_early(ctx->stream, blocks, threads, kernel, tab);
      }
      kernel<<<blocks, threads, 0, ctx->stream>>>(tab);
      return cudaSuccess;
    };
    DR_TB(ctx);
    if (BITS == 32) {
      const unsigned blocks = std::min(tab.chunks, (unsigned)ctx->num_sms * 4);
      DR_CUDA(ctx, start(k_adamw<P, G, MASTER, CAP>, blocks, kOptThreads), "adamw");
    } else {
      auto* kernel = k_adamw8<P, G, MASTER, CAP>;
      // One wave of blocks that stay.
      int resident = 0;
      DR_CUDA(ctx, cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads8, 0), "adamw8");
      const unsigned blocks = std::min(tab.chunks, (unsigned)(ctx->num_sms * std::max(resident, 1)));
      DR_CUDA(ctx, start(kernel, blocks, kThreads8), "adamw8");
    }
    DR_LAUNCHED(ctx, BITS == 32 ? "adamw" : "adamw8");
  }
  return DR_OK;
}

template <typename P, typename G, bool MASTER>
dr_status launch_types(dr_ctx* ctx, const dr_adamw_tensor* t, int count, const AdamHyper& h, int bits, int pt,
                       int gt, bool* early) {
  int members = 0;
  for (int i = 0; i < count; ++i)
    members += t[i].n != 0 && t[i].param_type == pt && t[i].grad_type == gt && (t[i].master != nullptr) == MASTER;
  if (members == 0) return DR_OK;
  if (members <= kSmall)
    return bits == 32 ? launch<P, G, MASTER, 32, kSmall>(ctx, t, count, h, pt, gt, early)
                      : launch<P, G, MASTER, 8, kSmall>(ctx, t, count, h, pt, gt, early);
  return bits == 32 ? launch<P, G, MASTER, 32, kLarge>(ctx, t, count, h, pt, gt, early)
                    : launch<P, G, MASTER, 8, kLarge>(ctx, t, count, h, pt, gt, early);
}

}  // namespace
}  // namespace dr

using namespace dr;

extern "C" dr_status dr_adamw_step(dr_ctx* ctx, const dr_adamw_tensor* t, int count, double lr,
                                   const float* lr_device, double beta1, double beta2, double eps, int state_bits,
                                   double max_norm, float* norm, void* work, uint32_t* ticket) {
  DR_ENTER(ctx);
  DR_REQUIRE(ctx, count >= 0 && (count == 0 || t), "adamw: null list or count < 0");
  DR_REQUIRE(ctx, state_bits == 32 || state_bits == 8, "adamw: state_bits must be 32 or 8");
  DR_REQUIRE(ctx, ticket && (uintptr_t)ticket % 4 == 0, "adamw: a 4-byte aligned ticket is required");
  DR_REQUIRE(ctx, (uintptr_t)lr_device % 4 == 0 && (uintptr_t)norm % 4 == 0, "adamw: lr_device or norm is misaligned");
  DR_REQUIRE(ctx, lr_device || (lr >= 0.0 && lr < 1e30), "adamw: lr must be finite and not negative");
  DR_REQUIRE(ctx, beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "adamw: betas must be in [0, 1)");
  DR_REQUIRE(ctx, eps >= 0x1p-126 && eps < 1e30, "adamw: eps must be at least 2^-126 and finite");
  DR_REQUIRE(ctx, max_norm >= 0.0 && max_norm < 1e300, "adamw: max_norm must be finite and not negative");
  DR_REQUIRE(ctx, max_norm == 0.0 || (norm && work && ((uintptr_t)work & 7) == 0),
             "adamw: clipping needs norm and an 8-byte aligned work");
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    const dr_adamw_tensor& x = t[i];
    DR_REQUIRE(ctx, x.n >= 0 && x.n < kOptMostElements && (chunks += opt_chunks(x.n)) < INT32_MAX,
               "adamw: tensor %d: n < 0, or too many elements", i);
    DR_REQUIRE(ctx, x.n == 0 || (x.param && x.grad && x.m && x.v && x.clock), "adamw: tensor %d: null pointer", i);
    DR_REQUIRE(ctx, x.n == 0 || state_bits == 32 || (x.m_scale && x.v_scale), "adamw: tensor %d: scales are required",
               i);
    DR_REQUIRE(ctx, valid_type(x.param_type) && valid_type(x.grad_type) &&
                        (x.grad_type == x.param_type || x.grad_type == DR_F32 || x.param_type == DR_F32),
               "adamw: tensor %d: types %d and %d", i, x.param_type, x.grad_type);
    DR_REQUIRE(ctx, !x.master || x.param_type != DR_F32, "adamw: tensor %d: fp32 has no master weights", i);
    const uintptr_t ps = x.param_type == DR_F32 ? 4 : 2, gs = x.grad_type == DR_F32 ? 4 : 2;
    const uintptr_t ss = state_bits == 32 ? 4 : 1;
    DR_REQUIRE(ctx, (uintptr_t)x.param % ps == 0 && (uintptr_t)x.grad % gs == 0 && (uintptr_t)x.m % ss == 0 &&
                        (uintptr_t)x.v % ss == 0 && (uintptr_t)x.master % 4 == 0 && (uintptr_t)x.m_scale % 4 == 0 &&
                        (uintptr_t)x.v_scale % 4 == 0 && (uintptr_t)x.clock % 8 == 0,
               "adamw: tensor %d: misaligned pointer", i);
    DR_REQUIRE(ctx, x.lr_ratio >= 0.0 && x.lr_ratio < 1e30 && x.weight_decay >= 0.0 && x.weight_decay < 1e30,
               "adamw: tensor %d: lr_ratio and weight_decay must be finite and not negative", i);
  }
  AdamHyper h = {lr, beta1, beta2, max_norm, lr_device, (float)eps, nullptr, 0, norm, ticket,
                 {(float)beta1, (float)beta2, (float)(1.0 - beta1), (float)(1.0 - beta2), 1.0f}};
  if (max_norm > 0.0) {
    dr_grad_tensor* g = new (std::nothrow) dr_grad_tensor[(size_t)count + 1];
    if (!g) return fail(ctx, DR_ENOMEM, "adamw: no host memory for %d tensors", count);
    for (int i = 0; i < count; ++i) g[i] = {const_cast<void*>(t[i].grad), t[i].n, t[i].grad_type, 0};
    const dr_status st = grad_norm_parts(ctx, g, count, (double*)work, &h.parts, nullptr, 0.0);
    delete[] g;
    if (st != DR_OK) return st;
    h.part = (const double*)work;
    if (h.parts == 0) return grad_norm_finish(ctx, (const double*)work, 0, norm);
  }
  bool early = h.part != nullptr;
#define DR_ADAMW(P, G, MASTER, PT, GT)                                                                  \
  do {                                                                                                  \
    const dr_status st = launch_types<P, G, MASTER>(ctx, t, count, h, state_bits, PT, GT, &early);              \
    if (st != DR_OK) return st;                                                                         \
  } while (0)
  DR_ADAMW(float, float, false, DR_F32, DR_F32);
  DR_ADAMW(float, __nv_bfloat16, false, DR_F32, DR_BF16);
  DR_ADAMW(float, __half, false, DR_F32, DR_F16);
  DR_ADAMW(__nv_bfloat16, __nv_bfloat16, false, DR_BF16, DR_BF16);
  DR_ADAMW(__nv_bfloat16, float, false, DR_BF16, DR_F32);
  DR_ADAMW(__nv_bfloat16, __nv_bfloat16, true, DR_BF16, DR_BF16);
  DR_ADAMW(__nv_bfloat16, float, true, DR_BF16, DR_F32);
  DR_ADAMW(__half, __half, false, DR_F16, DR_F16);
  DR_ADAMW(__half, float, false, DR_F16, DR_F32);
  DR_ADAMW(__half, __half, true, DR_F16, DR_F16);
  DR_ADAMW(__half, float, true, DR_F16, DR_F32);
#undef DR_ADAMW
  return DR_OK;
}
