// AdamW over many tensors in one launch, with the moments in float32 or in 8 bits, and the norm of all gradients with
// its clip factor.
//
//   g' = c g                        c: the clip factor, or 1
//   m' = b1 m + (1 - b1) g'         v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// Moments in 8 bits: m and s = sqrt(v) are held as e4m3 values (4 exponent, 3 mantissa bits) with one float32 scale per
// 256 consecutive elements, x = value * scale, scale = max|x| / 448.  s instead of v: the format spans 2^17.8 and the
// second moment of a block spans the square of its gradients' range.  A positive s never rounds to zero (it takes the
// smallest value): an element whose s were lost while its m survived would step by m / eps.  The scale is a float32 and
// not a power of two: moments that shrink or grow together keep their 8-bit values and move the scale, where a scale
// in powers of two would round b2 = 0.999 back to where it came from for ever.  What moves against its block does get rounded
// back: a byte changes only where sqrt(b2 + (1 - b2) (g/s)^2) leaves 1 by half a step of the format, h = 1/32 to 1/16, so s
// stays while |g| < s sqrt(((1 + h)^2 - b2) / (1 - b2)), 8 to 11 s for b2 = 0.999, and never falls.
//
// The update itself is done in float32 with the roundings of the written formula, one per operation, no contraction of
// the moments' sums: a moment next to a border between two 8-bit values then falls on the side on which the formula
// evaluated operation by operation falls.  The quotient m' / (...) alone is approximate (1 unit of the reciprocal).
//
// What bounds it: memory.  28 bytes per element in float32 (parameter and moments in and out, gradient in), 16 with 8-bit
// moments, 10 with bf16 parameters and gradients too.  Measured on one B200 (copy 6.57 TB/s; device time, states larger
// than L2): 116 M float32 elements 469 us (6.9 TB/s); 17.4 M with 8-bit moments 48 us (5.8 TB/s, of which 4 are launches);
// 116 M bf16 with 8-bit moments 201 us (5.8 TB/s; 41 instructions per element, 69 % of the issue slots), the norm of
// their gradients 50 us before it; 60 k float32 elements 6 us, two launches.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fsgs_common.cuh"
#include "fsgs_two.cuh"

namespace fsgs {

constexpr int kOptThreads = 256;
constexpr int kOptWarps = kOptThreads / 32;
constexpr int kOptBlock = FSGS_ADAMW_BLOCK;   // elements that share a scale: one warp, 8 consecutive ones per lane
constexpr int kOptCapacity = 256;             // tensors in one launch's argument table
constexpr float kTop = 448.0f;                // largest e4m3 value
constexpr float kLow = 0.001953125f;          // smallest positive e4m3 value, 2^-9
constexpr float kTiny = 7.70371978e-34f;      // 2^-110: below it 448 / max overflows and max / 448 is denormal
constexpr float kSafe = 7.88860905e-31f;      // 2^-100: from here up the root below needs no special cases

// ---- eight consecutive elements of any of the types ----------------------------------------------------------

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_fp8_e4m3 x) { return float(x); }
__device__ __forceinline__ void from_f32(float &d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16 &d, float x) { d = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(__half &d, float x) { d = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_fp8_e4m3 &d, float x) { d.__x = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ unsigned bits_of(__nv_bfloat162 x) { return *reinterpret_cast<const unsigned *>(&x); }
__device__ __forceinline__ unsigned bits_of(__half2 x) { return *reinterpret_cast<const unsigned *>(&x); }

// As they lie in memory: 32, 16 or 8 bytes, one or two accesses per lane.
template <typename T>
struct Packed;
template <>
struct Packed<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float *p) {
    a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
  }
  __device__ __forceinline__ void get(float *x) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
  __device__ __forceinline__ unsigned bits() const {  // zero where all eight are (as below)
    float x[8];
    get(x);
    unsigned r = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) r |= __float_as_uint(x[u]);
    return r;
  }
  static __device__ __forceinline__ void store(float *p, const float *x) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};
template <>
struct Packed<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) { a = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float *x) const {
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) x[2 * u] = __uint_as_float(w[u] << 16), x[2 * u + 1] = __uint_as_float(w[u] & 0xffff0000u);
  }
  __device__ __forceinline__ unsigned bits() const { return a.x | a.y | a.z | a.w; }
  static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(bits_of(__floats2bfloat162_rn(x[0], x[1])), bits_of(__floats2bfloat162_rn(x[2], x[3])),
                                               bits_of(__floats2bfloat162_rn(x[4], x[5])), bits_of(__floats2bfloat162_rn(x[6], x[7])));
  }
};
template <>
struct Packed<__half> {
  uint4 a;
  __device__ __forceinline__ void load(const __half *p) { a = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void get(float *x) const {
    const unsigned w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[u]));
      x[2 * u] = f.x, x[2 * u + 1] = f.y;
    }
  }
  __device__ __forceinline__ unsigned bits() const { return a.x | a.y | a.z | a.w; }
  static __device__ __forceinline__ void store(__half *p, const float *x) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(bits_of(__floats2half2_rn(x[0], x[1])), bits_of(__floats2half2_rn(x[2], x[3])),
                                               bits_of(__floats2half2_rn(x[4], x[5])), bits_of(__floats2half2_rn(x[6], x[7])));
  }
};
template <>
struct Packed<__nv_fp8_e4m3> {
  uint2 a;
  __device__ __forceinline__ void load(const __nv_fp8_e4m3 *p) { a = *reinterpret_cast<const uint2 *>(p); }
  __device__ __forceinline__ void get(float *x) const {
    const unsigned w[2] = {a.x, a.y};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((unsigned short) (w[u >> 1] >> (16 * (u & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[2 * u] = f.x, x[2 * u + 1] = f.y;
    }
  }
  static __device__ __forceinline__ void store(__nv_fp8_e4m3 *p, const float *x) {
    unsigned c[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) c[u] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * u], x[2 * u + 1]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2 *>(p) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
};

// the same eight elements one by one, for a tensor's last block and for addresses that are not aligned
template <typename T>
__device__ __forceinline__ void load_some(const T *p, long long left, float *x) {
#pragma unroll
  for (int u = 0; u < 8; ++u) x[u] = u < left ? to_f32(p[u]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_some(T *p, long long left, const float *x) {
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (u < left) from_f32(p[u], x[u]);
}

__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rsqrt(float x) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// ------------------------------------------------------------------------------------------------
// the step
// ------------------------------------------------------------------------------------------------

struct AdamWEntry {
  void *param;
  const void *grad;
  void *m, *v;
  float *m_scale, *v_scale;
  float *master;
  long long numel;
  float keep;  // 1 - lr * weight_decay
};

// The argument table of a launch, for CAP tensors: 20 KB for 256, 1.3 KB for 16.  The driver copies it with every launch;
// most optimisers have few tensors and take the small one (a step of 3: 10.1 us on the host against 11.2).
template <int CAP>
struct AdamWTable {
  AdamWEntry t[CAP];
  int chunk_start[CAP + 1];  // prefix sums of thread blocks
  uint8_t vec[CAP];          // every array aligned for the packed accesses
  int n;
};
constexpr int kOptFew = 16;

struct AdamWScalars {
  float b1, b2, c1, c2, eps;   // c = 1 - b, formed in double
};

// index of the tensor that holds a block: the last k with start[k] <= block
__device__ __forceinline__ int tensor_of(const int *start, int n, int block) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// largest magnitude and largest value of eight; a NaN among them is the largest magnitude
__device__ __forceinline__ float top8(const float *x) {
  float t;
  asm("{\n\t.reg .f32 a, b, c;\n\t"
      "max.NaN.abs.f32 a, %1, %2, %3;\n\tmax.NaN.abs.f32 b, %4, %5, %6;\n\t"
      "max.NaN.abs.f32 c, %7, %8, a;\n\tmax.NaN.abs.f32 %0, b, c, c;\n\t}"
      : "=f"(t) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return t;
}
__device__ __forceinline__ float high8(const float *x) {
  float t;
  asm("{\n\t.reg .f32 a, b, c;\n\t"
      "max.f32 a, %1, %2, %3;\n\tmax.f32 b, %4, %5, %6;\n\t"
      "max.f32 c, %7, %8, a;\n\tmax.f32 %0, b, c, c;\n\t}"
      : "=f"(t) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
  return t;
}

// The negatives s = -sqrt(-v) of the roots of eight numbers -v.  From 2^-100 up: the hardware's approximate reciprocal
// root and one step of Newton's method on the residual s^2 - (-v).  The result is the correctly rounded root: compared with
// __fsqrt_rn for each of the 2^24 floats of [1, 4), [2^-100, 2^-98) and [2^126, 2^128), none differs (a power of four more
// or less changes exponents alone).  `plain`: all eight lie there and are finite.  (Negatives, because the residual wants -v.)
__device__ __forceinline__ void neg_roots(const float *v, float *s, bool plain) {
  if (plain) {
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      const Two r = two(fast_rsqrt(fabsf(v[u])), fast_rsqrt(fabsf(v[u + 1]))), n = two(v[u], v[u + 1]);
      const Two q = mul2(n, r);
      split(fma2(fma2(q, q, n), mul2(r, both(0.5f)), q), s[u], s[u + 1]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) s[u] = -__fsqrt_rn(-v[u]);
  }
}

// One block of 256 elements, eight per lane: m (decoded where 8 bits), v (sqrt(v) decoded where 8 bits), p in and out;
// 8 bits: m and v come out as multiples of the block's new scales.
template <bool EIGHT>
__device__ __forceinline__ void update(const float *g, float *m, float *v, float *p, float scale, float ms, float vs,
    const AdamWScalars &s, float step, float root, float keep, float *m_scale, float *v_scale, int lane) {
#pragma unroll
  for (int u = 0; u < 8; u += 2) {
    const Two gs = mul2(two(g[u], g[u + 1]), both(scale));
    Two a = two(m[u], m[u + 1]), b = two(v[u], v[u + 1]);
    if (EIGHT) a = mul2(a, both(ms)), b = mul2(b, both(vs)), b = mul2(b, b);
    plain_sum(mul2(a, both(s.b1)), mul2(gs, both(s.c1)), m[u], m[u + 1]);
    plain_sum(mul2(b, both(-s.b2)), mul2(mul2(gs, gs), both(-s.c2)), v[u], v[u + 1]);  // -v'
  }
  // a NaN among others passes: its own root is a NaN either way
  const bool plain = high8(v) <= -kSafe && !(top8(v) == INFINITY);
  float q[8];  // -sqrt(v')
  neg_roots(v, q, plain);
#pragma unroll
  for (int u = 0; u < 8; u += 2) {
    float d0, d1;
    split(fma2(two(q[u], q[u + 1]), both(-root), both(s.eps)), d0, d1);
    const Two w = mul2(two(m[u], m[u + 1]), two(fast_rcp(d0), fast_rcp(d1)));
    split(fma2(w, both(-step), mul2(two(p[u], p[u + 1]), both(keep))), p[u], p[u + 1]);
  }
  if (!EIGHT) {
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = -v[u];
  }
  if (EIGHT) {
    // maxima over the warp as the bit patterns of non-negative floats order; odd lanes go on with the one of sqrt(v)
    const unsigned mt = __reduce_max_sync(0xffffffffu, __float_as_uint(top8(m)));
    const unsigned vt = __reduce_max_sync(0xffffffffu, __float_as_uint(top8(q)));
    const float top = __uint_as_float(lane & 1 ? vt : mt);
    const bool zero = top < kTiny;  // a block of nothing but zeros (or denormals) has scale 0 and values 0
    const float inv = zero ? 0.0f : __fmul_rn(__frcp_rn(top), kTop);
    if (lane < 2) *(lane ? v_scale : m_scale) = zero ? 0.0f : __fmul_rn(top, 1.0f / kTop);
    const float mr = __shfl_sync(0xffffffffu, inv, 0), vr = __shfl_sync(0xffffffffu, inv, 1);
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      split(mul2(two(m[u], m[u + 1]), both(mr)), m[u], m[u + 1]);
      split(mul2(two(q[u], q[u + 1]), both(-vr)), v[u], v[u + 1]);
    }
    if (plain && vr > 0.0f) {
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = fmaxf(v[u], kLow);
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = v[u] > 0.0f && v[u] < kLow ? kLow : v[u];
    }
  }
}

// what the update needs of a tensor's step count
struct AdamWFactors {
  float step, root;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};

template <int CAP>
struct AdamWBegin {
  float *step[CAP];
  float lr[CAP];
  int n;
};

// Decides whether the step is taken, counts it and forms the bias corrections, one thread per tensor; scale_out < 0 tells
// the kernel behind it that the step is dropped.
template <int CAP>
__global__ void __launch_bounds__(CAP) adamw_begin_kernel(const __grid_constant__ AdamWBegin<CAP> a, double log_b1, double log_b2,
    const float *grad_scale, const float *gate, float *scale_out, AdamWFactors *out) {
  const float scale = grad_scale ? *grad_scale : 1.0f;
  const bool open = !(gate && !(*gate > 0.0f)) && scale > 0.0f && scale < INFINITY;
  if (threadIdx.x == 0) *scale_out = open ? scale : -1.0f;
  const int k = threadIdx.x;
  if (!open || k >= a.n) return;
  const double t = (double) *a.step[k] + 1.0;
  *a.step[k] = (float) t;
  out[k].step = (float) (a.lr[k] / (1.0 - exp(log_b1 * t)));
  out[k].root = (float) (1.0 / sqrt(1.0 - exp(log_b2 * t)));
}

// One warp per block of 256 elements, or per two blocks whose loads go out together.  The grid covers the tensors and
// leaves the order to the hardware, which hands out thread blocks as others finish, each reading all that it needs before
// it writes: the memory in use at any moment is one short stretch of every array, and DRAM pages are opened once.  Measured
// (us; 116 M elements in float32 with float32 moments | bf16 with 8-bit moments, the norm before it included):
//   this order                                                                  469 | 256
//   a grid that fills the device, blocks interleaved (2 / 3 thread blocks an SM)  507 / 598 | 320
//   every warp a run of its own                                                 588 | 269
//   bulk copies through a ring in shared memory, 3 thread blocks an SM            - | 293, and 272 with no arithmetic at all
//   this order, a warp's second block loaded while the first is computed        592 | 290
// Two blocks per warp where an element brings 4 bytes of parameter and gradient (256 against 281: half the address and
// argument work per element), one where it brings more (49 against 57 us for 17.4 M float32 elements: the second
// block's registers push the loads behind the first block's stores).
template <typename P, typename G, bool EIGHT, bool MASTER>
struct PerWarp {
  static constexpr int blocks = EIGHT && sizeof(G) + (MASTER ? 4 : sizeof(P)) <= 4 ? 2 : 1;
  static constexpr int elements = kOptWarps * kOptBlock * blocks;  // of a thread block
};

template <typename P, typename G, bool EIGHT, bool MASTER, int CAP>
__global__ void __launch_bounds__(kOptThreads, EIGHT ? 4 : 3) adamw_kernel(const __grid_constant__ AdamWTable<CAP> a, const AdamWScalars s,
    const float *__restrict__ scale_in, const AdamWFactors *__restrict__ factors) {
  using S = typename std::conditional<EIGHT, __nv_fp8_e4m3, float>::type;
  using W = typename std::conditional<MASTER, float, P>::type;  // where the parameter's value is read from
  constexpr int NB = PerWarp<P, G, EIGHT, MASTER>::blocks;
  const int lane = threadIdx.x & 31;
  const int k = tensor_of(a.chunk_start, a.n, blockIdx.x);
  const AdamWEntry &t = a.t[k];
  const long long block = (long long) (blockIdx.x - a.chunk_start[k]) * (kOptWarps * NB) + (threadIdx.x >> 5);
  const float scale = *scale_in;
  const AdamWFactors f = factors[k];
  const bool vec = a.vec[k] != 0;
  const long long at = block * kOptBlock + 8 * lane;
  const long long left = t.numel - block * kOptBlock;  // elements from the block's start on
  const G *g_at = (const G *) t.grad + at;
  S *m_at = (S *) t.m + at, *v_at = (S *) t.v + at;
  P *p_at = (P *) t.param + at;
  W *w_at = MASTER ? (W *) t.master + at : (W *) p_at;
  float *ms_at = EIGHT ? t.m_scale + block : nullptr, *vs_at = EIGHT ? t.v_scale + block : nullptr;
  constexpr int hop = kOptWarps * kOptBlock;
  Packed<G> ng[NB];
  Packed<S> nm[NB], nv[NB];
  Packed<W> nw[NB];
  float nms[NB], nvs[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    if (vec && left >= i * hop + kOptBlock) {
      ng[i].load(g_at + i * hop), nm[i].load(m_at + i * hop), nv[i].load(v_at + i * hop), nw[i].load(w_at + i * hop);
      if (EIGHT) nms[i] = ms_at[i * kOptWarps], nvs[i] = vs_at[i * kOptWarps];
    }
  }
  if (scale < 0.0f) return;  // dropped
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const long long here = left - i * hop, some = here - 8 * lane;
    if (here <= 0) return;
    const bool whole = vec && here >= kOptBlock;
    float g[8], m[8], v[8], p[8], ms = 1.0f, vs = 1.0f;
    if (whole) {
      ng[i].get(g), nm[i].get(m), nv[i].get(v), nw[i].get(p);
      if (EIGHT) ms = nms[i], vs = nvs[i];
    } else {  // a tensor's last block, or addresses that are not aligned
      load_some(g_at + i * hop, some, g), load_some(m_at + i * hop, some, m), load_some(v_at + i * hop, some, v);
      load_some(w_at + i * hop, some, p);
      if (EIGHT) ms = ms_at[i * kOptWarps], vs = vs_at[i * kOptWarps];
    }
    __syncwarp();  // every lane has the old scales
    update<EIGHT>(g, m, v, p, scale, ms, vs, s, f.step, f.root, t.keep, EIGHT ? ms_at + i * kOptWarps : nullptr,
                  EIGHT ? vs_at + i * kOptWarps : nullptr, lane);
    if (whole) {
      if (MASTER) Packed<W>::store(w_at + i * hop, p);
      Packed<P>::store(p_at + i * hop, p);
      Packed<S>::store(m_at + i * hop, m);
      Packed<S>::store(v_at + i * hop, v);
    } else {
      if (MASTER) store_some(w_at + i * hop, some, p);
      store_some(p_at + i * hop, some, p);
      store_some(m_at + i * hop, some, m);
      store_some(v_at + i * hop, some, v);
    }
  }
}

struct AdamWCall {
  int n;
  const fsgs_adamw_tensor *tensors;
  AdamWScalars scalars;
  double log_b1, log_b2;
  const float *grad_scale, *gate;
  float *scale;       // workspace: the factor, then the bias corrections
  AdamWFactors *factors;
  cudaStream_t stream;
};

template <typename P, typename G, bool EIGHT, bool MASTER, int CAP>
static int adamw_launches(const AdamWCall &c) {
  constexpr int per = PerWarp<P, G, EIGHT, MASTER>::elements;
  for (int first = 0; first < c.n;) {
    AdamWTable<CAP> a;
    AdamWBegin<CAP> begin;
    a.n = 0, a.chunk_start[0] = 0;
    for (; first < c.n && a.n < CAP; ++first) {
      const fsgs_adamw_tensor &t = c.tensors[first];
      const int64_t chunks = (t.numel + per - 1) / per;
      if (a.chunk_start[a.n] + chunks > INT32_MAX) break;  // the rest in a launch of its own
      AdamWEntry &d = a.t[a.n];
      d.param = t.param, d.grad = t.grad, d.m = t.exp_avg, d.v = t.exp_avg_sq, d.m_scale = t.exp_avg_scale;
      d.v_scale = t.exp_avg_sq_scale, d.master = t.master, d.numel = t.numel;
      d.keep = (float) (1.0 - (double) t.lr * (double) t.weight_decay);
      begin.step[a.n] = t.step, begin.lr[a.n] = t.lr;
      a.vec[a.n] = !((((uintptr_t) t.param | (uintptr_t) t.grad | (uintptr_t) t.master) & 15) |
                     (((uintptr_t) t.exp_avg | (uintptr_t) t.exp_avg_sq) & (EIGHT ? 7 : 15)));
      a.chunk_start[a.n + 1] = a.chunk_start[a.n] + (int) chunks;
      begin.n = ++a.n;
    }
    adamw_begin_kernel<CAP><<<1, CAP, 0, c.stream>>>(begin, c.log_b1, c.log_b2, c.grad_scale, c.gate, c.scale, c.factors);
    FSGS_LAUNCH_CHECK();
    if (a.chunk_start[a.n] == 0) continue;
    adamw_kernel<P, G, EIGHT, MASTER, CAP><<<a.chunk_start[a.n], kOptThreads, 0, c.stream>>>(a, c.scalars, c.scale, c.factors);
    FSGS_LAUNCH_CHECK();
  }
  return FSGS_OK;
}

template <typename P, typename G, bool EIGHT, bool MASTER>
static int adamw_run(const AdamWCall &c) {
  constexpr int per = PerWarp<P, G, EIGHT, MASTER>::elements;
  for (int k = 0; k < c.n; ++k)
    if ((c.tensors[k].numel + per - 1) / per > INT32_MAX) return FSGS_ERR_LIMIT;
  return c.n <= kOptFew ? adamw_launches<P, G, EIGHT, MASTER, kOptFew>(c) : adamw_launches<P, G, EIGHT, MASTER, kOptCapacity>(c);
}

template <typename P, typename G>
static int adamw_pick(bool eight, bool master, const AdamWCall &c) {
  if (eight) return master ? adamw_run<P, G, true, true>(c) : adamw_run<P, G, true, false>(c);
  return master ? adamw_run<P, G, false, true>(c) : adamw_run<P, G, false, false>(c);
}

// ------------------------------------------------------------------------------------------------
// the norm of all gradients
// ------------------------------------------------------------------------------------------------

// One pass over all gradients, bound by its read: 464 MB of float32 in 70 us (6.6 TB/s), 232 MB of bf16 in 39 us call after
// call (part of them from L2), 50 us in front of a step; a small call is two launches, 4 us.  Every thread block adds its share in double and leaves it in a slot of its own; a block of a
// second launch adds the slots.  No counter, nothing to prepare: a workspace can be used again as soon as a call is done.
struct NormEntry {
  const void *data;
  long long numel;
};

struct NormTable {
  NormEntry t[kOptCapacity];
  int chunk_start[kOptCapacity + 1];  // prefix sums of ceil(numel / kNormChunk)
  uint8_t type[kOptCapacity], vec[kOptCapacity];
  int n;
};

constexpr int kNormPart = kOptWarps * kOptBlock;   // elements of one pass of a thread block
constexpr int kNormChunk = 4 * kNormPart;
constexpr int kNormSlots = FSGS_GRAD_NORM_SLOTS;
constexpr double kLost = 1.0 / (1ull << 56) / (1ull << 56);  // 2^-112

// Sum of the squares of this thread's elements of a chunk.  Eight squares are added in float32 (two sums of four) and the
// eights in double: the float32 part rounds each eight by 5 x 2^-24 at most.  An eight overflows above |g| = 6e18, and what
// its squares lose below 2^-126, 2^-150 each, shows where nearly all gradients are below 1e-18: the kernel looks at its sum
// for both.  `bits`: all elements' bits, zero where the gradients are.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, bool vec, long long left, int warp, int lane, unsigned &bits) {
  constexpr int parts = kNormChunk / kNormPart;
  auto squares = [](const float *x) {
    Two q = both(0.0f);
#pragma unroll
    for (int u = 0; u < 8; u += 2) q = fma2(two(x[u], x[u + 1]), two(x[u], x[u + 1]), q);
    float a, b;
    split(q, a, b);
    return (double) (a + b);
  };
  double sum = 0.0;
  float x[8];
  p += warp * kOptBlock + 8 * lane;
  if (vec && left >= kNormChunk) {  // as many loads under way as the registers take
    Packed<T> w[parts];
#pragma unroll
    for (int j = 0; j < parts; ++j) w[j].load(p + j * kNormPart);
#pragma unroll
    for (int j = 0; j < parts; ++j) w[j].get(x), bits |= w[j].bits(), sum += squares(x);
  } else {
    left -= warp * kOptBlock + 8 * lane;
#pragma unroll 1
    for (int j = 0; j < parts && left > 0; ++j, p += kNormPart, left -= kNormPart) {
      if (vec && left >= 8) {
        Packed<T> w;
        w.load(p);
        w.get(x);
      } else {
        load_some(p, left, x);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) bits |= __float_as_uint(x[u]);
      sum += squares(x);
    }
  }
  return sum;
}

// The same over a warp's elements of a chunk, every square in double, whose range holds that of every float32.
template <typename T>
__device__ __noinline__ double warp_squares(const T *p, long long left, int warp, int lane) {
  double sum = 0.0;
#pragma unroll 1
  for (int e = warp * kOptBlock; e < kNormChunk; e += kNormPart)
#pragma unroll 1
    for (int i = e + lane; i < e + kOptBlock && i < left; i += 32) {
      const double x = (double) to_f32(p[i]);
      sum += x * x;
    }
  return sum;
}

__device__ __forceinline__ double warp_total(double sum) {
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

// `filled`: sums that earlier launches of the same call have left in the slots
__global__ void __launch_bounds__(kOptThreads) grad_norm_kernel(const __grid_constant__ NormTable a, double *slots, int filled) {
  __shared__ double s_sum[kOptThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = a.chunk_start[a.n];
  double sum = 0.0;
  unsigned bits = 0;
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int k = tensor_of(a.chunk_start, a.n, chunk);
    const long long e0 = (long long) (chunk - a.chunk_start[k]) * kNormChunk;
    const long long left = a.t[k].numel - e0;
    const bool vec = a.vec[k] != 0;
    if (a.type[k] == FSGS_F32) sum += chunk_squares((const float *) a.t[k].data + e0, vec, left, warp, lane, bits);
    else if (a.type[k] == FSGS_BF16) sum += chunk_squares((const __nv_bfloat16 *) a.t[k].data + e0, vec, left, warp, lane, bits);
    else sum += chunk_squares((const __half *) a.t[k].data + e0, vec, left, warp, lane, bits);
  }
  sum = warp_total(sum);
  // a warp's 1024 elements of a chunk lose 2^-140 at most; again in double where that may be above 2^-28 of the sum, and
  // where the sum has overflowed (or holds a NaN, which stays)
  const double least = kLost * (double) ((total - 1 - (int) blockIdx.x) / (int) gridDim.x + 1);
  if (__any_sync(0xffffffffu, bits != 0) && !(sum >= least && sum < INFINITY)) {
    sum = 0.0;
    for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
      const int k = tensor_of(a.chunk_start, a.n, chunk);
      const long long e0 = (long long) (chunk - a.chunk_start[k]) * kNormChunk;
      const long long left = a.t[k].numel - e0;
      if (a.type[k] == FSGS_F32) sum += warp_squares((const float *) a.t[k].data + e0, left, warp, lane);
      else if (a.type[k] == FSGS_BF16) sum += warp_squares((const __nv_bfloat16 *) a.t[k].data + e0, left, warp, lane);
      else sum += warp_squares((const __half *) a.t[k].data + e0, left, warp, lane);
    }
    sum = warp_total(sum);
  }
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double t = 0.0;
  for (int w = 0; w < kOptThreads / 32; ++w) t += s_sum[w];
  slots[blockIdx.x] = (int) blockIdx.x < filled ? slots[blockIdx.x] + t : t;
}

// Adds the slots in a fixed order: the same gradients give the same norm, bit for bit.
__global__ void __launch_bounds__(kOptThreads) grad_norm_close_kernel(const double *__restrict__ slots, int n, float max_norm,
    float *__restrict__ out) {
  __shared__ double s_sum[kOptThreads / 32];
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
#pragma unroll 5
  for (int i = threadIdx.x; i < n; i += kOptThreads) sum += slots[i];
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double t = 0.0;
  for (int w = 0; w < kOptThreads / 32; ++w) t += s_sum[w];
  const float norm = (float) sqrt(t);
  // a norm that is not a number or infinite: factor 0, which drops the step that is given it
  out[0] = norm;
  out[1] = norm < INFINITY ? fminf(1.0f, __fmul_rn(__frcp_rn(__fadd_rn(norm, 1e-6f)), max_norm)) : 0.0f;
}

static bool is_type(int type) { return type == FSGS_F32 || type == FSGS_BF16 || type == FSGS_F16; }

}  // namespace fsgs

using namespace fsgs;

extern "C" size_t fsgs_adamw_workspace_bytes(void) { return 16 + sizeof(AdamWFactors) * kOptCapacity; }

extern "C" int fsgs_adamw_multi(int n_tensors, const fsgs_adamw_tensor *tensors, int param_type, int grad_type,
    int state_bits, double beta1, double beta2, float eps, const float *grad_scale, const float *gate, void *workspace,
    size_t workspace_bytes, fsgs_stream_t stream) {
  FSGS_REQUIRE(n_tensors >= 0 && (tensors || n_tensors == 0) && is_type(param_type) && is_type(grad_type));
  FSGS_REQUIRE(state_bits == 8 || state_bits == 32);
  FSGS_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0);
  if (param_type == FSGS_F32 ? grad_type != FSGS_F32 : grad_type != FSGS_F32 && grad_type != param_type) return FSGS_ERR_UNSUPPORTED;
  if (n_tensors == 0) return FSGS_OK;
  const bool eight = state_bits == 8, master = tensors[0].master != nullptr;
  if (master && param_type == FSGS_F32) return FSGS_ERR_UNSUPPORTED;
  for (int k = 0; k < n_tensors; ++k) {
    const fsgs_adamw_tensor &t = tensors[k];
    FSGS_REQUIRE(t.numel >= 0 && t.step && (t.master != nullptr) == master);
    FSGS_REQUIRE(t.numel == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq));
    FSGS_REQUIRE(t.numel == 0 || !eight || (t.exp_avg_scale && t.exp_avg_sq_scale));
  }
  if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < fsgs_adamw_workspace_bytes()) return FSGS_ERR_WORKSPACE;
  AdamWCall c;
  c.n = n_tensors, c.tensors = tensors;
  c.scalars = {(float) beta1, (float) beta2, (float) (1.0 - beta1), (float) (1.0 - beta2), eps};
  c.log_b1 = log(beta1), c.log_b2 = log(beta2);  // beta 0: -infinity, whose exponential is 0
  c.grad_scale = grad_scale, c.gate = gate, c.stream = (cudaStream_t) stream;
  c.scale = (float *) workspace, c.factors = (AdamWFactors *) ((char *) workspace + 16);
  if (param_type == FSGS_F32) return eight ? adamw_run<float, float, true, false>(c) : adamw_run<float, float, false, false>(c);
  if (param_type == FSGS_BF16)
    return grad_type == FSGS_F32 ? adamw_pick<__nv_bfloat16, float>(eight, master, c) : adamw_pick<__nv_bfloat16, __nv_bfloat16>(eight, master, c);
  return grad_type == FSGS_F32 ? adamw_pick<__half, float>(eight, master, c) : adamw_pick<__half, __half>(eight, master, c);
}

extern "C" size_t fsgs_grad_norm_workspace_bytes(void) { return sizeof(double) * kNormSlots; }

extern "C" int fsgs_grad_norm(int n_tensors, const fsgs_norm_tensor *tensors, float max_norm, void *workspace,
    size_t workspace_bytes, float *out, fsgs_stream_t stream) {
  FSGS_REQUIRE(n_tensors >= 0 && (tensors || n_tensors == 0) && out && max_norm > 0.0f);
  if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < fsgs_grad_norm_workspace_bytes()) return FSGS_ERR_WORKSPACE;
  for (int k = 0; k < n_tensors; ++k) {
    FSGS_REQUIRE(tensors[k].numel >= 0 && is_type(tensors[k].type) && (tensors[k].data || tensors[k].numel == 0));
    if (tensors[k].numel / kNormChunk >= INT32_MAX - (1 << 20)) return FSGS_ERR_LIMIT;
  }
  double *slots = (double *) workspace;
  int filled = 0;
  for (int first = 0; first < n_tensors;) {
    NormTable a;
    a.n = 0, a.chunk_start[0] = 0;
    for (; first < n_tensors && a.n < kOptCapacity; ++first) {
      const fsgs_norm_tensor &t = tensors[first];
      const int64_t chunks = (t.numel + kNormChunk - 1) / kNormChunk;
      if (a.chunk_start[a.n] + chunks > INT32_MAX - (1 << 20)) break;  // the rest in a launch of its own
      a.t[a.n].data = t.data, a.t[a.n].numel = t.numel, a.type[a.n] = (uint8_t) t.type;
      a.vec[a.n] = ((uintptr_t) t.data & 15) == 0;
      a.chunk_start[a.n + 1] = a.chunk_start[a.n] + (int) chunks;
      ++a.n;
    }
    const int chunks = a.chunk_start[a.n], grid = chunks < kNormSlots ? chunks : kNormSlots;
    if (grid == 0) continue;
    grad_norm_kernel<<<grid, kOptThreads, 0, (cudaStream_t) stream>>>(a, slots, filled);
    FSGS_LAUNCH_CHECK();
    if (grid > filled) filled = grid;
  }
  grad_norm_close_kernel<<<1, kOptThreads, 0, (cudaStream_t) stream>>>(slots, filled, max_norm, out);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}
