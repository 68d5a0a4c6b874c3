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
// in powers of two would round b2 = 0.999 back to where it came from for ever.
//
// The update itself is done in float32 with the roundings of the written formula, one per operation, no contraction of
// the moments' sums: a moment next to a border between two 8-bit values then falls on the side on which the formula
// evaluated operation by operation falls.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "fsgs_common.cuh"

namespace fsgs {

constexpr int kOptThreads = 256;
constexpr int kOptBlock = FSGS_ADAMW_BLOCK;               // elements that share a scale: one warp, 8 per lane
constexpr int kOptChunk = (kOptThreads / 32) * kOptBlock;  // elements of one pass of a thread block
constexpr int kOptCapacity = 256;                          // tensors in one launch's argument table
constexpr float kTop = 448.0f;                             // largest e4m3 value
constexpr float kLow = 0.001953125f;                       // smallest positive e4m3 value, 2^-9
constexpr float kTiny = 7.70371978e-34f;                   // 2^-110: below it 448 / max overflows and max / 448 is denormal

// ---- four consecutive elements of any of the types, as float32 ---------------------------------------------

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_fp8_e4m3 x) { return float(x); }
__device__ __forceinline__ void from_f32(float &d, float x) { d = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16 &d, float x) { d = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(__half &d, float x) { d = __float2half_rn(x); }
__device__ __forceinline__ void from_f32(__nv_fp8_e4m3 &d, float x) { d.__x = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ void load4(const float *p, float *x) {
  const float4 v = *reinterpret_cast<const float4 *>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *x) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
  x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const __half *p, float *x) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ float2 pair_f32(unsigned short v) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(v, __NV_E4M3);
  return __half22float2(__half2(h));
}
__device__ __forceinline__ void load4(const __nv_fp8_e4m3 *p, float *x) {
  const unsigned v = *reinterpret_cast<const unsigned *>(p);
  const float2 a = pair_f32((unsigned short) v), b = pair_f32((unsigned short) (v >> 16));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void store4(float *p, const float *x) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float *x) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}
__device__ __forceinline__ void store4(__half *p, const float *x) {
  const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}
__device__ __forceinline__ void store4(__nv_fp8_e4m3 *p, const float *x) {
  const unsigned a = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const unsigned b = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<unsigned *>(p) = a | (b << 16);
}

// Lane's eight elements of a 256-element block: 4 lane + {0..3} and 128 + 4 lane + {0..3}, so that every access of a
// warp covers consecutive memory.  `left`: elements from the block's start to the tensor's end.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, long long left, int lane, float *x) {
  if (vec && left >= kOptBlock) {
    load4(p + 4 * lane, x);
    load4(p + 128 + 4 * lane, x + 4);
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = (u >> 2) * 128 + 4 * lane + (u & 3);
      x[u] = e < left ? to_f32(p[e]) : 0.0f;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, long long left, int lane, const float *x) {
  if (vec && left >= kOptBlock) {
    store4(p + 4 * lane, x);
    store4(p + 128 + 4 * lane, x + 4);
  } else {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int e = (u >> 2) * 128 + 4 * lane + (u & 3);
      if (e < left) from_f32(p[e], x[u]);
    }
  }
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
  float *step;
  long long numel;
  float lr, keep;  // keep = 1 - lr * weight_decay
};

struct AdamWTable {
  AdamWEntry t[kOptCapacity];
  int chunk_start[kOptCapacity + 1];  // prefix sums of ceil(numel / kOptChunk)
  uint8_t vec[kOptCapacity];          // every array aligned for four-element accesses
  int n;
};

struct AdamWScalars {
  float b1, b2, c1, c2, eps;   // c = 1 - b, formed in double
  double log_b1, log_b2;
  const float *grad_scale, *gate;
  int *ticket;
};

// index of the tensor that holds `chunk`: the last k with chunk_start[k] <= chunk
template <typename Table>
__device__ __forceinline__ int tensor_of(const Table &a, int chunk) {
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.chunk_start[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// max over the warp of non-negative floats, as their bit patterns order (a NaN comes out on top)
__device__ __forceinline__ float warp_max_abs(const float *x) {
  unsigned top = 0;
#pragma unroll
  for (int u = 0; u < 8; ++u) top = max(top, __float_as_uint(x[u]) & 0x7fffffffu);
  return __uint_as_float(__reduce_max_sync(0xffffffffu, top));
}

template <typename P, typename G, bool EIGHT, bool MASTER>
__global__ void __launch_bounds__(kOptThreads) adamw_kernel(const __grid_constant__ AdamWTable a, const AdamWScalars s) {
  using S = typename std::conditional<EIGHT, __nv_fp8_e4m3, float>::type;
  using W = typename std::conditional<MASTER, float, P>::type;  // where the parameter's value is read from
  __shared__ float s_step, s_root;
  __shared__ int s_last;
  float scale = 1.0f;
  if (s.gate && !(*s.gate > 0.0f)) return;  // the same for every thread of the grid
  if (s.grad_scale) {
    scale = *s.grad_scale;
    if (!(scale > 0.0f && scale < INFINITY)) return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = a.chunk_start[a.n];
  int have = -1;
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int k = tensor_of(a, chunk);
    const AdamWEntry &t = a.t[k];
    const long long e0 = (long long) (chunk - a.chunk_start[k]) * kOptChunk + warp * kOptBlock;
    const long long left = t.numel - e0;
    const bool vec = a.vec[k] != 0;
    float g[8], m[8], v[8], p[8];
    if (left > 0) {
      load8((const G *) t.grad + e0, vec, left, lane, g);
      load8((const S *) t.m + e0, vec, left, lane, m);
      load8((const S *) t.v + e0, vec, left, lane, v);
      if (MASTER) load8((const float *) t.master + e0, vec, left, lane, p);
      else load8((const W *) t.param + e0, vec, left, lane, p);
      if (EIGHT) {
        const float ms = t.m_scale[e0 / kOptBlock], vs = t.v_scale[e0 / kOptBlock];
#pragma unroll
        for (int u = 0; u < 8; ++u) m[u] = __fmul_rn(m[u], ms), v[u] = __fmul_rn(v[u], vs), v[u] = __fmul_rn(v[u], v[u]);
      }
    }
    if (k != have) {  // bias corrections of this tensor: two exponentials in double, by one thread of two warps each
      __syncthreads();
      if (threadIdx.x == 0) s_step = (float) (t.lr / (1.0 - exp(s.log_b1 * ((double) *t.step + 1.0))));
      if (threadIdx.x == 32) s_root = (float) (1.0 / sqrt(1.0 - exp(s.log_b2 * ((double) *t.step + 1.0))));
      __syncthreads();
      have = k;
    }
    if (left <= 0) continue;
    const float step = s_step, root = s_root, keep = t.keep;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float gs = __fmul_rn(g[u], scale);
      m[u] = __fadd_rn(__fmul_rn(m[u], s.b1), __fmul_rn(gs, s.c1));
      v[u] = __fadd_rn(__fmul_rn(v[u], s.b2), __fmul_rn(__fmul_rn(gs, gs), s.c2));
      const float sq = __fsqrt_rn(v[u]);
      p[u] = p[u] * keep - step * __fdividef(m[u], sq * root + s.eps);
      if (EIGHT) v[u] = sq;
    }
    if (MASTER) store8(t.master + e0, vec, left, lane, p);
    store8((P *) t.param + e0, vec, left, lane, p);
    if (EIGHT) {
      const float mt = warp_max_abs(m), vt = warp_max_abs(v);
      // a block of nothing but zeros (or denormals) has scale 0 and values 0
      const bool mz = mt < kTiny, vz = vt < kTiny;
      const float mr = mz ? 0.0f : __fmul_rn(__frcp_rn(mt), kTop), vr = vz ? 0.0f : __fmul_rn(__frcp_rn(vt), kTop);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        m[u] = __fmul_rn(m[u], mr);
        const float y = __fmul_rn(v[u], vr);
        v[u] = y > 0.0f && y < kLow ? kLow : y;
      }
      if (lane == 0) {
        t.m_scale[e0 / kOptBlock] = mz ? 0.0f : __fdiv_rn(mt, kTop);
        t.v_scale[e0 / kOptBlock] = vz ? 0.0f : __fdiv_rn(vt, kTop);
      }
    }
    store8((S *) t.m + e0, vec, left, lane, m);
    store8((S *) t.v + e0, vec, left, lane, v);
  }
  // the block that finishes last counts the step: by then every block has read the counts
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(s.ticket, 1) == (int) gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  for (int k = threadIdx.x; k < a.n; k += kOptThreads) *a.t[k].step += 1.0f;
  if (threadIdx.x == 0) *s.ticket = 0;
}

template <typename P, typename G, bool EIGHT, bool MASTER>
static int adamw_launch(const AdamWTable &a, const AdamWScalars &s, cudaStream_t st) {
  int dev = 0, sms = 0, per_sm = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, adamw_kernel<P, G, EIGHT, MASTER>, kOptThreads, 0) != cudaSuccess)
    return FSGS_ERR_LAUNCH;
  const int total = a.chunk_start[a.n], most = sms * (per_sm > 0 ? per_sm : 1);
  adamw_kernel<P, G, EIGHT, MASTER><<<total < most ? (total > 0 ? total : 1) : most, kOptThreads, 0, st>>>(a, s);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

template <typename P, typename G>
static int adamw_pick(bool eight, bool master, const AdamWTable &a, const AdamWScalars &s, cudaStream_t st) {
  if (eight) return master ? adamw_launch<P, G, true, true>(a, s, st) : adamw_launch<P, G, true, false>(a, s, st);
  return master ? adamw_launch<P, G, false, true>(a, s, st) : adamw_launch<P, G, false, false>(a, s, st);
}

// ------------------------------------------------------------------------------------------------
// the norm of all gradients
// ------------------------------------------------------------------------------------------------

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

constexpr int kNormChunk = 4 * kOptChunk;
constexpr int kNormSlots = FSGS_GRAD_NORM_SLOTS;

struct NormArgs {
  double *slots;
  int *ticket;
  float *out;
  float max_norm;
  int filled;  // slots written by earlier launches of the same call
  int last;    // this launch closes the sum
};

// Sum of the squares of this thread's elements of a chunk.  Eight squares are added in float32 and the eights in double:
// the float32 part rounds each eight by 4 x 2^-24 at most, and no sum of squares leaves the range of double unless a
// single eight leaves that of float32 (|g| > 6e18: the norm comes out infinite and the step is dropped).
template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, bool vec, long long left, int warp, int lane) {
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < kNormChunk / kOptChunk; ++j) {
    const long long e0 = (long long) j * kOptChunk + warp * kOptBlock;
    if (left - e0 > 0) {
      float x[8];
      load8(p + e0, vec, left - e0, lane, x);
      float q = 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) q = fmaf(x[u], x[u], q);
      sum += (double) q;
    }
  }
  return sum;
}

__global__ void __launch_bounds__(kOptThreads) grad_norm_kernel(const __grid_constant__ NormTable a, const NormArgs s) {
  __shared__ double s_sum[kOptThreads / 32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int total = a.chunk_start[a.n];
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < total; chunk += gridDim.x) {
    const int k = tensor_of(a, chunk);
    const long long e0 = (long long) (chunk - a.chunk_start[k]) * kNormChunk;
    const long long left = a.t[k].numel - e0;
    const bool vec = a.vec[k] != 0;
    if (a.type[k] == FSGS_F32) sum += chunk_squares((const float *) a.t[k].data + e0, vec, left, warp, lane);
    else if (a.type[k] == FSGS_BF16) sum += chunk_squares((const __nv_bfloat16 *) a.t[k].data + e0, vec, left, warp, lane);
    else sum += chunk_squares((const __half *) a.t[k].data + e0, vec, left, warp, lane);
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kOptThreads / 32; ++w) t += s_sum[w];
    s.slots[blockIdx.x] = (int) blockIdx.x < s.filled ? s.slots[blockIdx.x] + t : t;
    __threadfence();
    s_last = s.last && atomicAdd(s.ticket, 1) == (int) gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  // the last block adds the slots in a fixed order: the same gradients give the same norm, bit for bit
  const int n = max(s.filled, (int) gridDim.x);
  sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kOptThreads) sum += __ldcg(s.slots + i);
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int w = 0; w < kOptThreads / 32; ++w) t += s_sum[w];
    const float norm = (float) sqrt(t);
    // a norm that is not a number or infinite: factor 0, which drops the step that is given it
    s.out[0] = norm;
    s.out[1] = norm < INFINITY ? fminf(1.0f, __fmul_rn(__frcp_rn(__fadd_rn(norm, 1e-6f)), s.max_norm)) : 0.0f;
    *s.ticket = 0;
  }
}

static int type_bytes(int type) { return type == FSGS_F32 ? 4 : 2; }
static bool is_type(int type) { return type == FSGS_F32 || type == FSGS_BF16 || type == FSGS_F16; }

}  // namespace fsgs

using namespace fsgs;

extern "C" int fsgs_adamw_multi(int n_tensors, const fsgs_adamw_tensor *tensors, int param_type, int grad_type,
    int state_bits, double beta1, double beta2, float eps, const float *grad_scale, const float *gate, int32_t *ticket,
    fsgs_stream_t stream) {
  FSGS_REQUIRE(n_tensors >= 0 && (tensors || n_tensors == 0) && ticket && is_type(param_type) && is_type(grad_type));
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
  AdamWScalars s;
  s.b1 = (float) beta1, s.b2 = (float) beta2, s.c1 = (float) (1.0 - beta1), s.c2 = (float) (1.0 - beta2), s.eps = eps;
  s.log_b1 = log(beta1), s.log_b2 = log(beta2);  // beta 0: -infinity, whose exponential is 0
  s.grad_scale = grad_scale, s.gate = gate, s.ticket = ticket;
  const uintptr_t pa = 4 * type_bytes(param_type) - 1, ga = 4 * type_bytes(grad_type) - 1, sa = eight ? 3 : 15;
  for (int first = 0; first < n_tensors;) {
    AdamWTable a;
    a.n = 0, a.chunk_start[0] = 0;
    int64_t chunks = 0;
    for (; first < n_tensors && a.n < kOptCapacity; ++first) {
      const fsgs_adamw_tensor &t = tensors[first];
      const int64_t c = (t.numel + kOptChunk - 1) / kOptChunk;
      if (c > INT32_MAX - (1 << 20)) return FSGS_ERR_LIMIT;
      if (chunks + c > INT32_MAX - (1 << 20)) break;  // the rest in a launch of its own
      AdamWEntry &d = a.t[a.n];
      d.param = t.param, d.grad = t.grad, d.m = t.exp_avg, d.v = t.exp_avg_sq, d.m_scale = t.exp_avg_scale;
      d.v_scale = t.exp_avg_sq_scale, d.master = t.master, d.step = t.step, d.numel = t.numel, d.lr = t.lr;
      d.keep = (float) (1.0 - (double) t.lr * (double) t.weight_decay);
      a.vec[a.n] = !(((uintptr_t) t.param & pa) | ((uintptr_t) t.grad & ga) | ((uintptr_t) t.exp_avg & sa) |
                     ((uintptr_t) t.exp_avg_sq & sa) | ((uintptr_t) t.master & 15));
      chunks += c;
      a.chunk_start[++a.n] = (int) chunks;
    }
    cudaStream_t st = (cudaStream_t) stream;
    int rc;
    if (param_type == FSGS_F32) rc = eight ? adamw_launch<float, float, true, false>(a, s, st) : adamw_launch<float, float, false, false>(a, s, st);
    else if (param_type == FSGS_BF16)
      rc = grad_type == FSGS_F32 ? adamw_pick<__nv_bfloat16, float>(eight, master, a, s, st)
                                 : adamw_pick<__nv_bfloat16, __nv_bfloat16>(eight, master, a, s, st);
    else
      rc = grad_type == FSGS_F32 ? adamw_pick<__half, float>(eight, master, a, s, st)
                                 : adamw_pick<__half, __half>(eight, master, a, s, st);
    if (rc != FSGS_OK) return rc;
  }
  return FSGS_OK;
}

extern "C" size_t fsgs_grad_norm_workspace_bytes(void) { return 16 + sizeof(double) * kNormSlots; }

extern "C" int fsgs_grad_norm(int n_tensors, const fsgs_norm_tensor *tensors, float max_norm, void *workspace,
    size_t workspace_bytes, float *out, fsgs_stream_t stream) {
  FSGS_REQUIRE(n_tensors >= 0 && (tensors || n_tensors == 0) && out && max_norm > 0.0f);
  if (!workspace || ((uintptr_t) workspace & 15) || workspace_bytes < fsgs_grad_norm_workspace_bytes()) return FSGS_ERR_WORKSPACE;
  for (int k = 0; k < n_tensors; ++k)
    FSGS_REQUIRE(tensors[k].numel >= 0 && is_type(tensors[k].type) && (tensors[k].data || tensors[k].numel == 0));
  NormArgs s;
  s.ticket = (int *) workspace, s.slots = (double *) ((char *) workspace + 16), s.out = out, s.max_norm = max_norm, s.filled = 0;
  int first = 0;
  do {  // at least one launch: no tensors have norm 0
    NormTable a;
    a.n = 0, a.chunk_start[0] = 0;
    int64_t chunks = 0;
    for (; first < n_tensors && a.n < kOptCapacity; ++first) {
      const fsgs_norm_tensor &t = tensors[first];
      const int64_t c = (t.numel + kNormChunk - 1) / kNormChunk;
      if (c > INT32_MAX - (1 << 20)) return FSGS_ERR_LIMIT;
      if (chunks + c > INT32_MAX - (1 << 20)) break;
      a.t[a.n].data = t.data, a.t[a.n].numel = t.numel, a.type[a.n] = (uint8_t) t.type;
      a.vec[a.n] = ((uintptr_t) t.data & (4 * type_bytes(t.type) - 1)) == 0;
      chunks += c;
      a.chunk_start[++a.n] = (int) chunks;
    }
    s.last = first >= n_tensors;
    const int grid = chunks < kNormSlots ? (chunks > 0 ? (int) chunks : 1) : kNormSlots;
    grad_norm_kernel<<<grid, kOptThreads, 0, (cudaStream_t) stream>>>(a, s);
    FSGS_LAUNCH_CHECK();
    if (grid > s.filled) s.filled = grid;
  } while (first < n_tensors);
  return FSGS_OK;
}
