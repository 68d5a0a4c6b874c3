// Balance loss over the superpoints, their counts, and its gradients.
//
// N Gaussians are bound to K of M superpoints each: idx [N,K].  With c_m the number of pairs that name superpoint m
// (rows that the mask leaves out and indices outside 0 .. M-1 do not count), T = sum c, n the rows that count,
//   L = M sum_m (c_m / T) P_m,     P_m = (1/n) sum of the weights of the pairs that name m           (pairs form)
//                                  P_m = (1/n) sum_i softmax(table_i)_m                              (table form)
// L is 1 where every superpoint has its share and grows as few of them take most.  The counts carry no gradient:
//   dL/dw_ik = M c_idx / (T n),    dL/dz_im = M/(T n) p_im (c_m - sum_e p_ie c_e).
// In the table form any constant may be taken off all c_m, because the p of a row add up to 1; with the mean T / M taken
// off the difference is between small numbers, where M c_m / T are all near 1 and their difference would lose the digits
// that they have in common.  The counts are integers, so the centred share (M c_m - T) / (T n) is exact up to its one
// rounding to float32.
//
// What bounds it: memory.  Pairs: 8 bytes of index, 4 of weight and 4 of gradient per pair and, between the two passes,
// 2 bytes of code that mostly stay in L2; table: the table in and its gradient out, once each.  Measured on one B200 (copy
// 6.57 TB/s; device time): 2 M x 8 pairs over 4096 superpoints 59 us, 30 counting (160 MB at 5.3 TB/s; neither the
// shared-memory atomics nor their flush show: 30.9 and 29.0 us without them) and 27 for loss and gradient (160 MB at 5.9
// TB/s); 300 k x 3 over 512 12 us in three nodes; table 300 k x 512 float32, value and gradient, 178 us (6.9 TB/s) and 12
// of counting and closing; bf16 171 us in all (3.7 TB/s, bound by instructions: 28 per column, about 10 of them the row's
// arithmetic, the others for rows off a boundary of four, partial groups and masked rows).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fsgs_common.cuh"
#include "fsgs_two.cuh"

namespace fsgs {

// Superpoints whose histogram or shares are kept in shared memory (32 KB).  Above, a pair is an atomic on a 64-bit count in
// memory: 2 M x 8 evenly over 8192 superpoints 62 us, over 8193 234 us, and 2.4 ms where a few of them take most pairs.
constexpr int kBalSharedPoints = 8192;
constexpr int kCountThreads = 1024;
constexpr int kPairThreads = 512;
constexpr int kTableThreads = 256;
constexpr int kBalSlots = 296;            // partial sums of the pairs form: two blocks an SM

// The workspace: this, then the codes of the pairs (pairs form) or four copies of the shares, copy s moved up by s places
// (table form).
struct BalanceHead {
  int closed, bad;          // pairs: blocks that have finished summing; table: a sum that is not finite
  long long dead;           // table: rows that count and have no probabilities
  double slots[kBalSlots];  // pairs: the blocks' sums; table: kFixedSlots sums in fixed point
};
constexpr int kFixedSlots = 32;

// floats of one copy of the shares
static inline __host__ __device__ size_t share_copy(int M) { return ((size_t) M + 3 + 3) & ~(size_t) 3; }

static inline size_t pad16(size_t n) { return (n + 15) & ~(size_t) 15; }
static inline size_t code_bytes(int M) { return M < 65536 ? 2 : 4; }

struct BalanceSpace {
  BalanceHead *head;
  float *share;    // table form
  void *codes;     // pairs form: [N K]
};

static BalanceSpace balance_space(void *ws) {
  BalanceSpace w;
  w.head = (BalanceHead *) ws;
  w.codes = (char *) ws + pad16(sizeof(BalanceHead));
  w.share = (float *) w.codes;
  return w;
}

// Table form: the sum over the rows of inner = sum_m p_m share_m is at most M + 1 in magnitude, any part of it too, and is
// added in whole numbers of 2^-fixed_bits: the order of the additions does not change it.
static inline __host__ __device__ int fixed_bits(int M) {
  int bits = 1;
  while (bits < 31 && (M >> bits) != 0) ++bits;
  return 60 - bits;
}

// ---- counts -----------------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ T block_total(T v, T *scratch) {  // valid in the first warp
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = lane < warps ? scratch[lane] : T(0);
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// One pass over the indices: a histogram per block in shared memory, added to the 64-bit counts at the end.  In the pairs
// form the superpoint of every pair is kept as a 16- or 32-bit code (all ones: does not count) for the pass that needs the
// complete counts, which then reads 2 bytes per pair instead of 8 and no mask, most of it from L2 (the indices are read,
// and the weights and gradients of that pass streamed, so as not to displace the codes).  In the table form the block that finishes
// last turns the counts into shares.  Bound by instructions, 41 per pair and 70 % of the issue slots at 2 M x 8 with a mask
// (quotient, mask and code beside the atomic on shared memory), next to the read of the indices at 5.3 TB/s.
template <typename Code, bool SHARED>
__global__ void __launch_bounds__(kCountThreads, 2) balance_count_kernel(long long N, int K, int M, const int64_t *__restrict__ idx,
    const uint8_t *__restrict__ mask, int wide, unsigned magic, unsigned long long *__restrict__ counts, BalanceHead *__restrict__ head,
    float *__restrict__ share, Code *__restrict__ codes) {
  extern __shared__ int s_hist[];   // [M + 1]: the last one takes what does not count
  __shared__ long long s_red[kCountThreads / 32];
  __shared__ int s_last;
  if (SHARED) {
    for (int m = threadIdx.x; m <= M; m += kCountThreads) s_hist[m] = 0;
    __syncthreads();
  }
  const long long pairs = N * K, stride = (long long) gridDim.x * kCountThreads;
  const long long first = (long long) blockIdx.x * kCountThreads + threadIdx.x;
  long long named = 0, rows = 0;
  auto take = [&](int64_t m, bool on) -> Code {
    const unsigned bin = on && (unsigned) (m >> 32) == 0 ? min((unsigned) m, (unsigned) M) : (unsigned) M;
    if (SHARED) {
      atomicAdd(s_hist + bin, 1);
    } else if (bin < (unsigned) M) {
      ++named;
      atomicAdd(counts + bin, 1ull);
    }
    return bin < (unsigned) M ? (Code) bin : (Code) ~(Code) 0;
  };
  const long long quads = wide ? pairs / 4 : 0;
  for (long long q = first; q < quads; q += stride) {
    const longlong2 a = __ldcs(reinterpret_cast<const longlong2 *>(idx) + 2 * q), b = __ldcs(reinterpret_cast<const longlong2 *>(idx) + 2 * q + 1);
    bool on[4] = {true, true, true, true};
    if (mask) {
      long long row;
      if (magic) {  // 4 q / K for 32-bit values: the high product is the quotient or one less
        unsigned r = __umulhi((unsigned) (4 * q), magic);
        if ((unsigned) (4 * q) - r * (unsigned) K >= (unsigned) K) ++r;
        row = r;
      } else {
        row = 4 * q / K;
      }
      int col = (int) (4 * q - row * K);
      if (K >= 4) {  // at most two rows
        const bool r0 = mask[row] != 0, r1 = col + 3 >= K ? mask[row + 1] != 0 : r0;
#pragma unroll
        for (int u = 0; u < 4; ++u) on[u] = col + u < K ? r0 : r1;
      } else {
        on[0] = mask[row] != 0;
#pragma unroll
        for (int u = 1; u < 4; ++u) {
          on[u] = on[u - 1];
          if (++col == K) col = 0, on[u] = mask[++row] != 0;
        }
      }
    }
    const Code c[4] = {take(a.x, on[0]), take(a.y, on[1]), take(b.x, on[2]), take(b.y, on[3])};
    if (codes) {
      if (sizeof(Code) == 2) reinterpret_cast<uint2 *>(codes)[q] = make_uint2(c[0] | ((unsigned) c[1] << 16), c[2] | ((unsigned) c[3] << 16));
      else reinterpret_cast<uint4 *>(codes)[q] = make_uint4(c[0], c[1], c[2], c[3]);
    }
  }
  for (long long e = 4 * quads + first; e < pairs; e += stride) {
    const Code c = take(idx[e], !mask || mask[e / K] != 0);
    if (codes) codes[e] = c;
  }
  if (mask)
    for (long long i = first; i < N; i += stride) rows += mask[i] != 0;
  __syncthreads();
  if (SHARED)
    for (int m = threadIdx.x; m < M; m += kCountThreads) {
      const int c = s_hist[m];
      if (c) atomicAdd(counts + m, (unsigned long long) c);
      named += c;
    }
  // both sums in one: below 2^31 each in a block
  const long long both = block_total((named << 32) + rows, s_red);
  if (threadIdx.x == 0) {
    const unsigned long long n = !mask ? blockIdx.x == 0 ? (unsigned long long) N : 0 : (unsigned long long) (both & 0xffffffffll);
    if (both >> 32) atomicAdd(counts + M, (unsigned long long) (both >> 32));
    if (n) atomicAdd(counts + M + 1, n);
    if (blockIdx.x == 0) head->closed = 0;
  }
  if (codes) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(counts + M + 2, 1ull) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const long long total = (long long) __ldcg(counts + M), n = (long long) __ldcg(counts + M + 1);
  const double unit = total > 0 && n > 0 ? 1.0 / ((double) total * (double) n) : 0.0;
  const size_t copy = share_copy(M);
  for (int m = threadIdx.x; m < M; m += kCountThreads) {
    const float f = (float) (((double) M * (double) (long long) __ldcg(counts + m) - (double) total) * unit);
#pragma unroll
    for (int k = 0; k < 4; ++k) share[k * copy + m + k] = f;
  }
  if (threadIdx.x < 4) {  // what a whole group reads beside its row's shares
    float *c = share + threadIdx.x * copy;
    for (int m = 0; m < (int) threadIdx.x; ++m) c[m] = 0.0f;
    for (size_t m = (size_t) M + threadIdx.x; m < copy; ++m) c[m] = 0.0f;
  }
  if (threadIdx.x < kFixedSlots) ((long long *) head->slots)[threadIdx.x] = 0;
  if (threadIdx.x == 0) head->bad = 0, head->dead = 0;
}

// ---- pairs form ---------------------------------------------------------------------------------------------

struct PairsArgs {
  long long pairs;
  int M, wide;
  const float *w;
  float scale;
  const float *upstream;             // null: 1
  float *loss, *g;                   // either may be null
  int accumulate;
  BalanceHead *head;
  const long long *counts;
};

// Eight pairs per thread and turn: 16 bytes of codes, 32 of weights in, 32 of gradients out, the shares from shared memory.
template <typename Code>
__global__ void __launch_bounds__(kPairThreads, 2) balance_pairs_kernel(PairsArgs a, const Code *__restrict__ codes) {
  extern __shared__ float s_share[];
  __shared__ double s_sum[kPairThreads / 32];
  __shared__ int s_last;
  const bool in_shared = a.M <= kBalSharedPoints;
  const long long stride = (long long) gridDim.x * kPairThreads, first = (long long) blockIdx.x * kPairThreads + threadIdx.x;
  const long long eights = a.wide ? a.pairs / 8 : 0;
  constexpr int kWords = sizeof(Code) / 2;  // 16-byte words of eight codes
  uint4 nc[kWords];
  float4 nw[2] = {};
  auto fetch = [&](long long q) {
#pragma unroll
    for (int u = 0; u < kWords; ++u) nc[u] = reinterpret_cast<const uint4 *>(codes)[kWords * q + u];
    if (a.loss) nw[0] = __ldcs(reinterpret_cast<const float4 *>(a.w) + 2 * q), nw[1] = __ldcs(reinterpret_cast<const float4 *>(a.w) + 2 * q + 1);
  };
  if (first < eights) fetch(first);
  const double parts = (double) a.counts[a.M] * (double) a.counts[a.M + 1], unit = parts > 0.0 ? (double) a.M / parts : 0.0;
  if (in_shared) {
    for (int m = threadIdx.x; m < a.M; m += kPairThreads) s_share[m] = (float) ((double) a.counts[m] * unit);
    __syncthreads();
  }
  const float up = a.scale * (a.upstream ? *a.upstream : 1.0f);
  double sum = 0.0;
  // Two products are added in float32, 2 x 2^-24 of each, and the twos in double: 3 x 2^-24 with the share's own rounding.
  // (Eight in float32 would be 9, a double product of every pair 0.5 us more at 2 M x 8.)
  // a weight that does not count is not read into the sum: it may be anything, a NaN too
  auto one = [&](Code c, float w, float &part) {
    const bool on = c != (Code) ~(Code) 0;
    const float share = !on ? 0.0f : in_shared ? s_share[c] : (float) ((double) a.counts[c] * unit);
    if (on) part = fmaf(w, share, part);
    return up * share;
  };
  for (long long q = first; q < eights; q += stride) {
    if (q != first) fetch(q);
    alignas(16) Code c[8];
    alignas(16) float w[8];
#pragma unroll
    for (int u = 0; u < kWords; ++u) reinterpret_cast<uint4 *>(c)[u] = nc[u];
    reinterpret_cast<float4 *>(w)[0] = nw[0], reinterpret_cast<float4 *>(w)[1] = nw[1];
    float g[8];
#pragma unroll
    for (int u = 0; u < 8; u += 2) {
      float part = 0.0f;
      g[u] = one(c[u], w[u], part), g[u + 1] = one(c[u + 1], w[u + 1], part);
      sum += (double) part;
    }
    if (a.g) {
      float4 *o = reinterpret_cast<float4 *>(a.g) + 2 * q;
      float4 x = make_float4(g[0], g[1], g[2], g[3]), y = make_float4(g[4], g[5], g[6], g[7]);
      if (a.accumulate) {
        const float4 ox = o[0], oy = o[1];
        x.x += ox.x, x.y += ox.y, x.z += ox.z, x.w += ox.w, y.x += oy.x, y.y += oy.y, y.z += oy.z, y.w += oy.w;
      }
      __stcs(o, x), __stcs(o + 1, y);
    }
  }
  for (long long e = 8 * eights + first; e < a.pairs; e += stride) {
    float part = 0.0f;
    const float g = one(codes[e], a.loss ? a.w[e] : 0.0f, part);
    sum += (double) part;
    if (a.g) a.g[e] = a.accumulate ? a.g[e] + g : g;
  }
  if (!a.loss) return;
  sum = block_total(sum, s_sum);
  if (threadIdx.x == 0) {
    a.head->slots[blockIdx.x] = sum;
    __threadfence();
    s_last = atomicAdd(&a.head->closed, 1) == (int) gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  // the block that arrives last adds the sums in a fixed order
  __threadfence();
  sum = 0.0;
  for (int i = threadIdx.x; i < (int) gridDim.x; i += kPairThreads) sum += __ldcg(a.head->slots + i);
  sum = block_total(sum, s_sum);
  if (threadIdx.x == 0) *a.loss = (float) (sum * (double) up), a.head->closed = 0;
}

// ---- table form ---------------------------------------------------------------------------------------------

struct TableArgs {
  long long N, stride, g_stride;     // row strides in elements
  int M;
  const void *table;
  const uint8_t *mask;
  float scale;
  const float *upstream;
  void *g;
  const float *share;
  BalanceHead *head;                 // null: no loss
  bool eager;
};

__device__ __forceinline__ float get(const float *p) { return *p; }
__device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
// four neighbouring elements, as they lie in memory and as float32
template <typename T>
struct Four {
  uint2 a;
};
template <>
struct Four<float> {
  float4 a;
};
template <typename T>
__device__ __forceinline__ Four<T> load4(const T *p) { return *reinterpret_cast<const Four<T> *>(p); }
__device__ __forceinline__ void open4(const Four<float> &v, float *x) { x[0] = v.a.x, x[1] = v.a.y, x[2] = v.a.z, x[3] = v.a.w; }
__device__ __forceinline__ void open4(const Four<__nv_bfloat16> &v, float *x) {
  x[0] = __uint_as_float(v.a.x << 16), x[1] = __uint_as_float(v.a.x & 0xffff0000u);
  x[2] = __uint_as_float(v.a.y << 16), x[3] = __uint_as_float(v.a.y & 0xffff0000u);
}
__device__ __forceinline__ void open4(const Four<__half> &v, float *x) {
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.a.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.a.y));
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void put4(float *p, const float *x) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void put4(__nv_bfloat16 *p, const float *x) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}
__device__ __forceinline__ void put4(__half *p, const float *x) {
  const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
}

// max / sum over the G threads that share a row (part of a warp, a warp, or the block); NaN are passed over by the max
template <int G>
__device__ __forceinline__ float row_max(float v, float *scratch) {
  if (G < 32) {
    for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(v) : "f"(v));
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < G / 32; ++w) v = fmaxf(v, scratch[w]);
  }
  return v;
}
template <int G>
__device__ __forceinline__ float2 row_sum(float2 v, float2 *scratch) {
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < G / 32; ++w) v.x += scratch[w].x, v.y += scratch[w].y;
  }
  return v;
}

__device__ __forceinline__ float max3(float x, float y, float z) {  // passes over NaN, as fmaxf does
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// G threads per row, one row each, PER columns per thread in groups of four neighbours (PER 0: any number of columns, the
// row is read again for each of three passes).  The groups are those of memory: where a row starts s elements past a
// boundary of four, group k holds columns 4 k - s .. 4 k - s + 3, so that groups are one access whatever the width of the
// table, and the shares come from the copy that is moved up by s.  What a group holds beside its row belongs to the
// neighbouring rows; it is read and not used (the first and the last rows read element by element where there is no such
// neighbour).  exp(z - max) is the hardware's exp2 of (z - max) log2(e); the difference is taken first, because z log2(e)
// overflows for the type's lowest value, which stands for masked columns in places.  Both are rounded, so an exponential is
// 2^-23 times the row's range off beside the 2 units of exp2, and the sum's inverse is the approximate one (2 units): loss and
// gradient stay within 8.1e-8 of 64 bits where separate float32 operations are at 7.6e-8 (300 k x 512).  The row stays in registers from its
// one read to the write of its gradient; the grid covers the rows and leaves the order to the hardware.
template <typename T, int G, int PER, int ROWS>
__global__ void __launch_bounds__(kTableThreads) balance_table_kernel(TableArgs a) {
  constexpr float kLog2e = 1.44269504f;
  constexpr int kGroups = kTableThreads / G;
  __shared__ float s_max[kTableThreads / 32];
  __shared__ float2 s_sum[kTableThreads / 32];
  __shared__ float s_inner[kGroups * ROWS];  // of the block's rows; NaN and infinities pass through
  __shared__ int s_dead[kGroups * ROWS];
  const int t = threadIdx.x % G;
  const float up = a.scale * (a.upstream ? *a.upstream : 1.0f);
  auto row_of = [&](int r) { return ((long long) blockIdx.x * ROWS + r) * kGroups + threadIdx.x / G; };
  // the table goes on for three elements before and behind this row
  auto inside = [&](long long i) { return i * a.stride >= 3 && (a.N - 1 - i) * a.stride >= 3; };
  auto moved_of = [&](const T *z) { return (int) ((uintptr_t) z / sizeof(T) & 3); };
  Four<T> raw[ROWS][PER > 0 ? PER / 4 : 1];
  bool on[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const long long i = row_of(r);
    on[r] = i < a.N && (!a.mask || a.mask[i] != 0);
    const T *z = (const T *) a.table + (i < a.N ? i : 0) * a.stride;
    const int moved = moved_of(z);
    const bool past = i < a.N && inside(i), read = a.eager ? i < a.N : on[r];  // eager: not wait for the mask before the row
#pragma unroll
    for (int u = 0; u < PER; u += 4) {
      const int m = u * G + 4 * t - moved;
      if (read && m < a.M && (past || (m >= 0 && m + 4 <= a.M))) raw[r][u / 4] = load4(z + m);
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const long long i = row_of(r);
    const T *z = (const T *) a.table + (i < a.N ? i : 0) * a.stride;
    T *g = a.g && i < a.N ? (T *) a.g + i * a.g_stride : nullptr;
    const int moved = moved_of(z);
    const float *copy = a.share + moved * share_copy(a.M);  // copy[m + moved] = share of m
    float x[PER > 0 ? PER : 1];  // values, then exponentials
    float top = -INFINITY;
    if (PER > 0) {
      const bool past = i < a.N && inside(i);
#pragma unroll
      for (int u = 0; u < PER; u += 4) {
        const int m = u * G + 4 * t - moved;
        const bool part = m < 0 || m + 4 > a.M;
        if (!on[r] || m >= a.M) {
#pragma unroll
          for (int j = 0; j < 4; ++j) x[u + j] = -INFINITY;
          continue;
        }
        open4(raw[r][u / 4], x + u);
        if (part) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool in = m + j >= 0 && m + j < a.M;
            if (in && !past) x[u + j] = get(z + m + j);
            if (!in) x[u + j] = -INFINITY;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < PER; u += 4) top = max3(max3(top, x[u], x[u + 1]), x[u + 2], x[u + 3]);
    } else if (on[r]) {
      for (int m = t; m < a.M; m += G) top = fmaxf(top, get(z + m));
    }
    top = row_max<G>(top, s_max);
    // a row of nothing but -infinity has no probabilities: it adds nothing and has no gradient
    const float base = top == -INFINITY ? 0.0f : top;
    float2 s = make_float2(0.0f, 0.0f);
    if (PER > 0) {
      Two sx = both(0.0f), sy = both(0.0f);
#pragma unroll
      for (int u = 0; u < PER; u += 4) {
        if (u * G + 4 * t - moved >= a.M) continue;
        const float4 sh = *reinterpret_cast<const float4 *>(copy + u * G + 4 * t);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          split(mul2(add2(two(x[u + j], x[u + j + 1]), both(-base)), both(kLog2e)), x[u + j], x[u + j + 1]);
          const Two e = two(x[u + j] = fast_exp2(x[u + j]), x[u + j + 1] = fast_exp2(x[u + j + 1]));
          sx = add2(sx, e), sy = fma2(e, j ? two(sh.z, sh.w) : two(sh.x, sh.y), sy);
        }
      }
      float hx, hy;
      split(sx, s.x, hx), split(sy, s.y, hy);
      s.x += hx, s.y += hy;
    } else if (on[r]) {
      for (int m = t; m < a.M; m += G) {
        const float e = fast_exp2((get(z + m) - base) * kLog2e);
        s.x += e, s.y = fmaf(e, copy[m + moved], s.y);
      }
    }
    s = row_sum<G>(s, s_sum);
    const float inv = s.x == 0.0f ? 0.0f : __fdividef(1.0f, s.x), inner = s.y * inv;
    if (g) {
      const float k = up * inv, less = -k * inner;
      const bool alike = moved_of(g) == moved;  // the gradient's groups lie as the table's
      if (PER > 0) {
#pragma unroll
        for (int u = 0; u < PER; u += 4) {
          const int m = u * G + 4 * t - moved;
          if (m >= a.M) continue;
          const float4 sh = *reinterpret_cast<const float4 *>(copy + u * G + 4 * t);
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const Two f = fma2(both(k), j ? two(sh.z, sh.w) : two(sh.x, sh.y), both(less));
            split(mul2(two(x[u + j], x[u + j + 1]), f), x[u + j], x[u + j + 1]);
            if (!on[r]) x[u + j] = x[u + j + 1] = 0.0f;
          }
          if (alike && m >= 0 && m + 4 <= a.M) {
            put4(g + m, x + u);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (m + j >= 0 && m + j < a.M) put(g + m + j, x[u + j]);
          }
        }
      } else {
        for (int m = t; m < a.M; m += G)
          put(g + m, on[r] ? fast_exp2((get(z + m) - base) * kLog2e) * fmaf(k, copy[m + moved], less) : 0.0f);
      }
    }
    if (a.head && t == 0)
      s_inner[r * kGroups + threadIdx.x / G] = on[r] ? inner : 0.0f, s_dead[r * kGroups + threadIdx.x / G] = on[r] && s.x == 0.0f;
  }
  if (!a.head) return;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.0;
    int dead = 0;
    for (int r = 0; r < kGroups * ROWS; ++r) sum += (double) s_inner[r], dead += s_dead[r];
    const bool fine = fabs(sum) <= 2.0 * a.M;
    if (fine) atomicAdd((unsigned long long *) a.head->slots + blockIdx.x % kFixedSlots,
                        (unsigned long long) __double2ll_rn(ldexp(sum, fixed_bits(a.M))));
    else atomicOr(&a.head->bad, 1);
    if (dead) atomicAdd((unsigned long long *) &a.head->dead, (unsigned long long) dead);
  }
}

// The loss from the sums; rows with probabilities add 1 / n each, what the shares were centred by.  Leaves the sums at zero.
__global__ void __launch_bounds__(32) balance_close_kernel(BalanceHead *head, const long long *__restrict__ counts, int M, float scale,
    const float *__restrict__ upstream, float *__restrict__ loss) {
  long long *slot = (long long *) head->slots + threadIdx.x, sum = *slot;
  *slot = 0;
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x != 0) return;
  const double n = (double) counts[M + 1], up = (double) (scale * (upstream ? *upstream : 1.0f));
  const double value = n > 0.0 && counts[M] > 0 ? ldexp((double) sum, -fixed_bits(M)) + (n - (double) head->dead) / n : 0.0;
  *loss = head->bad ? NAN : (float) (value * up);
  head->bad = 0, head->dead = 0;
}
static_assert(kFixedSlots == 32, "one warp closes the sum");

template <typename T, int G, int PER, int ROWS>
static int table_launch(TableArgs &a, cudaStream_t st) {
  const int rows = kTableThreads / G * ROWS;
  const int64_t blocks = (a.N + rows - 1) / rows;
  if (blocks > INT32_MAX) return FSGS_ERR_LIMIT;
  if (blocks == 0) return FSGS_OK;
  // Rows are loaded beside their mask in calls of a few waves, where waiting for it shows, and only if they count in longer
  // ones, where what they would read does (us, value and gradient, eager | after the mask; 3 % masked, then half): 20 k x
  // 333 bf16 24.6 | 25.4, 25.5 | 25.5; 20 k x 512 float32 20.9 | 20.8, 22.3 | 21.3; 60 k x 512 float32 (7500 blocks) 52.0 |
  // 51.4, 51.6 | 46.7; 300 k x 512 float32 202 | 200, 201 | 179, bf16 174 | 188, 172 | 181.
  a.eager = blocks <= 4096;
  balance_table_kernel<T, G, PER, ROWS><<<(int) blocks, kTableThreads, 0, st>>>(a);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

// Threads per row: as few as the registers allow, so that many columns share a row's reductions and addresses; tables of
// 16 bits, whose rows are instructions rather than bytes, have the next row's loads under way meanwhile.  Measured, value
// and gradient (us; one row a thread group | two): 300 k x 512 bf16 177 | 171, 400 k x 256 bf16 140 | 123, 1 M x 100 bf16
// 148 | 155, 2 M x 40 bf16 209 | 189; float32 is bound by memory (300 k x 512: 190 us, 6.5 TB/s) and takes one.  A warp
// per row reaches to 1024 columns (100 k x 1000: 138 us, a block per row 244), a block per row lies above.  Rows of more than
// 8192 columns do not fit the registers and are read three times: 12 k x 8192 float32 141 us (5.6 TB/s), 12 k x 8200 192,
// 12 k x 20 000 655 (2.9 TB/s); bf16 150, 151.
//
// `reach`: columns from the first group of four to the row's end, M where every row starts on a boundary of four elements.
template <typename T>
static int table_pick(TableArgs &a, int reach, cudaStream_t st) {
  constexpr int R = sizeof(T) == 2 ? 2 : 1;
  if (reach <= 64) return table_launch<T, 8, 8, R>(a, st);
  if (reach <= 128) return table_launch<T, 8, 16, 1>(a, st);
  if (reach <= 256) return table_launch<T, 16, 16, R>(a, st);
  if (reach <= 384) return table_launch<T, 32, 12, R>(a, st);
  if (reach <= 512) return table_launch<T, 32, 16, R>(a, st);
  if (reach <= 768) return table_launch<T, 32, 24, 1>(a, st);
  if (reach <= 1024) return table_launch<T, 32, 32, 1>(a, st);
  if (reach <= 2048) return table_launch<T, 256, 8, 1>(a, st);
  if (reach <= 4096) return table_launch<T, 256, 16, 1>(a, st);
  if (reach <= 8192) return table_launch<T, 256, 32, 1>(a, st);
  return table_launch<T, 256, 0, 1>(a, st);  // reads the row three times
}

static bool balance_sizes(int64_t N, int64_t per_row) { return N <= (1ll << 36) / per_row; }

static int balance_blocks(int64_t work, int threads, int most) {
  const int64_t blocks = (work + threads - 1) / threads;
  return (int) (blocks < 1 ? 1 : blocks < most ? blocks : most);
}

}  // namespace fsgs

using namespace fsgs;

extern "C" size_t fsgs_balance_workspace_bytes(int64_t N, int K, int M, int form) {
  const bool table = form == FSGS_BALANCE_TABLE;
  if (N < 0 || K <= 0 || M <= 0 || !balance_sizes(N, table && M > K ? M : K) || (!table && form != FSGS_BALANCE_PAIRS)) return 0;
  return pad16(sizeof(BalanceHead)) + (table ? 4 * sizeof(float) * share_copy(M) : pad16((size_t) N * K * code_bytes(M)));
}

static bool balance_workspace(int64_t N, int K, int M, int form, const void *workspace, size_t bytes) {
  return workspace && ((uintptr_t) workspace & 15) == 0 && bytes >= fsgs_balance_workspace_bytes(N, K, M, form);
}

extern "C" int fsgs_balance_count(int64_t N, int K, int M, const int64_t *idx, const uint8_t *mask, int form, int64_t *counts,
    void *workspace, size_t workspace_bytes, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && K > 0 && M > 0 && counts && (idx || N == 0) && (form == FSGS_BALANCE_PAIRS || form == FSGS_BALANCE_TABLE));
  if (!balance_sizes(N, form == FSGS_BALANCE_TABLE && M > K ? M : K)) return FSGS_ERR_LIMIT;
  if (!balance_workspace(N, K, M, form, workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t) stream;
  const BalanceSpace w = balance_space(workspace);
  if (cudaMemsetAsync(counts, 0, sizeof(int64_t) * ((size_t) M + 4), st) != cudaSuccess) return FSGS_ERR_LAUNCH;
  const int grid = balance_blocks((N * K + 3) / 4, kCountThreads, 2 * 148);
  const size_t smem = M <= kBalSharedPoints ? sizeof(int) * ((size_t) M + 1) : 0;
  unsigned long long *c = (unsigned long long *) counts;
  const int wide = ((uintptr_t) idx & 15) == 0;
  const unsigned magic = K > 1 && N * K < (1ll << 32) ? (unsigned) ((1ull << 32) / (unsigned) K) : 0u;
  void *codes = form == FSGS_BALANCE_PAIRS ? w.codes : nullptr;
  const auto kernel32 = balance_count_kernel<uint32_t, false>;  // 65536 superpoints and more are never in shared memory
  if (M <= kBalSharedPoints) balance_count_kernel<uint16_t, true><<<grid, kCountThreads, smem, st>>>(N, K, M, idx, mask, wide, magic, c, w.head, w.share, (uint16_t *) codes);
  else if (code_bytes(M) == 2) balance_count_kernel<uint16_t, false><<<grid, kCountThreads, 0, st>>>(N, K, M, idx, mask, wide, magic, c, w.head, w.share, (uint16_t *) codes);
  else kernel32<<<grid, kCountThreads, 0, st>>>(N, K, M, idx, mask, wide, magic, c, w.head, w.share, (uint32_t *) codes);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_pairs(int64_t N, int K, int M, const float *weights, const int64_t *counts, void *workspace,
    size_t workspace_bytes, float scale, const float *upstream, float *loss, float *g_weights, int accumulate, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && K > 0 && M > 0 && counts && (weights || !loss || N == 0));
  if (!balance_sizes(N, K)) return FSGS_ERR_LIMIT;
  if (!balance_workspace(N, K, M, FSGS_BALANCE_PAIRS, workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_weights || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  const BalanceSpace w = balance_space(workspace);
  const int wide = (((uintptr_t) weights | (uintptr_t) g_weights) & 15) == 0;
  const PairsArgs a = {N * K, M, wide, weights, scale, upstream, loss, g_weights, accumulate, w.head, (const long long *) counts};
  const int grid = balance_blocks((N * K + 7) / 8, kPairThreads, kBalSlots);
  const size_t smem = M <= kBalSharedPoints ? sizeof(float) * (size_t) M : 0;
  if (code_bytes(M) == 2) balance_pairs_kernel<uint16_t><<<grid, kPairThreads, smem, st>>>(a, (const uint16_t *) w.codes);
  else balance_pairs_kernel<uint32_t><<<grid, kPairThreads, smem, st>>>(a, (const uint32_t *) w.codes);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_table(int64_t N, int M, int type, const void *table, int64_t row_stride, const uint8_t *mask,
    const int64_t *counts, void *workspace, size_t workspace_bytes, float scale, const float *upstream, float *loss, void *g_table,
    int64_t g_row_stride, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && M > 0 && (counts || !loss) && (table || N == 0) && row_stride >= M && (!g_table || g_row_stride >= M));
  FSGS_REQUIRE(type == FSGS_F32 || type == FSGS_BF16 || type == FSGS_F16);
  if (!balance_sizes(N, M)) return FSGS_ERR_LIMIT;
  if (!balance_workspace(N, 1, M, FSGS_BALANCE_TABLE, workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_table || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  const BalanceSpace w = balance_space(workspace);
  const bool plain = row_stride % 4 == 0 && (uintptr_t) table % (type == FSGS_F32 ? 16 : 8) == 0;
  const int reach = M + (plain ? 0 : 3);
  TableArgs a = {N, row_stride, g_row_stride, M, table, mask, scale, upstream, g_table, w.share, loss ? w.head : nullptr, false};
  const int rc = type == FSGS_F32 ? table_pick<float>(a, reach, st) : type == FSGS_BF16 ? table_pick<__nv_bfloat16>(a, reach, st)
                                                                                  : table_pick<__half>(a, reach, st);
  if (rc != FSGS_OK) return rc;
  if (!loss) return FSGS_OK;
  balance_close_kernel<<<1, kFixedSlots, 0, st>>>(w.head, (const long long *) counts, M, scale, upstream, loss);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}
