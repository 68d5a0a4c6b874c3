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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fsgs_common.cuh"

namespace fsgs {

constexpr int kBalSharedPoints = 8192;    // superpoints whose histogram or shares are kept in shared memory (32 KB)
constexpr int kCountThreads = 1024;
constexpr int kPairThreads = 512;
constexpr int kTableThreads = 256;
constexpr int kBalSlots = 1184;           // partial sums of the pairs form

// The workspace: this, the share of every superpoint as float32, then the codes of the pairs (pairs form) or the sums of
// the thread blocks (table form).
struct BalanceHead {
  int closed, pad;          // ticket: blocks that have finished summing
  double total, rows;       // T and n
  double slots[kBalSlots];
};

static inline size_t pad16(size_t n) { return (n + 15) & ~(size_t) 15; }
static inline size_t code_bytes(int M) { return M < 65536 ? 2 : 4; }

struct BalanceSpace {
  BalanceHead *head;
  float *share;
  void *codes;     // [N K]
  double *sums;    // [blocks]
};

static BalanceSpace balance_space(void *ws, int M) {
  BalanceSpace w;
  w.head = (BalanceHead *) ws;
  w.share = (float *) ((char *) ws + pad16(sizeof(BalanceHead)));
  w.codes = (char *) w.share + pad16(sizeof(float) * (size_t) M);
  w.sums = (double *) w.codes;
  return w;
}

// ---- counts -----------------------------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ T block_total(T v, T *scratch) {  // valid in thread 0
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < (int) (blockDim.x >> 5); ++w) v += scratch[w];
  return v;
}

// One pass over the indices: a histogram per block in shared memory, added to the 64-bit counts at the end.  In the pairs
// form the superpoint of every pair is kept as a 16- or 32-bit code (all ones: does not count) for the pass that needs the
// complete counts, which then reads 2 bytes per pair instead of 8 and no mask.  The block that finishes last turns the
// counts into shares.  Bound by the read of the indices and, beside it, by one shared-memory atomic per pair.
template <typename Code>
__global__ void __launch_bounds__(kCountThreads, 2) balance_count_kernel(long long N, int K, int M, const int64_t *__restrict__ idx,
    const uint8_t *__restrict__ mask, int wide, unsigned long long *__restrict__ counts, BalanceHead *__restrict__ head,
    float *__restrict__ share, Code *__restrict__ codes) {
  extern __shared__ int s_hist[];   // [M + 1]: the last one takes what does not count
  __shared__ long long s_red[kCountThreads / 32];
  __shared__ int s_last;
  const bool in_shared = M <= kBalSharedPoints;
  if (in_shared) {
    for (int m = threadIdx.x; m <= M; m += kCountThreads) s_hist[m] = 0;
    __syncthreads();
  }
  const long long pairs = N * K, stride = (long long) gridDim.x * kCountThreads;
  const long long first = (long long) blockIdx.x * kCountThreads + threadIdx.x;
  long long named = 0, rows = 0;
  auto take = [&](int64_t m, bool on) -> Code {
    on = on && (uint64_t) m < (uint64_t) M;
    if (in_shared) {
      atomicAdd(s_hist + (on ? (int) m : M), 1);
    } else if (on) {
      ++named;
      atomicAdd(counts + m, 1ull);
    }
    return on ? (Code) m : (Code) ~(Code) 0;
  };
  const long long quads = wide ? pairs / 4 : 0;
  for (long long q = first; q < quads; q += stride) {
    const longlong2 a = reinterpret_cast<const longlong2 *>(idx)[2 * q], b = reinterpret_cast<const longlong2 *>(idx)[2 * q + 1];
    bool on[4] = {true, true, true, true};
    if (mask) {
      long long row = pairs < (1ll << 32) ? (long long) ((unsigned) (4 * q) / (unsigned) K) : 4 * q / K;
      int col = (int) (4 * q - row * K);
      on[0] = mask[row] != 0;
#pragma unroll
      for (int u = 1; u < 4; ++u) {
        on[u] = on[u - 1];
        if (++col == K) col = 0, on[u] = mask[++row] != 0;
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
  if (in_shared)
    for (int m = threadIdx.x; m < M; m += kCountThreads) {
      const int c = s_hist[m];
      if (c) atomicAdd(counts + m, (unsigned long long) c);
      named += c;
    }
  named = block_total(named, s_red);
  rows = block_total(rows, s_red);
  if (threadIdx.x == 0) {
    if (named) atomicAdd(counts + M, (unsigned long long) named);
    if (!mask && blockIdx.x == 0) rows = N;
    if (rows) atomicAdd(counts + M + 1, (unsigned long long) rows);
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) s_last = atomicAdd(counts + M + 2, 1ull) == gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const long long total = (long long) __ldcg(counts + M), n = (long long) __ldcg(counts + M + 1);
  const bool any = total > 0 && n > 0;
  const double unit = any ? 1.0 / ((double) total * (double) n) : 0.0;
  const double mean = codes ? 0.0 : (double) total;
  for (int m = threadIdx.x; m < M; m += kCountThreads)
    share[m] = (float) (((double) M * (double) (long long) __ldcg(counts + m) - mean) * unit);
  if (threadIdx.x == 0) head->closed = 0, head->total = any ? (double) total : 0.0, head->rows = any ? (double) n : 0.0;
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
  const float *share;
};

// Eight pairs per thread and turn: 16 bytes of codes, 32 of weights in, 32 of gradients out, the shares from shared memory.
template <typename Code>
__global__ void __launch_bounds__(kPairThreads, 3) balance_pairs_kernel(PairsArgs a, const Code *__restrict__ codes) {
  extern __shared__ float s_share[];
  __shared__ double s_sum[kPairThreads / 32];
  __shared__ int s_last;
  const bool in_shared = a.M <= kBalSharedPoints;
  if (in_shared) {
    for (int m = threadIdx.x; m < a.M; m += kPairThreads) s_share[m] = a.share[m];
    __syncthreads();
  }
  const float up = a.scale * (a.upstream ? *a.upstream : 1.0f);
  double sum = 0.0;
  const long long stride = (long long) gridDim.x * kPairThreads, first = (long long) blockIdx.x * kPairThreads + threadIdx.x;
  // a weight that does not count is not read into the sum: it may be anything, a NaN too
  auto one = [&](Code c, float w, float &part) {
    const bool on = c != (Code) ~(Code) 0;
    const float share = !on ? 0.0f : in_shared ? s_share[c] : a.share[c];
    if (on) part = fmaf(w, share, part);
    return up * share;
  };
  const long long eights = a.wide ? a.pairs / 8 : 0;
  for (long long q = first; q < eights; q += stride) {
    alignas(16) Code c[8];
    if (sizeof(Code) == 2) {
      *reinterpret_cast<uint4 *>(c) = reinterpret_cast<const uint4 *>(codes)[q];
    } else {
      reinterpret_cast<uint4 *>(c)[0] = reinterpret_cast<const uint4 *>(codes)[2 * q];
      reinterpret_cast<uint4 *>(c)[1] = reinterpret_cast<const uint4 *>(codes)[2 * q + 1];
    }
    alignas(16) float w[8] = {};
    float g[8], part = 0.0f;
    if (a.loss) {
      *reinterpret_cast<float4 *>(w) = reinterpret_cast<const float4 *>(a.w)[2 * q];
      *reinterpret_cast<float4 *>(w + 4) = reinterpret_cast<const float4 *>(a.w)[2 * q + 1];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) g[u] = one(c[u], w[u], part);
    sum += (double) part;
    if (a.g) {
      float4 *o = reinterpret_cast<float4 *>(a.g) + 2 * q;
      float4 x = make_float4(g[0], g[1], g[2], g[3]), y = make_float4(g[4], g[5], g[6], g[7]);
      if (a.accumulate) {
        const float4 ox = o[0], oy = o[1];
        x.x += ox.x, x.y += ox.y, x.z += ox.z, x.w += ox.w, y.x += oy.x, y.y += oy.y, y.z += oy.z, y.w += oy.w;
      }
      o[0] = x, o[1] = y;
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
  double *sums;                      // null: no loss; one per block: sum of inner + rows / n
  const BalanceHead *head;
};

__device__ __forceinline__ float get(const float *p) { return *p; }
__device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void get4(const float *p, float *x) { *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(p); }
template <typename H>
__device__ __forceinline__ void get4(const H *p, float *x) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  const H *h = reinterpret_cast<const H *>(&v);
#pragma unroll
  for (int u = 0; u < 4; ++u) x[u] = get(h + u);
}
__device__ __forceinline__ void put4(float *p, const float *x) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
template <typename H>
__device__ __forceinline__ void put4(H *p, const float *x) {
  uint2 v;
  H *h = reinterpret_cast<H *>(&v);
#pragma unroll
  for (int u = 0; u < 4; ++u) put(h + u, x[u]);
  *reinterpret_cast<uint2 *>(p) = v;
}

// max / sum over the G threads that share a row (part of a warp, a warp, or the block)
template <int G>
__device__ __forceinline__ float row_max(float v, float *scratch) {
  for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// G threads per row, one row each, V neighbouring columns per access and PER columns per thread in all (PER 0: any number
// of columns, the row is read again for each of three passes).  The row stays in registers from its one read to the write
// of its gradient; the grid covers the rows and leaves the order to the hardware.
template <typename T, int G, int V, int PER>
__global__ void __launch_bounds__(kTableThreads) balance_table_kernel(TableArgs a) {
  __shared__ float s_max[kTableThreads / 32];
  __shared__ float2 s_sum[kTableThreads / 32];
  __shared__ double s_total[kTableThreads / 32];
  const int t = threadIdx.x % G;
  const long long i = (long long) blockIdx.x * (kTableThreads / G) + threadIdx.x / G;
  const bool here = i < a.N, on = here && (!a.mask || a.mask[i] != 0);
  const T *z = (const T *) a.table + (here ? i : 0) * a.stride;
  T *g = a.g && here ? (T *) a.g + i * a.g_stride : nullptr;
  constexpr int R = PER > 0 ? PER : V;
  alignas(16) float x[R], sh[R];  // values, then exponentials; shares
  float top = -INFINITY;
  if (PER > 0) {
#pragma unroll
    for (int u = 0; u < PER; u += V) {
      const int m = (u / V * G + t) * V;
      if (V == 4 && on && m + V <= a.M) {
        get4(z + m, x + u);
        get4(a.share + m, sh + u);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const bool in = on && m + j < a.M;
          x[u + j] = in ? get(z + m + j) : -INFINITY;
          sh[u + j] = in ? a.share[m + j] : 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) top = fmaxf(top, x[u]);  // passes over a NaN; the row's sum below does not
  } else if (on) {
    for (int m = t; m < a.M; m += G) top = fmaxf(top, get(z + m));
  }
  top = row_max<G>(top, s_max);
  // a row of nothing but -infinity has no probabilities: it adds nothing and has no gradient
  const float base = top == -INFINITY ? 0.0f : top;
  float2 s = make_float2(0.0f, 0.0f);
  if (PER > 0) {
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      x[u] = expf(x[u] - base);
      s.x += x[u], s.y = fmaf(x[u], sh[u], s.y);
    }
  } else if (on) {
    for (int m = t; m < a.M; m += G) {
      const float e = expf(get(z + m) - base);
      s.x += e, s.y = fmaf(e, a.share[m], s.y);
    }
  }
  s = row_sum<G>(s, s_sum);
  const float inv = s.x == 0.0f ? 0.0f : 1.0f / s.x, inner = s.y * inv;
  if (g) {
    const float k = a.scale * (a.upstream ? *a.upstream : 1.0f) * inv;
    if (PER > 0) {
#pragma unroll
      for (int u = 0; u < PER; u += V) {
        const int m = (u / V * G + t) * V;
        if (V == 4 && m + V <= a.M) {
#pragma unroll
          for (int j = 0; j < V; ++j) x[u + j] = on ? k * x[u + j] * (sh[u + j] - inner) : 0.0f;
          put4(g + m, x + u);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (m + j < a.M) put(g + m + j, on ? k * x[u + j] * (sh[u + j] - inner) : 0.0f);
        }
      }
    } else {
      for (int m = t; m < a.M; m += G) put(g + m, on ? k * expf(get(z + m) - base) * (a.share[m] - inner) : 0.0f);
    }
  }
  if (!a.sums) return;
  double sum = 0.0;
  if (t == 0 && on && s.x != 0.0f && a.head->rows > 0.0) sum = 1.0 / a.head->rows + (double) inner;
  sum = block_total(sum, s_total);
  if (threadIdx.x == 0) a.sums[blockIdx.x] = sum;
}

// The blocks' sums in a fixed order.
__global__ void __launch_bounds__(1024) balance_close_kernel(int n, const double *__restrict__ sums, float scale,
    const float *__restrict__ upstream, float *__restrict__ loss) {
  __shared__ double s_sum[32];
  double sum = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 1024) sum += sums[i];
  sum = block_total(sum, s_sum);
  if (threadIdx.x == 0) *loss = (float) (sum * (double) (scale * (upstream ? *upstream : 1.0f)));
}

static int rows_per_block(int M) { return M <= 64 ? kTableThreads / 8 : M <= 512 ? kTableThreads / 32 : 1; }

template <typename T, int G, int V, int PER>
static int table_launch(const TableArgs &a, cudaStream_t st) {
  balance_table_kernel<T, G, V, PER><<<(int) ((a.N + kTableThreads / G - 1) / (kTableThreads / G)), kTableThreads, 0, st>>>(a);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

template <typename T, int V>
static int table_pick(const TableArgs &a, cudaStream_t st) {
  if (a.M <= 64) return table_launch<T, 8, V, 8>(a, st);
  if (a.M <= 128) return table_launch<T, 32, V, 4>(a, st);
  if (a.M <= 256) return table_launch<T, 32, V, 8>(a, st);
  if (a.M <= 512) return table_launch<T, 32, V, 16>(a, st);
  if (a.M <= 1024) return table_launch<T, 256, V, 4>(a, st);
  if (a.M <= 2048) return table_launch<T, 256, V, 8>(a, st);
  if (a.M <= 4096) return table_launch<T, 256, V, 16>(a, st);
  if (a.M <= 8192) return table_launch<T, 256, V, 32>(a, st);
  return table_launch<T, 256, 1, 0>(a, st);
}

static bool balance_sizes(int64_t N, int64_t per_row) { return N <= (1ll << 36) / per_row; }

static int balance_blocks(int64_t work, int threads, int most) {
  const int64_t blocks = (work + threads - 1) / threads;
  return (int) (blocks < 1 ? 1 : blocks < most ? blocks : most);
}

}  // namespace fsgs

using namespace fsgs;

extern "C" size_t fsgs_balance_workspace_bytes(int64_t N, int K, int M, int form) {
  if (N < 0 || K <= 0 || M <= 0 || !balance_sizes(N, form == FSGS_BALANCE_TABLE && M > K ? M : K) || (form != FSGS_BALANCE_PAIRS && form != FSGS_BALANCE_TABLE)) return 0;
  const size_t more = form == FSGS_BALANCE_PAIRS ? (size_t) N * K * code_bytes(M)
                                                 : sizeof(double) * ((size_t) N / rows_per_block(M) + 1);
  return pad16(sizeof(BalanceHead)) + pad16(sizeof(float) * (size_t) M) + pad16(more);
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
  const BalanceSpace w = balance_space(workspace, M);
  if (cudaMemsetAsync(counts, 0, sizeof(int64_t) * ((size_t) M + 4), st) != cudaSuccess) return FSGS_ERR_LAUNCH;
  const int grid = balance_blocks((N * K + 3) / 4, kCountThreads, 2 * 148);
  const size_t smem = M <= kBalSharedPoints ? sizeof(int) * ((size_t) M + 1) : 0;
  unsigned long long *c = (unsigned long long *) counts;
  const int wide = ((uintptr_t) idx & 15) == 0;
  void *codes = form == FSGS_BALANCE_PAIRS ? w.codes : nullptr;
  if (code_bytes(M) == 2) balance_count_kernel<uint16_t><<<grid, kCountThreads, smem, st>>>(N, K, M, idx, mask, wide, c, w.head, w.share, (uint16_t *) codes);
  else balance_count_kernel<uint32_t><<<grid, kCountThreads, smem, st>>>(N, K, M, idx, mask, wide, c, w.head, w.share, (uint32_t *) codes);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_pairs(int64_t N, int K, int M, const float *weights, void *workspace, size_t workspace_bytes,
    float scale, const float *upstream, float *loss, float *g_weights, int accumulate, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && K > 0 && M > 0 && (weights || !loss || N == 0));
  if (!balance_sizes(N, K)) return FSGS_ERR_LIMIT;
  if (!balance_workspace(N, K, M, FSGS_BALANCE_PAIRS, workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_weights || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  const BalanceSpace w = balance_space(workspace, M);
  const int wide = (((uintptr_t) weights | (uintptr_t) g_weights) & 15) == 0;
  const PairsArgs a = {N * K, M, wide, weights, scale, upstream, loss, g_weights, accumulate, w.head, w.share};
  const int grid = balance_blocks((N * K + 7) / 8, kPairThreads, 3 * 148);
  const size_t smem = M <= kBalSharedPoints ? sizeof(float) * (size_t) M : 0;
  if (code_bytes(M) == 2) balance_pairs_kernel<uint16_t><<<grid, kPairThreads, smem, st>>>(a, (const uint16_t *) w.codes);
  else balance_pairs_kernel<uint32_t><<<grid, kPairThreads, smem, st>>>(a, (const uint32_t *) w.codes);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_table(int64_t N, int M, int type, const void *table, int64_t row_stride, const uint8_t *mask,
    void *workspace, size_t workspace_bytes, float scale, const float *upstream, float *loss, void *g_table,
    int64_t g_row_stride, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && M > 0 && (table || N == 0) && row_stride >= M && (!g_table || g_row_stride >= M));
  FSGS_REQUIRE(type == FSGS_F32 || type == FSGS_BF16 || type == FSGS_F16);
  if (!balance_sizes(N, M)) return FSGS_ERR_LIMIT;
  if (!balance_workspace(N, 1, M, FSGS_BALANCE_TABLE, workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_table || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  if (N == 0) return cudaMemsetAsync(loss, 0, sizeof(float), st) == cudaSuccess ? FSGS_OK : FSGS_ERR_LAUNCH;
  const BalanceSpace w = balance_space(workspace, M);
  const int64_t blocks = (N + rows_per_block(M) - 1) / rows_per_block(M);
  if (blocks > INT32_MAX) return FSGS_ERR_LIMIT;
  const TableArgs a = {N, row_stride, g_row_stride, M, table, mask, scale, upstream, g_table, w.share, loss ? w.sums : nullptr, w.head};
  // four columns per access where every row of both tables starts on a boundary of four elements
  const size_t four = type == FSGS_F32 ? 16 : 8;
  const bool wide = row_stride % 4 == 0 && (uintptr_t) table % four == 0 && (!g_table || (g_row_stride % 4 == 0 && (uintptr_t) g_table % four == 0));
  int rc;
  if (type == FSGS_F32) rc = wide ? table_pick<float, 4>(a, st) : table_pick<float, 1>(a, st);
  else if (type == FSGS_BF16) rc = wide ? table_pick<__nv_bfloat16, 4>(a, st) : table_pick<__nv_bfloat16, 1>(a, st);
  else rc = wide ? table_pick<__half, 4>(a, st) : table_pick<__half, 1>(a, st);
  if (rc != FSGS_OK || !loss) return rc;
  balance_close_kernel<<<1, 1024, 0, st>>>((int) blocks, w.sums, scale, upstream, loss);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}
