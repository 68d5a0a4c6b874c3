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

constexpr int kBalThreads = 256;
constexpr int kBalSlots = 1184;           // 148 SMs x 8 blocks
constexpr int kBalSharedPoints = 8192;    // superpoints whose table is kept in shared memory (32 KB)
constexpr int kCountThreads = 1024;

struct BalanceHead {  // start of the workspace
  int ticket;
  int pad[3];
  double slots[kBalSlots];
  long long live[kBalSlots];
};

// ---- counts -----------------------------------------------------------------------------------------------

// One pass over the indices: a histogram per block in shared memory, added to the 64-bit counts at the end; the
// superpoint of every pair is kept as a 16- or 32-bit code (all ones: does not count) for the pass that needs the
// complete counts, which then reads 2 bytes per pair instead of 8 and no mask.
template <typename Code>
__global__ void __launch_bounds__(kCountThreads) balance_count_kernel(long long N, int K, int M, const int64_t *__restrict__ idx,
    const uint8_t *__restrict__ mask, unsigned long long *__restrict__ counts, Code *__restrict__ codes,
    BalanceHead *__restrict__ head) {
  extern __shared__ int s_hist[];
  __shared__ int s_red[2][kCountThreads / 32];
  const bool in_shared = M <= kBalSharedPoints;
  if (blockIdx.x == 0 && threadIdx.x == 0) head->ticket = 0;  // for the kernel that closes the sum of the loss
  if (in_shared) {
    for (int m = threadIdx.x; m < M; m += kCountThreads) s_hist[m] = 0;
    __syncthreads();
  }
  const long long pairs = N * K, stride = (long long) gridDim.x * kCountThreads;
  int named = 0, rows = 0;
  for (long long e = (long long) blockIdx.x * kCountThreads + threadIdx.x; e < pairs; e += stride) {
    bool on = true;
    if (mask) {
      const long long row = pairs < (1ll << 32) ? (long long) ((unsigned) e / (unsigned) K) : e / K;
      on = mask[row] != 0;
    }
    const int64_t m = idx[e];
    on = on && m >= 0 && m < M;
    if (on) {
      ++named;
      if (in_shared) atomicAdd(s_hist + m, 1);
      else atomicAdd(counts + m, 1ull);
    }
    if (codes) codes[e] = on ? (Code) m : (Code) ~(Code) 0;
  }
  for (long long i = (long long) blockIdx.x * kCountThreads + threadIdx.x; i < N; i += stride) rows += !mask || mask[i] != 0;
  for (int o = 16; o > 0; o >>= 1) {
    named += __shfl_xor_sync(0xffffffffu, named, o);
    rows += __shfl_xor_sync(0xffffffffu, rows, o);
  }
  if ((threadIdx.x & 31) == 0) s_red[0][threadIdx.x >> 5] = named, s_red[1][threadIdx.x >> 5] = rows;
  __syncthreads();
  if (threadIdx.x < 2) {
    unsigned long long t = 0;
    for (int w = 0; w < kCountThreads / 32; ++w) t += s_red[threadIdx.x][w];
    if (t) atomicAdd(counts + M + threadIdx.x, t);
  }
  if (in_shared)
    for (int m = threadIdx.x; m < M; m += kCountThreads)
      if (s_hist[m]) atomicAdd(counts + m, (unsigned long long) s_hist[m]);
}

// ---- closing the sum of the loss ----------------------------------------------------------------------------

// Adds the blocks' sums in a fixed order in the block that arrives last; thread 0 of that block gets true.
__device__ __forceinline__ bool close_sum(BalanceHead *h, double sum, long long live, double &total, long long &rows) {
  __shared__ double s_sum[32];
  __shared__ long long s_live[32];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (lane == 0) s_sum[warp] = sum, s_live[warp] = live;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < warps; ++w) sum += s_sum[w], live += s_live[w];
    h->slots[blockIdx.x] = sum, h->live[blockIdx.x] = live;
    __threadfence();
    s_last = atomicAdd(&h->ticket, 1) == (int) gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return false;
  __threadfence();
  sum = 0.0, live = 0;
  for (int i = threadIdx.x; i < (int) gridDim.x; i += blockDim.x) sum += __ldcg(h->slots + i), live += __ldcg(h->live + i);
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (lane == 0) s_sum[warp] = sum, s_live[warp] = live;
  __syncthreads();
  if (threadIdx.x != 0) return false;
  for (int w = 1; w < warps; ++w) sum += s_sum[w], live += s_live[w];
  total = sum, rows = live;
  h->ticket = 0;
  return true;
}

// ---- pairs form ---------------------------------------------------------------------------------------------

struct PairsArgs {
  long long pairs;
  int M;
  const float *w;                    // null: no loss
  const long long *counts;            // [M + 2]: the counts, T, n
  float scale;
  const float *upstream;             // null: 1
  float *loss, *g;                   // either may be null
  int accumulate;
  BalanceHead *head;
};

__device__ __forceinline__ float pair_share(long long c, int M, double denom) {
  return denom > 0.0 ? (float) ((double) M * (double) c / denom) : 0.0f;
}

template <typename Code>
__global__ void __launch_bounds__(kBalThreads) balance_pairs_kernel(PairsArgs a, const Code *__restrict__ codes) {
  extern __shared__ float s_share[];
  const bool in_shared = a.M <= kBalSharedPoints;
  const double denom = (double) a.counts[a.M] * (double) a.counts[a.M + 1];
  if (in_shared) {
    for (int m = threadIdx.x; m < a.M; m += kBalThreads) s_share[m] = pair_share(a.counts[m], a.M, denom);
    __syncthreads();
  }
  const float up = a.scale * (a.upstream ? *a.upstream : 1.0f);
  double sum = 0.0;
  const long long stride = (long long) gridDim.x * kBalThreads;
  for (long long e = (long long) blockIdx.x * kBalThreads + threadIdx.x; e < a.pairs; e += stride) {
    const Code c = codes[e];
    const bool on = c != (Code) ~(Code) 0;
    const float share = !on ? 0.0f : in_shared ? s_share[c] : pair_share(a.counts[c], a.M, denom);
    // a weight that does not count is not read into the sum: it may be anything, a NaN too
    if (a.loss && on) sum += (double) (a.w[e] * share);
    if (a.g) a.g[e] = a.accumulate ? a.g[e] + up * share : up * share;
  }
  if (!a.loss) return;
  double total;
  long long rows;
  if (close_sum(a.head, sum, 0, total, rows)) *a.loss = (float) (total * (double) up);
}

// ---- table form ---------------------------------------------------------------------------------------------

struct TableArgs {
  long long N, stride, g_stride;     // row strides in elements
  int M;
  const void *table;
  const uint8_t *mask;
  const long long *counts;            // [M + 2]: the counts, T, n
  float scale;
  const float *upstream;
  float *loss;
  void *g;
  BalanceHead *head;
};

__device__ __forceinline__ float get(const float *p) { return *p; }
__device__ __forceinline__ float get(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ float get(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }

__device__ __forceinline__ float centred_share(long long c, int M, long long total, double denom) {
  return denom > 0.0 ? (float) (((double) M * (double) c - (double) total) / denom) : 0.0f;
}

// max / sum over the G threads that share a row (a warp, or the block)
template <int G>
__device__ __forceinline__ float row_max(float v, float *scratch) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (G > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
    for (int w = 1; w < G / 32; ++w) v = fmaxf(v, scratch[w]);
  }
  return v;
}
template <int G>
__device__ __forceinline__ float2 row_sum(float2 v, float2 *scratch) {
  for (int o = 16; o > 0; o >>= 1) {
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

// G threads per row, PER columns per thread (PER 0: any number of columns, the row is read again for each of the three
// passes); the shares of a thread's columns stay in registers over all its rows.
template <typename T, int G, int PER>
__global__ void __launch_bounds__(kBalThreads) balance_table_kernel(TableArgs a) {
  __shared__ float s_max[kBalThreads / 32];
  __shared__ float2 s_sum[kBalThreads / 32];
  const int t = threadIdx.x % G;
  const long long total = a.counts[a.M], n = a.counts[a.M + 1];
  const double denom = (double) total * (double) n;
  const float up = a.scale * (a.upstream ? *a.upstream : 1.0f);
  float share[PER > 0 ? PER : 1];
#pragma unroll
  for (int u = 0; u < PER; ++u) share[u] = t + u * G < a.M ? centred_share(a.counts[t + u * G], a.M, total, denom) : 0.0f;
  double sum = 0.0;
  long long live = 0;
  const long long step = (long long) gridDim.x * (kBalThreads / G);
  for (long long i = (long long) blockIdx.x * (kBalThreads / G) + threadIdx.x / G; i < a.N; i += step) {
    T *g = a.g ? (T *) a.g + i * a.g_stride : nullptr;
    if (a.mask && !a.mask[i]) {
      if (g)
        for (int m = t; m < a.M; m += G) put(g + m, 0.0f);
      continue;
    }
    const T *z = (const T *) a.table + i * a.stride;
    float x[PER > 0 ? PER : 1], top = -INFINITY;
    if (PER > 0) {
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        x[u] = t + u * G < a.M ? get(z + t + u * G) : -INFINITY;
        // fmaxf passes over a NaN; the row's sum below does not
        top = fmaxf(top, x[u]);
      }
    } else {
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
        s.x += x[u], s.y = fmaf(x[u], share[u], s.y);
      }
    } else {
      for (int m = t; m < a.M; m += G) {
        const float e = expf(get(z + m) - base);
        s.x += e, s.y = fmaf(e, centred_share(a.counts[m], a.M, total, denom), s.y);
      }
    }
    s = row_sum<G>(s, s_sum);
    const float inv = s.x == 0.0f ? 0.0f : 1.0f / s.x, inner = s.y * inv;
    if (t == 0 && s.x != 0.0f) sum += (double) inner, ++live;
    if (!g) continue;
    const float k = up * inv;
    if (PER > 0) {
#pragma unroll
      for (int u = 0; u < PER; ++u)
        if (t + u * G < a.M) put(g + t + u * G, k * x[u] * (share[u] - inner));
    } else {
      for (int m = t; m < a.M; m += G)
        put(g + m, k * expf(get(z + m) - base) * (centred_share(a.counts[m], a.M, total, denom) - inner));
    }
  }
  if (!a.loss) return;
  double all;
  long long rows;
  if (close_sum(a.head, sum, live, all, rows)) *a.loss = denom > 0.0 ? (float) (((double) rows / (double) n + all) * (double) up) : 0.0f;
}

template <typename T, int G, int PER>
static int table_launch(const TableArgs &a, cudaStream_t st) {
  const int64_t blocks = (a.N + kBalThreads / G - 1) / (kBalThreads / G);
  balance_table_kernel<T, G, PER><<<(int) (blocks < kBalSlots ? blocks : kBalSlots), kBalThreads, 0, st>>>(a);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

template <typename T>
static int table_pick(const TableArgs &a, cudaStream_t st) {
  if (a.M <= 128) return table_launch<T, 32, 4>(a, st);
  if (a.M <= 512) return table_launch<T, 32, 16>(a, st);
  if (a.M <= 2048) return table_launch<T, 256, 8>(a, st);
  if (a.M <= 8192) return table_launch<T, 256, 32>(a, st);
  return table_launch<T, 256, 0>(a, st);
}

static size_t code_bytes(int M) { return M < 65536 ? 2 : 4; }

}  // namespace fsgs

using namespace fsgs;

extern "C" size_t fsgs_balance_workspace_bytes(void) { return sizeof(BalanceHead); }

extern "C" size_t fsgs_balance_codes_bytes(int64_t N, int K, int M) {
  return N > 0 && K > 0 && M > 0 ? (size_t) N * K * code_bytes(M) : 0;
}

static bool balance_workspace(void *workspace, size_t bytes) {
  return workspace && ((uintptr_t) workspace & 15) == 0 && bytes >= sizeof(BalanceHead);
}

extern "C" int fsgs_balance_count(int64_t N, int K, int M, const int64_t *idx, const uint8_t *mask, int64_t *counts,
    void *codes, void *workspace, size_t workspace_bytes, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && K > 0 && M > 0 && counts && (idx || N == 0));
  if (N > (1ll << 36) / K) return FSGS_ERR_LIMIT;
  if (!balance_workspace(workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  cudaStream_t st = (cudaStream_t) stream;
  if (cudaMemsetAsync(counts, 0, sizeof(int64_t) * ((size_t) M + 2), st) != cudaSuccess) return FSGS_ERR_LAUNCH;
  const int64_t blocks = (N * K + kCountThreads - 1) / kCountThreads;
  const int grid = (int) (blocks < 2 * 148 ? (blocks > 0 ? blocks : 1) : 2 * 148);
  const size_t smem = M <= kBalSharedPoints ? sizeof(int) * (size_t) M : 0;
  unsigned long long *c = (unsigned long long *) counts;
  BalanceHead *h = (BalanceHead *) workspace;
  if (code_bytes(M) == 2) balance_count_kernel<uint16_t><<<grid, kCountThreads, smem, st>>>(N, K, M, idx, mask, c, (uint16_t *) codes, h);
  else balance_count_kernel<uint32_t><<<grid, kCountThreads, smem, st>>>(N, K, M, idx, mask, c, (uint32_t *) codes, h);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_pairs(int64_t N, int K, int M, const float *weights, const void *codes, const int64_t *counts,
    float scale, const float *upstream, float *loss, float *g_weights, int accumulate, void *workspace,
    size_t workspace_bytes, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && K > 0 && M > 0 && counts && (codes || N == 0) && (weights || !loss || N == 0));
  if (N > (1ll << 36) / K) return FSGS_ERR_LIMIT;
  if (loss && !balance_workspace(workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_weights || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  PairsArgs a = {N * K, M, weights, (const long long *) counts, scale, upstream, loss, g_weights, accumulate,
                 (BalanceHead *) workspace};
  const int64_t blocks = (N * K + kBalThreads - 1) / kBalThreads;
  const int grid = (int) (blocks < kBalSlots ? (blocks > 0 ? blocks : 1) : kBalSlots);
  const size_t smem = M <= kBalSharedPoints ? sizeof(float) * (size_t) M : 0;
  if (code_bytes(M) == 2) balance_pairs_kernel<uint16_t><<<grid, kBalThreads, smem, st>>>(a, (const uint16_t *) codes);
  else balance_pairs_kernel<uint32_t><<<grid, kBalThreads, smem, st>>>(a, (const uint32_t *) codes);
  FSGS_LAUNCH_CHECK();
  return FSGS_OK;
}

extern "C" int fsgs_balance_table(int64_t N, int M, int type, const void *table, int64_t row_stride, const uint8_t *mask,
    const int64_t *counts, float scale, const float *upstream, float *loss, void *g_table, int64_t g_row_stride,
    void *workspace, size_t workspace_bytes, fsgs_stream_t stream) {
  FSGS_REQUIRE(N >= 0 && M > 0 && counts && (table || N == 0) && row_stride >= M && (!g_table || g_row_stride >= M));
  FSGS_REQUIRE(type == FSGS_F32 || type == FSGS_BF16 || type == FSGS_F16);
  if (N > (1ll << 40) / M) return FSGS_ERR_LIMIT;
  if (loss && !balance_workspace(workspace, workspace_bytes)) return FSGS_ERR_WORKSPACE;
  if (!loss && (!g_table || N == 0)) return FSGS_OK;
  cudaStream_t st = (cudaStream_t) stream;
  if (N == 0) return cudaMemsetAsync(loss, 0, sizeof(float), st) == cudaSuccess ? FSGS_OK : FSGS_ERR_LAUNCH;
  TableArgs a = {N, row_stride, g_row_stride, M, table, mask, (const long long *) counts, scale, upstream, loss, g_table,
                 (BalanceHead *) workspace};
  if (type == FSGS_F32) return table_pick<float>(a, st);
  if (type == FSGS_BF16) return table_pick<__nv_bfloat16>(a, st);
  return table_pick<__half>(a, st);
}
