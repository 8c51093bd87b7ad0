// Scaled embedding lookup and its gradient by sorted tokens.
#include <algorithm>

#include "vocab_row.h"

namespace icap {
namespace {

template <int DTYPE>
__global__ __launch_bounds__(256) void embedding_scaled_kernel(const void* table, const int32_t* ids,
                                                               void* out, int N, int V, int D, float scale,
                                                               int pad) {
  typedef Elem<DTYPE> E;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (n >= N) return;
  const int id = ids[n];
  const bool ok = id >= 0 && id < V && id != pad;
  const typename E::type* src = (const typename E::type*)table + (ok ? (size_t)id * D : 0);
  typename E::type* dst = (typename E::type*)out + (size_t)n * D;
  for (int c = lane * E::kVec; c < D; c += 64 * E::kVec) {
    float v[E::kVec] = {};
    if (ok) load_vec<DTYPE>(src, c, D, 0.f, v);
#pragma unroll
    for (int i = 0; i < E::kVec; ++i) v[i] *= scale;
    store_vec<DTYPE>(dst, c, D, v);
  }
}

// ---- gradient: tokens sorted by id, then one sum per row of the table -----------------------

constexpr int kSortWaves = 16;
constexpr int kSortRows = 512;      // table rows of one sorting workgroup at most

// Workgroup b owns the ids [b * rows, (b + 1) * rows) and reads all N tokens twice: once to count
// (how many belong to earlier workgroups, and per wave and row how many to this one), once to
// write their positions, in ascending order within a row, behind those counts.  Every count is
// an integer and every place follows from the counts, so nothing depends on timing.
__global__ __launch_bounds__(kSortWaves * 64) void embed_sort_kernel(const int32_t* ids, int N, int V, int pad,
                                                                     int rows, int32_t* row_start,
                                                                     int32_t* sorted) {
  __shared__ int s_cnt[kSortWaves][kSortRows];
  __shared__ int s_wave[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = blockIdx.x * rows, hi = min(V, lo + rows), mine = hi - lo;
  for (int i = tid; i < kSortWaves * kSortRows; i += kSortWaves * 64) (&s_cnt[0][0])[i] = 0;
  __syncthreads();
  const int per = ((N + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int from = min(N, wave * per), to = min(N, from + per);
  int below = 0;
  for (int i = from + lane; i < to; i += 64) {
    const int id = ids[i];
    if (id < 0 || id >= V || id == pad) continue;
    below += id < lo;
    if (id >= lo && id < hi) atomicAdd(&s_cnt[wave][id - lo], 1);
  }
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d, 64);
  if (lane == 0) s_wave[wave] = below;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += s_wave[w];
  __syncthreads();
  int total = 0;
  if (tid < mine)
    for (int w = 0; w < kSortWaves; ++w) total += s_cnt[w][tid];
  int upto = total;       // inclusive scan over the rows
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) base += s_wave[w];
  if (tid < mine) {
    int at = base + upto - total;
    row_start[lo + tid] = at;
    if (lo + tid == V - 1) row_start[V] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = s_cnt[w][tid];
      s_cnt[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    const int id = i < to ? ids[i] : -1;
    unsigned long long left = __ballot(id >= lo && id < hi && id != pad);
    while (left) {        // the lanes of one id at a time
      const int leader = __ffsll(left) - 1;
      const int r = __shfl(id, leader, 64);
      const unsigned long long same = __ballot(id == r) & left;
      const int at = s_cnt[wave][r - lo];
      if ((same >> lane) & 1) sorted[at + __popcll(same & ((1ull << lane) - 1))] = i;
      if (lane == leader) s_cnt[wave][r - lo] = at + __popcll(same);
      left &= ~same;
    }
  }
}

// dtable[v] = scale * sum of the rows of `grad` whose token is v, in the tokens' order.
template <int DTYPE>
__global__ __launch_bounds__(256) void embed_sum_kernel(const void* grad, void* dtable, int V, int D,
                                                        float scale, const int32_t* row_start,
                                                        const int32_t* sorted) {
  typedef Elem<DTYPE> E;
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (v >= V) return;
  const int from = row_start[v], to = row_start[v + 1];
  for (int c = lane * E::kVec; c < D; c += 64 * E::kVec) {
    float acc[E::kVec] = {};
    for (int i = from; i < to; ++i) {
      float x[E::kVec];
      load_vec<DTYPE>((const typename E::type*)grad + (size_t)sorted[i] * D, c, D, 0.f, x);
#pragma unroll
      for (int j = 0; j < E::kVec; ++j) acc[j] += x[j];
    }
#pragma unroll
    for (int j = 0; j < E::kVec; ++j) acc[j] *= scale;
    store_vec<DTYPE>((typename E::type*)dtable + (size_t)v * D, c, D, acc);
  }
}

int check(const char* what, int dtype, int N, int V, int D) {
  ICAP_REQUIRE(dtype == ICAP_DTYPE_F32 || dtype == ICAP_DTYPE_BF16 || dtype == ICAP_DTYPE_F16,
               "%s: unknown dtype %d", what, dtype);
  ICAP_REQUIRE(N >= 0 && V > 0 && D > 0, "%s: bad shape", what);
  ICAP_REQUIRE(N <= 0x7fffff00 && V <= 0x7fff0000 && D <= 0x7fff0000, "%s: shape too large", what);
  return ICAP_OK;
}

}  // namespace
}  // namespace icap

using namespace icap;

extern "C" {

int icap_embedding_scaled(const void* table, int dtype, const int32_t* ids, void* out, int N, int V,
                          int D, float scale, int pad_token, icap_stream_t stream) {
  ICAP_REQUIRE(table && ids && out, "embedding_scaled: null pointer");
  if (int rc = check("embedding_scaled", dtype, N, V, D)) return rc;
  if (N == 0) return ICAP_OK;
  const dim3 grid(ceil_div(N, 4));
#define LAUNCH(T)                                                                                 \
  hipLaunchKernelGGL(embedding_scaled_kernel<T>, grid, dim3(256), 0, (hipStream_t)stream, table, ids, \
                     out, N, V, D, scale, pad_token)
  if (dtype == ICAP_DTYPE_F32) LAUNCH(ICAP_DTYPE_F32);
  else if (dtype == ICAP_DTYPE_BF16) LAUNCH(ICAP_DTYPE_BF16);
  else LAUNCH(ICAP_DTYPE_F16);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("embedding_scaled_kernel");
  return ICAP_OK;
}

size_t icap_embedding_grad_workspace_bytes(int N, int V, int D) {
  if (N < 0 || V <= 0 || D <= 0) return 0;
  return ((size_t)N + (size_t)V + 1) * sizeof(int32_t);
}

int icap_embedding_grad(const void* grad, int dtype, const int32_t* ids, void* dtable, int N, int V,
                        int D, float scale, int pad_token, void* workspace, size_t workspace_bytes,
                        icap_stream_t stream) {
  ICAP_REQUIRE(grad && ids && dtable && workspace, "embedding_grad: null pointer");
  if (int rc = check("embedding_grad", dtype, N, V, D)) return rc;
  ICAP_REQUIRE(aligned16(workspace) && workspace_bytes >= icap_embedding_grad_workspace_bytes(N, V, D),
               "embedding_grad: workspace too small or not aligned");
  int32_t* row_start = (int32_t*)workspace;
  int32_t* sorted = row_start + V + 1;
  const int rows = std::min(kSortRows, std::max(1, ceil_div(V, 256)));
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(embed_sort_kernel, dim3(ceil_div(V, rows)), dim3(kSortWaves * 64), 0, s, ids, N, V,
                     pad_token, rows, row_start, sorted);
  ICAP_LAUNCH_CHECK("embed_sort_kernel");
  const dim3 grid(ceil_div(V, 4));
#define LAUNCH(T)                                                                                  \
  hipLaunchKernelGGL(embed_sum_kernel<T>, grid, dim3(256), 0, s, grad, dtable, V, D, scale, row_start, \
                     sorted)
  if (dtype == ICAP_DTYPE_F32) LAUNCH(ICAP_DTYPE_F32);
  else if (dtype == ICAP_DTYPE_BF16) LAUNCH(ICAP_DTYPE_BF16);
  else LAUNCH(ICAP_DTYPE_F16);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("embed_sum_kernel");
  return ICAP_OK;
}

}  // extern "C"
