// Log probabilities of given tokens with the entropy of their rows and the best alternatives,
// their gradient, and the loss against a teacher's top logits with its gradient.
#include <algorithm>

#include "vocab_row.h"

namespace icap {
namespace {

constexpr int NT = 256;

struct ScoreArgs {
  const void* logits;
  RowView view;
  const int32_t* tokens;
  int N, V, pad, k;
  float *log_probs, *entropy, *stats;
  int32_t* top_ids;
  float* top_log_probs;
};

// One workgroup per row, one pass for the statistics and one more per alternative.
template <int DTYPE>
__global__ __launch_bounds__(NT) void token_log_probs_kernel(ScoreArgs p) {
  typedef Elem<DTYPE> E;
  __shared__ RowStats s_part[NT / 64];
  __shared__ unsigned long long s_key[NT / 64];
  const int row = blockIdx.y * gridDim.x + blockIdx.x, tid = threadIdx.x;
  if (row >= p.N) return;
  const int token = p.tokens[row];
  if (token == p.pad) {
    if (tid == 0) {
      p.log_probs[row] = 0.f;
      p.entropy[row] = 0.f;
      p.stats[2 * (size_t)row] = p.stats[2 * (size_t)row + 1] = 0.f;
    }
    for (int i = tid; i < p.k; i += NT) {
      p.top_ids[(size_t)row * p.k + i] = -1;
      p.top_log_probs[(size_t)row * p.k + i] = 0.f;
    }
    return;
  }
  const typename E::type* x = (const typename E::type*)p.logits + p.view.at(row);
  RowStats a = row_stats_empty();
  for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) {
    float v[E::kVec];
    load_vec<DTYPE>(x, c, p.V, -INFINITY, v);
    row_stats_add(a, v, kLog2e);
  }
  a = row_stats_block<NT / 64>(a, kLog2e, s_part);
  const bool none = a.s == 0.f;                 // every logit is -inf
  const float m = none ? -INFINITY : a.m;
  const float log_s = none ? 0.f : logf(a.s);
  if (tid == 0) {
    float lp;
    if (token < 0 || token >= p.V) lp = NAN;
    else if (none) lp = -INFINITY;
    else lp = (E::up(x[token]) - m) - log_s;
    p.log_probs[row] = lp;
    p.entropy[row] = none ? 0.f : log_s - a.w / a.s;
    p.stats[2 * (size_t)row] = m;
    p.stats[2 * (size_t)row + 1] = log_s;
  }
  unsigned long long below = ~0ull;
  for (int i = 0; i < p.k; ++i) {
    unsigned long long best = 0;
    for (int c = tid; c < p.V; c += NT) {
      const unsigned long long key = rank_key(E::up(x[c]), c);
      if (key < below && key > best) best = key;
    }
    for (int d = 32; d > 0; d >>= 1) best = max(best, (unsigned long long)__shfl_xor(best, d, 64));
    __syncthreads();
    if ((tid & 63) == 0) s_key[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) best = max(best, s_key[w]);
    below = best;
    if (tid == 0) {
      const int col = rank_col(best);
      p.top_ids[(size_t)row * p.k + i] = col;
      p.top_log_probs[(size_t)row * p.k + i] = none ? -INFINITY : (E::up(x[col]) - m) - log_s;
    }
  }
}

struct ScoreGradArgs {
  const void* logits;
  RowView view;
  const int32_t* tokens;
  int N, V, pad;
  const float *stats, *entropy, *g_lp, *g_h;
  void* out;
  RowView out_view;
};

// d log p_t / d x_j = [j = t] - p_j,   d H / d x_j = -p_j (log p_j + H)
template <int DTYPE>
__global__ __launch_bounds__(NT) void token_log_probs_grad_kernel(ScoreGradArgs p) {
  typedef Elem<DTYPE> E;
  const int row = blockIdx.y * gridDim.x + blockIdx.x, tid = threadIdx.x;
  if (row >= p.N) return;
  const int token = p.tokens[row];
  const typename E::type* x = (const typename E::type*)p.logits + p.view.at(row);
  typename E::type* g = (typename E::type*)p.out + p.out_view.at(row);
  float g_lp = p.g_lp ? p.g_lp[row] : 0.f;
  const float g_h = p.g_h ? p.g_h[row] : 0.f;
  const float m = p.stats[2 * (size_t)row], log_s = p.stats[2 * (size_t)row + 1], h = p.entropy[row];
  if (token == p.pad || m == -INFINITY || (g_lp == 0.f && g_h == 0.f)) {
    const float zero[E::kVec] = {};
    for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) store_vec<DTYPE>(g, c, p.V, zero);
    return;
  }
  if ((token < 0 || token >= p.V) && g_lp != 0.f) g_lp = NAN;
  const float inv_s = __builtin_amdgcn_exp2f(-log_s * kLog2e);
  for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) {
    float v[E::kVec];
    load_vec<DTYPE>(x, c, p.V, -INFINITY, v);
#pragma unroll
    for (int i = 0; i < E::kVec; ++i) {
      const float d = v[i] - m;
      const float e = __builtin_amdgcn_exp2f(d * kLog2e) * inv_s;
      const float u = fmaxf(d, kFarBelow) - log_s + h;
      v[i] = -e * (g_lp + g_h * u) + (c + i == token ? g_lp : 0.f);
    }
    store_vec<DTYPE>(g, c, p.V, v);
  }
}

constexpr int kMaxTeacher = ICAP_MAX_TEACHER_LOGITS;

struct DistillArgs {
  const void* logits;
  RowView view;
  const void* t_logits;
  int t_dtype;
  const int32_t* t_ids;
  int N, V, K;
  float tau;
  const float* g_loss;
  float* loss;
  void* out;
  RowView out_view;
};

__device__ __forceinline__ float load_typed(const void* p, int dtype, size_t i) {
  if (dtype == ICAP_DTYPE_F32) return ((const float*)p)[i];
  if (dtype == ICAP_DTYPE_BF16) return (float)((const __bf16*)p)[i];
  return (float)((const _Float16*)p)[i];
}

// loss = tau^2 sum_k q_k (log q_k - log p[id_k]),  q = soft-max of the teacher's K logits at tau,
// p = soft-max of the row at tau;   d loss / d x_j = tau (p_j - sum over k with id_k = j of q_k)
template <int DTYPE>
__global__ __launch_bounds__(NT) void distill_loss_kernel(DistillArgs p) {
  typedef Elem<DTYPE> E;
  __shared__ RowStats s_part[NT / 64];
  __shared__ int s_id[kMaxTeacher];
  __shared__ float s_q[kMaxTeacher], s_log_q[kMaxTeacher], s_x[kMaxTeacher];
  __shared__ int s_alive, s_bad;
  const int row = blockIdx.y * gridDim.x + blockIdx.x, tid = threadIdx.x;
  if (row >= p.N) return;
  const typename E::type* x = (const typename E::type*)p.logits + p.view.at(row);
  typename E::type* g = p.out ? (typename E::type*)p.out + p.out_view.at(row) : nullptr;
  const float inv_tau = 1.f / p.tau, rate = kLog2e * inv_tau;
  if (tid < 64) {
    float top = -INFINITY;
    bool alive = false, bad = false;
    for (int k = tid; k < p.K; k += 64) {
      const int id = p.t_ids[(size_t)row * p.K + k];
      const bool in = id >= 0 && id < p.V;
      const float t = id == -1 ? -INFINITY : load_typed(p.t_logits, p.t_dtype, (size_t)row * p.K + k);
      bad |= id != -1 && !in;
      alive |= !(t == -INFINITY);
      s_id[k] = in ? id : -1;
      s_log_q[k] = t;
      s_x[k] = in ? E::up(x[id]) : 0.f;
      top = fmaxf(top, t);
    }
    alive = __any(alive);
    bad = __any(bad);
    top = wave_max(top);
    float sum = 0.f;
    for (int k = tid; k < p.K; k += 64) {
      const float e = s_log_q[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((s_log_q[k] - top) * rate);
      s_q[k] = e;
      sum += e;
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum);
    for (int k = tid; k < p.K; k += 64) {
      s_log_q[k] = (s_log_q[k] - top) * inv_tau - log_sum;
      s_q[k] /= sum;
    }
    if (tid == 0) { s_alive = alive; s_bad = bad; }
  }
  __syncthreads();
  const float coef = p.g_loss ? p.g_loss[row] * p.tau : 0.f;
  if (!s_alive && !s_bad) {
    if (tid == 0) p.loss[row] = 0.f;
    if (g) {
      const float zero[E::kVec] = {};
      for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) store_vec<DTYPE>(g, c, p.V, zero);
    }
    return;
  }
  RowStats a = row_stats_empty();
  for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) {
    float v[E::kVec];
    load_vec<DTYPE>(x, c, p.V, -INFINITY, v);
    row_stats_add(a, v, rate);
  }
  a = row_stats_block<NT / 64>(a, rate, s_part);
  const bool none = a.s == 0.f;
  const float log_s = logf(a.s), inv_s = 1.f / a.s;
  if (tid < 64) {
    float sum = 0.f;
    for (int k = tid; k < p.K; k += 64) {
      const float q = s_q[k];
      const float lp = none ? -INFINITY : (s_x[k] - a.m) * inv_tau - log_s;
      if (s_id[k] >= 0 && !(q == 0.f)) sum += q * (s_log_q[k] - lp);
    }
    sum = wave_sum(sum) * p.tau * p.tau;
    if (tid == 0) p.loss[row] = s_bad ? NAN : sum;
  }
  if (!g) return;
  const bool zero_row = coef == 0.f || (none && !s_bad);
  const float c0 = zero_row ? 0.f : s_bad ? NAN : coef;
  for (int c = tid * E::kVec; c < p.V; c += NT * E::kVec) {
    float v[E::kVec];
    load_vec<DTYPE>(x, c, p.V, -INFINITY, v);
#pragma unroll
    for (int i = 0; i < E::kVec; ++i)
      v[i] = zero_row ? 0.f : c0 * (__builtin_amdgcn_exp2f((v[i] - a.m) * rate) * inv_s);
    store_vec<DTYPE>(g, c, p.V, v);
  }
  if (zero_row || s_bad) return;
  __syncthreads();
  // the teacher's columns again, the first of several entries with the same id for all of them
  for (int k = tid; k < p.K; k += NT) {
    const int id = s_id[k];
    bool first = id >= 0;
    float q = 0.f;
    for (int j = 0; j < p.K; ++j)
      if (s_id[j] == id) {
        if (j < k) first = false;
        q += s_q[j];
      }
    if (first)
      g[id] = E::down(c0 * (__builtin_amdgcn_exp2f((s_x[k] - a.m) * rate) * inv_s - q));
  }
}

dim3 row_grid(int N) {
  const int x = N < 65536 ? N : 65536;
  return dim3((unsigned)x, (unsigned)ceil_div(N, x));
}

int check_rows(const char* what, int dtype, int N, int V, const RowView& v) {
  ICAP_REQUIRE(dtype == ICAP_DTYPE_F32 || dtype == ICAP_DTYPE_BF16 || dtype == ICAP_DTYPE_F16,
               "%s: unknown dtype %d", what, dtype);
  ICAP_REQUIRE(N > 0 && V > 0, "%s: bad shape", what);
  ICAP_REQUIRE(V <= 0x7fff0000, "%s: V too large", what);
  ICAP_REQUIRE(v.inner > 0 && v.ld >= 0 && v.ld_outer >= 0, "%s: bad strides", what);
  return ICAP_OK;
}

// Rows that are written may not share elements, whichever of the two strides is the larger.
int check_out(const char* what, int N, int V, const RowView& v) {
  const long long inner = std::min(N, v.inner), outer = ceil_div(N, v.inner);
  const long long near = v.ld <= v.ld_outer || outer == 1 ? v.ld : v.ld_outer;
  const long long far = near == v.ld ? v.ld_outer : v.ld;
  const long long run = near == v.ld ? inner : outer;
  ICAP_REQUIRE((run == 1 || near >= V) && (outer == 1 || inner == 1 || far >= (run - 1) * near + V) &&
                   (inner > 1 || outer == 1 || v.ld_outer >= V),
               "%s: rows of the gradient overlap", what);
  return ICAP_OK;
}

#define ICAP_BY_DTYPE(dtype, call)                                   \
  do {                                                               \
    if ((dtype) == ICAP_DTYPE_F32) { call(ICAP_DTYPE_F32); }         \
    else if ((dtype) == ICAP_DTYPE_BF16) { call(ICAP_DTYPE_BF16); }  \
    else { call(ICAP_DTYPE_F16); }                                   \
  } while (0)

}  // namespace
}  // namespace icap

using namespace icap;

extern "C" {

int icap_token_log_probs(const void* logits, int dtype, int N, int V, int rows_inner, long long ld,
                         long long ld_outer, const int32_t* tokens, int pad_token, int top_k,
                         float* log_probs, float* entropy, float* stats, int32_t* top_ids,
                         float* top_log_probs, icap_stream_t stream) {
  ICAP_REQUIRE(logits && tokens && log_probs && entropy && stats, "token_log_probs: null pointer");
  const RowView view{rows_inner, ld, ld_outer};
  if (int rc = check_rows("token_log_probs", dtype, N, V, view)) return rc;
  ICAP_REQUIRE(top_k >= 0 && top_k <= V, "token_log_probs: top_k outside 0 .. V");
  ICAP_REQUIRE(top_k == 0 || (top_ids && top_log_probs), "token_log_probs: null output of the alternatives");
  if (top_k > ICAP_MAX_ALTERNATIVES)
    return fail(ICAP_ERR_UNSUPPORTED, "token_log_probs: top_k %d is over %d", top_k, ICAP_MAX_ALTERNATIVES);
  ScoreArgs a{logits, view, tokens, N, V, pad_token, top_k, log_probs, entropy, stats, top_ids, top_log_probs};
#define LAUNCH(D) hipLaunchKernelGGL(token_log_probs_kernel<D>, row_grid(N), dim3(NT), 0, (hipStream_t)stream, a)
  ICAP_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("token_log_probs_kernel");
  return ICAP_OK;
}

int icap_token_log_probs_grad(const void* logits, int dtype, int N, int V, int rows_inner, long long ld,
                              long long ld_outer, const int32_t* tokens, int pad_token,
                              const float* stats, const float* entropy, const float* grad_log_probs,
                              const float* grad_entropy, void* dlogits, long long out_ld,
                              long long out_ld_outer, icap_stream_t stream) {
  ICAP_REQUIRE(logits && tokens && stats && entropy && dlogits, "token_log_probs_grad: null pointer");
  const RowView view{rows_inner, ld, ld_outer}, out{rows_inner, out_ld, out_ld_outer};
  if (int rc = check_rows("token_log_probs_grad", dtype, N, V, view)) return rc;
  if (int rc = check_rows("token_log_probs_grad", dtype, N, V, out)) return rc;
  if (int rc = check_out("token_log_probs_grad", N, V, out)) return rc;
  ScoreGradArgs a{logits, view, tokens, N, V, pad_token, stats, entropy, grad_log_probs, grad_entropy, dlogits, out};
#define LAUNCH(D) hipLaunchKernelGGL(token_log_probs_grad_kernel<D>, row_grid(N), dim3(NT), 0, (hipStream_t)stream, a)
  ICAP_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("token_log_probs_grad_kernel");
  return ICAP_OK;
}

int icap_distill_loss(const void* logits, int dtype, int N, int V, int rows_inner, long long ld,
                      long long ld_outer, const void* teacher_logits, int teacher_dtype,
                      const int32_t* teacher_ids, int K, float temperature, const float* grad_loss,
                      float* loss, void* dlogits, long long out_ld, long long out_ld_outer,
                      icap_stream_t stream) {
  ICAP_REQUIRE(logits && teacher_logits && teacher_ids && loss, "distill_loss: null pointer");
  const RowView view{rows_inner, ld, ld_outer}, out{rows_inner, out_ld, out_ld_outer};
  if (int rc = check_rows("distill_loss", dtype, N, V, view)) return rc;
  ICAP_REQUIRE(teacher_dtype == ICAP_DTYPE_F32 || teacher_dtype == ICAP_DTYPE_BF16 || teacher_dtype == ICAP_DTYPE_F16,
               "distill_loss: unknown teacher dtype %d", teacher_dtype);
  ICAP_REQUIRE(K > 0, "distill_loss: no teacher entries");
  if (K > kMaxTeacher)
    return fail(ICAP_ERR_UNSUPPORTED, "distill_loss: K %d is over %d", K, kMaxTeacher);
  ICAP_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, "distill_loss: temperature outside 0.001 .. 1000");
  ICAP_REQUIRE((grad_loss != nullptr) == (dlogits != nullptr), "distill_loss: grad_loss and dlogits go together");
  if (dlogits) {
    if (int rc = check_rows("distill_loss", dtype, N, V, out)) return rc;
    if (int rc = check_out("distill_loss", N, V, out)) return rc;
  }
  DistillArgs a{logits, view, teacher_logits, teacher_dtype, teacher_ids, N, V, K, temperature,
                grad_loss, loss, dlogits, out};
#define LAUNCH(D) hipLaunchKernelGGL(distill_loss_kernel<D>, row_grid(N), dim3(NT), 0, (hipStream_t)stream, a)
  ICAP_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("distill_loss_kernel");
  return ICAP_OK;
}

}  // extern "C"
