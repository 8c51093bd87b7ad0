// A row of logits over the vocabulary, read once: typed loads of 16 bytes and the running
// soft-max statistics (gfx950 only).  Shared by the operators that score tokens.
#pragma once

#include "icap_common.h"

namespace icap {

// Row r of a [N,V] view starts at (r / inner) * ld_outer + (r % inner) * ld elements: a matrix
// (inner >= N), or the first T - 1 positions of a [B,T,V] tensor (inner = T - 1).
struct RowView {
  int inner;
  long long ld, ld_outer;
  __host__ __device__ size_t at(int r) const {
    return r < inner ? (size_t)r * (size_t)ld
                     : (size_t)(r / inner) * (size_t)ld_outer + (size_t)(r % inner) * (size_t)ld;
  }
};

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
// A difference to the row's reference is held at this: -inf and the lowest float have at -1e30 all
// the same a weight of exactly 0, and 0 * -1e30 stays 0 where 0 * -inf would not.
constexpr float kFarBelow = -1e30f;

#if defined(__HIPCC__)

// Rows start at any element, so the loads are declared with the element's alignment only; the
// hardware takes global accesses of 16 bytes at any address.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int DTYPE>
struct Elem;

template <>
struct Elem<ICAP_DTYPE_F32> {
  typedef float type;
  static constexpr int kVec = 4;
  static constexpr uint32_t kNothing = 0xff800000u;      // 32 bits of -inf
  __device__ static float up(float v) { return v; }
  __device__ static float down(float v) { return v; }
  __device__ static void unpack(u32x4 raw, float (&x)[kVec]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(raw[i]);
  }
  __device__ static u32x4 pack(const float (&x)[kVec]) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(x[i]);
    return r;
  }
};

template <>
struct Elem<ICAP_DTYPE_BF16> {
  typedef __bf16 type;
  static constexpr int kVec = 8;
  static constexpr uint32_t kNothing = 0xff80ff80u;
  __device__ static float up(__bf16 v) { return (float)v; }
  __device__ static __bf16 down(float v) { return (__bf16)v; }
  __device__ static void unpack(u32x4 raw, float (&x)[kVec]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(raw[i] << 16);
      x[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u);
    }
  }
  __device__ static u32x4 pack(const float (&x)[kVec]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bf16x2 two = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
      r[i] = __builtin_bit_cast(uint32_t, two);
    }
    return r;
  }
};

template <>
struct Elem<ICAP_DTYPE_F16> {
  typedef _Float16 type;
  static constexpr int kVec = 8;
  static constexpr uint32_t kNothing = 0xfc00fc00u;
  __device__ static float up(_Float16 v) { return (float)v; }
  __device__ static _Float16 down(float v) { return (_Float16)v; }
  __device__ static void unpack(u32x4 raw, float (&x)[kVec]) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 two = __builtin_bit_cast(f16x2, (uint32_t)raw[i]);
      x[2 * i] = (float)two[0];
      x[2 * i + 1] = (float)two[1];
    }
  }
  __device__ static u32x4 pack(const float (&x)[kVec]) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f16x2 two = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      r[i] = __builtin_bit_cast(uint32_t, two);
    }
    return r;
  }
};

// 16 bytes from any address.  STREAM: data that nothing which follows will find in the caches - the
// last level holds 256 MB - and that need not push out what else is there (non-temporal).  A template
// parameter all the way: of two accesses in the branches of an if the compiler makes one.
template <bool STREAM>
__device__ __forceinline__ u32x4 load16(const void* p) {
  return STREAM ? __builtin_nontemporal_load((const u32x4_any*)p) : *(const u32x4_any*)p;
}
template <bool STREAM>
__device__ __forceinline__ void store16(void* p, u32x4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store((u32x4_any)v, (u32x4_any*)p);
  else *(u32x4_any*)p = v;
}

// n elements from p on, n = kVec (one 16-byte access) or 1.  No bounds and no branch, so that a
// batch of loads stays in flight together: the caller keeps col + n inside the row.
template <int DTYPE, int n>
struct Piece {
  typedef typename Elem<DTYPE>::type type;
  u32x4 raw;
  template <bool STREAM = false>
  __device__ __forceinline__ void load(const type* p) { raw = load16<STREAM>(p); }
  __device__ __forceinline__ void unpack(float (&x)[n]) const { Elem<DTYPE>::unpack(raw, x); }
  template <bool STREAM = false>
  __device__ static __forceinline__ void store(type* p, const float (&x)[n]) {
    store16<STREAM>(p, Elem<DTYPE>::pack(x));
  }
};
template <int DTYPE>
struct Piece<DTYPE, 1> {
  typedef typename Elem<DTYPE>::type type;
  type raw;
  template <bool STREAM = false>
  __device__ __forceinline__ void load(const type* p) { raw = *p; }
  __device__ __forceinline__ void unpack(float (&x)[1]) const { x[0] = Elem<DTYPE>::up(raw); }
  template <bool STREAM = false>
  __device__ static __forceinline__ void store(type* p, const float (&x)[1]) { *p = Elem<DTYPE>::down(x[0]); }
};

// Statistics of a soft-max over part of a row, in powers of two: with rate = log2(e) / tau and a
// reference c near rate * m, m the maximum so far,
//   y = rate * x - c (one fused multiply-add),   s = sum 2^y,   w = sum 2^y y.
// c is rate * m rounded; it is the same number for every element, so its rounding cancels.
//   log2 of the sum = c + log2 s,   entropy = ln 2 (log2 s - w / s)
// Parts join in a tree of a fixed shape, so a row's result does not depend on timing.  A part of -inf
// alone has m = -inf and, as its reference is finite (row_ref), s = 0 and no NaN.  A NaN, and the
// inf - inf of an infinite maximum, end in s and stay; m passes a NaN over.
struct RowStats {
  float m, s, w;
};

__device__ __forceinline__ RowStats row_stats_empty() { return {-INFINITY, 0.f, 0.f}; }

// Held within +-2^24, where the rounding of rate * m is at most one: a part further below has
// y <= 0 and next to no weight beside any other, and a row whose own maximum is further out is summed
// another way (row_stats_add_far).
constexpr float kRefLimit = 16777216.f;
__device__ __forceinline__ float row_ref(float m, float rate) {
  return fminf(fmaxf(m * rate, -kRefLimit), kRefLimit);
}

template <int n>
__device__ __forceinline__ void row_stats_add(float& s, float& w, const float (&x)[n], float rate, float c) {
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const float y = __builtin_fmaf(x[i], rate, -c);
    const float e = __builtin_amdgcn_exp2f(y);
    s += e;
    w = __builtin_fmaf(e, fmaxf(y, kFarBelow), w);
  }
}
template <int n>
__device__ __forceinline__ void row_sum_add(float& s, const float (&x)[n], float rate, float c) {
#pragma unroll
  for (int i = 0; i < n; ++i) s += __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], rate, -c));
}
template <int n>
__device__ __forceinline__ float row_max(float m, const float (&x)[n]) {
#pragma unroll
  for (int i = 0; i < n; ++i) m = fmaxf(m, x[i]);
  return m;
}
// Takes sums from reference a to reference b.  (No contraction here and in the join: a product
// fused into one side's addition would make the join of a and b differ from that of b and a, and the
// lanes of a butterfly end with different last bits.)
__device__ __forceinline__ void row_stats_move(float& s, float& w, float a, float b) {
#pragma clang fp contract(off)
  const float d = a - b;      // finite, both references are
  const float f = __builtin_amdgcn_exp2f(d);
  w = f * (w + s * d);
  s *= f;
}

__device__ __forceinline__ RowStats row_stats_join(RowStats a, RowStats b, float rate) {
#pragma clang fp contract(off)
  const float m = fmaxf(a.m, b.m), c = row_ref(m, rate);
  row_stats_move(a.s, a.w, row_ref(a.m, rate), c);
  row_stats_move(b.s, b.w, row_ref(b.m, rate), c);
  return {m, a.s + b.s, a.w + b.w};
}

// Joins the parts of `lanes` neighbouring lanes (a power of two); each of them gets the result.
template <int lanes>
__device__ __forceinline__ RowStats row_stats_lanes(RowStats a, float rate) {
#pragma unroll
  for (int d = lanes / 2; d > 0; d >>= 1) {
    const RowStats o = {__shfl_xor(a.m, d, 64), __shfl_xor(a.s, d, 64), __shfl_xor(a.w, d, 64)};
    a = row_stats_join(a, o, rate);
  }
  return a;
}

// One element of a row whose maximum m is known and so large that rate * x would overflow or round off
// what tells the elements apart: y = rate (x - m).
__device__ __forceinline__ void row_stats_add_far(RowStats& a, float x, float rate) {
  const float y = (x - a.m) * rate;
  const float e = __builtin_amdgcn_exp2f(y);
  a.s += e;
  a.w = __builtin_fmaf(e, fmaxf(y, kFarBelow), a.w);
}

// What a row's joined statistics say; far(m) sums the row again by row_stats_add_far.
struct RowResult {
  float m;          // the maximum; -inf in a row without a number: all -inf, or NaN as well
  float log_s;      // ln sum exp((x - m) / tau)
  float entropy;
  bool none;        // every element is -inf
  bool far;         // c stands too far out for rate * x - c to tell the elements apart
  float c, s;       // unless far: the reference, and the sum relative to it
};
template <class Far>
__device__ __forceinline__ RowResult row_result(RowStats a, float rate, Far far) {
  const float c = row_ref(a.m, rate);
  float off = __builtin_fmaf(a.m, rate, -c);      // of the maximum from the reference
  RowResult r;
  r.far = !(fabsf(c) < kRefLimit) && a.m != -INFINITY;
  if (r.far) {
    a = far(a.m);
    off = 0.f;
  }
  r.c = c;
  r.s = a.s;
  const float log_s = logf(a.s);
  r.none = a.s == 0.f;
  r.m = a.m;
  r.log_s = r.none ? 0.f : log_s - off * kLn2;
  r.entropy = r.none ? 0.f : log_s - kLn2 * (a.w / a.s);
  return r;
}

// A row in the hands of a workgroup of WAVES waves: pieces of kVec elements, thread t holding the
// pieces t, t + threads, ..., and the V % kVec elements behind the last whole piece one each.
// NV > 0: up to NV pieces a thread, which stay in registers, so that the row is read once;
// NV = 0: any length, read again for the second look.
template <int DTYPE, int WAVES, int NV, bool STREAM>
struct Row {
  typedef Elem<DTYPE> E;
  typedef typename E::type type;
  static constexpr int kThreads = WAVES * 64;
  static constexpr int kBatch = 4;      // loads in flight of a row that is not held
  static constexpr bool kHeld = NV > 0;
  const type* x;
  int V, pieces;
  u32x4 raw[kHeld ? NV : 1];
  float tail;          // -inf without one

  __device__ __forceinline__ u32x4 read(int i) const {
    // (a thread without an i-th piece reads the last one and forgets it: no branch round a load)
    u32x4 r = load16<STREAM && kHeld>(x + (size_t)min(i, pieces - 1) * E::kVec);
    if (i >= pieces) r = u32x4{E::kNothing, E::kNothing, E::kNothing, E::kNothing};
    return r;
  }
  __device__ __forceinline__ int tail_col() const { return pieces * E::kVec + (int)threadIdx.x; }

  __device__ __forceinline__ void open(const type* row, int n) {
    x = row;
    V = n;
    pieces = n / E::kVec;
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * kThreads < pieces) raw[j] = read(j * kThreads + threadIdx.x);
    }
    tail = tail_col() < n ? E::up(x[tail_col()]) : -INFINITY;
  }

  // f(values, first column) for each of this thread's pieces, then for its single element; columns
  // past the row's end are -inf
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * kThreads < pieces) {
          float v[E::kVec];
          E::unpack(raw[j], v);
          f(v, (j * kThreads + (int)threadIdx.x) * E::kVec);
        }
    } else {
      for (int i0 = 0; i0 < pieces; i0 += kBatch * kThreads) {
        u32x4 r[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) r[j] = read(i0 + j * kThreads + threadIdx.x);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          float v[E::kVec];
          E::unpack(r[j], v);
          f(v, (i0 + j * kThreads + (int)threadIdx.x) * E::kVec);
        }
      }
    }
    const float v[1] = {tail};
    f(v, tail_col());
  }

  // This thread's part of the sum; no entropy.
  __device__ __forceinline__ RowStats sums(float rate) const {
    RowStats a = row_stats_empty();
    if constexpr (kHeld) {
      each([&](const auto& v, int) { a.m = row_max(a.m, v); });
      const float c = row_ref(a.m, rate);
      each([&](const auto& v, int) { row_sum_add(a.s, v, rate, c); });
    } else {
      for (int i0 = 0; i0 < pieces; i0 += kBatch * kThreads) {
        float v[kBatch][E::kVec];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) E::unpack(read(i0 + j * kThreads + threadIdx.x), v[j]);
        float m = a.m;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) m = row_max(m, v[j]);
        const float c = row_ref(m, rate);
        row_stats_move(a.s, a.w, row_ref(a.m, rate), c);
        a.m = m;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) row_sum_add(a.s, v[j], rate, c);
      }
      const float v[1] = {tail};
      const float m = row_max(a.m, v), c = row_ref(m, rate);
      row_stats_move(a.s, a.w, row_ref(a.m, rate), c);
      a.m = m;
      row_sum_add(a.s, v, rate, c);
    }
    return a;
  }

  // out[column] = factor * exp((value - m) / tau - log_s) in the row's type; out may be the row
  // itself (each thread writes what it alone read)
  __device__ __forceinline__ void write_softmax(type* out, const RowResult& r, float rate, float factor) const {
    if (r.far) {
      const float inv_s = factor * __builtin_amdgcn_exp2f(-r.log_s * kLog2e);
      for (int i = threadIdx.x; i < V; i += kThreads)
        out[i] = E::down(__builtin_amdgcn_exp2f((E::up(x[i]) - r.m) * rate) * inv_s);
      return;
    }
    const float c = r.c, inv_s = factor / r.s;
    each([&](const auto& v, int col) {
      constexpr int n = sizeof(v) / sizeof(float);
      if (col + n > V) return;
      float g[n];
#pragma unroll
      for (int e = 0; e < n; ++e) g[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], rate, -c)) * inv_s;
      Piece<DTYPE, n>::template store<STREAM>(out + col, g);
    });
  }
};

// Whether a call's reads or writes count as a stream.  Measured with the next operator reading the
// result: written past the caches a lookup's 134 MB take 28 instead of 38 us and both together 82
// instead of 84, 67 MB 41.4 against 41.4; read past them 410 MB of logits take 64 instead of 73 us,
// but at 195 MB a gradient that follows loses more than that gains.
inline bool stream_reads(size_t bytes) { return bytes > (size_t)256 << 20; }
inline bool stream_writes(size_t bytes) { return bytes > (size_t)96 << 20; }

// Zeros in a row of V elements.
template <int DTYPE, int WAVES, bool STREAM>
__device__ __forceinline__ void write_zeros(typename Elem<DTYPE>::type* out, int V) {
  constexpr int n = Elem<DTYPE>::kVec;
  const float zero[n] = {}, one[1] = {};
  for (int i = threadIdx.x; i < V / n; i += WAVES * 64) Piece<DTYPE, n>::template store<STREAM>(out + (size_t)i * n, zero);
  const int c = V / n * n + (int)threadIdx.x;
  if (c < V) Piece<DTYPE, 1>::store(out + c, one);
}

// Order of the alternatives: by value, then by the lower column; -0 and +0 are equal, and a NaN
// counts as -inf.  A larger key is a better alternative and no two columns share one.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint((v == v ? v : -INFINITY) + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long rank_key(float v, int col) {
  return ((unsigned long long)order_of(v) << 32) | (0xffffffffu - (uint32_t)col);
}
__device__ __forceinline__ int rank_col(unsigned long long key) {
  return (int)(0xffffffffu - (uint32_t)key);
}

#endif  // __HIPCC__

}  // namespace icap
