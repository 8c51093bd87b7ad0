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

// Lanes of a wave exchange through LDS without a barrier of the workgroup: its LDS accesses are
// carried out in order, only the compiler has to keep them so.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kNotes = 128;        // batches, then columns, that a wave notes
constexpr int kBatchElems = 16;    // elements a lane reads at a time

struct TopScratch {                // of one wave
  float note_max[kNotes];
  int note[kNotes];
  unsigned long long key[kNotes];
};

// A value that at least k of the lanes reach, the k-th largest of their 64 or close below it: the bits
// of its order from the top down, until exactly k lanes reach it.  Lanes that tie have it exact.
__device__ __forceinline__ float kth_of_lanes(float v, int k) {
  const uint32_t mine = order_of(v);
  uint32_t bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t next = bound | (1u << bit);
    const int reach = __popcll(__ballot(mine >= next));
    if (reach >= k) bound = next;
    if (reach == k) break;
  }
  return fmaxf(order_value(bound), -INFINITY);      // (below -inf in the order: a NaN's bits)
}

// One wave's share of a row: pieces [from, to) of kVec elements, read once in batches of kBatch a
// lane, and for the row's last wave the elements behind the last whole piece.
template <int DTYPE, bool STREAM>
struct Share {
  typedef Elem<DTYPE> E;
  typedef typename E::type type;
  static constexpr int kBatch = kBatchElems / E::kVec;
  const type* x;
  int from, to, lane;
  int end;                     // columns of the share are [from * kVec, end)
  int tail_col;                // -1: no single element here
  float tail;

  __device__ __forceinline__ int piece(int b, int j) const { return from + (b * kBatch + j) * 64 + lane; }
  __device__ __forceinline__ u32x4 read(int i) const {
    u32x4 r = load16<STREAM>(x + (size_t)min(i, to - 1) * E::kVec);
    if (i >= to) r = u32x4{E::kNothing, E::kNothing, E::kNothing, E::kNothing};
    return r;
  }
};

// The share's statistics and, with TOP, its k best columns as ranked keys in best[0 .. k) (0: none
// left).  While the share is read the wave keeps a bound that at least k elements have reached - the
// k-th largest of the lanes' maxima so far, renewed after 1, 2, 4, 8 ... batches - and notes the
// batches of a lane that reach it; in the end some k to 2k of them are read again.  Batches come in
// the order of their columns, so what only equals a bound that stood before its batch has k better
// or equal elements at lower columns and is not noted: rows of equal logits (masked to the lowest
// value, or not trained yet) note one batch.  Where more batches than there are notes reach the
// bound before it is renewed, the share is read again for every alternative: 2560 rows of 50001 in
// bf16, 6000 columns at -inf and all others equal, take 2.3 ms with 16 alternatives.
template <int DTYPE, bool TOP, bool STREAM>
__device__ __forceinline__ RowStats share_scan(const Share<DTYPE, STREAM>& sh, float rate, int k, TopScratch& s,
                                               unsigned long long* best) {
  typedef Elem<DTYPE> E;
  constexpr int kBatch = Share<DTYPE, STREAM>::kBatch;
  const unsigned long long lower = (1ull << sh.lane) - 1;
  RowStats a = row_stats_empty();
  const int batches = (sh.to - sh.from + kBatch * 64 - 1) / (kBatch * 64);
  float lane_top = -INFINITY, bound = -INFINITY, stood = -INFINITY;
  int notes = 0, renew = 0;
  bool full = false;
  // a new bound, and of the notes only those that reach it
  auto squeeze = [&]() {
    bound = kth_of_lanes(lane_top, k);
    int kept = 0;
    wave_sync();
    for (int i0 = 0; i0 < notes; i0 += 64) {
      const int i = i0 + sh.lane;
      const bool there = i < notes;
      const float m = there ? s.note_max[i] : 0.f;
      const int what = there ? s.note[i] : 0;
      const bool keep = there && m >= bound;
      const unsigned long long mask = __ballot(keep);
      wave_sync();
      if (keep) {
        const int at = kept + __popcll(mask & lower);
        s.note_max[at] = m;
        s.note[at] = what;
      }
      kept += __popcll(mask);
      wave_sync();
    }
    notes = kept;
  };
  auto note = [&](float m, int what) {
    unsigned long long hit = __ballot(m >= bound && m > stood);
    if (hit && !full) {
      if (notes + __popcll(hit) > kNotes) {
        squeeze();
        hit = __ballot(m >= bound && m > stood);
        full = notes + __popcll(hit) > kNotes;
      }
      if (!full) {
        if ((hit >> sh.lane) & 1) {
          const int at = notes + __popcll(hit & lower);
          s.note_max[at] = m;
          s.note[at] = what;
        }
        notes += __popcll(hit);
      }
    }
    stood = bound;
  };
  for (int b = 0; b < batches; ++b) {
    u32x4 r[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) r[j] = sh.read(sh.piece(b, j));
    float v[kBatch][E::kVec];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      E::unpack(r[j], v[j]);
      top = row_max(top, v[j]);
    }
    const float m = fmaxf(a.m, top);
    const float c = row_ref(m, rate);
    row_stats_move(a.s, a.w, row_ref(a.m, rate), c);
    a.m = m;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) row_stats_add(a.s, a.w, v[j], rate, c);
    if constexpr (TOP) {
      lane_top = fmaxf(lane_top, top);
      if (b == renew) {
        bound = kth_of_lanes(lane_top, k);
        renew = 2 * b + 1;
      }
      note(top, b * 64 + sh.lane);
    }
  }
  const float tail[1] = {sh.tail};
  const float m = row_max(a.m, tail), c = row_ref(m, rate);
  row_stats_move(a.s, a.w, row_ref(a.m, rate), c);
  a.m = m;
  row_stats_add(a.s, a.w, tail, rate, c);
  if constexpr (TOP) {
    lane_top = fmaxf(lane_top, sh.tail);
    if (__any(sh.tail_col >= 0)) note(sh.tail_col >= 0 ? sh.tail : -INFINITY, -1 - sh.tail_col);
    squeeze();
    if (sh.lane < k) best[sh.lane] = 0;
    // f(value, column) for the elements of the noted batches, all lanes together (NaN: none here)
    auto each_noted = [&](auto f) {
      for (int t0 = 0; t0 < notes * kBatch; t0 += 64) {
        const int t = t0 + sh.lane;
        const bool there = t < notes * kBatch;
        const int what = there ? s.note[t / kBatch] : 0;
        const bool single = what < 0;      // one element behind the last piece
        const int i = sh.from + (what / 64 * kBatch + t % kBatch) * 64 + what % 64;
        float v[E::kVec];
#pragma unroll
        for (int e = 0; e < E::kVec; ++e) v[e] = NAN;
        if (there && !single && i < sh.to)
          E::unpack(*reinterpret_cast<const u32x4_any*>(sh.x + (size_t)i * E::kVec), v);
        if (there && single && t % kBatch == 0) v[0] = E::up(sh.x[-1 - what]);
#pragma unroll
        for (int e = 0; e < E::kVec; ++e) f(v[e], single ? -1 - what : i * E::kVec + e);
      }
    };
    // those that reach the bound, or if they are too many, as in rows of equal logits, or the bound is
    // -inf, those over it
    int count = kNotes + 1;
    for (int over = bound == -INFINITY; over < 2 && !full && count > kNotes; ++over) {
      count = 0;
      each_noted([&](float v, int col) {
        const bool is = over ? v > bound : v >= bound;
        const unsigned long long hit = __ballot(is);
        if (!hit) return;
        const int at = count + __popcll(hit & lower);
        if (is && at < kNotes) s.key[at] = rank_key(v, col);
        count += __popcll(hit);
      });
      wave_sync();
    }
    if (!full && count <= kNotes) {
      for (int i = sh.lane; i < count; i += 64) {
        const unsigned long long key = s.key[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += s.key[j] > key;
        if (rank < k) best[rank] = key;
      }
      if (count < k && bound == -INFINITY) {
        // the lowest of the other columns follow, all of which lie within the share's first 64
        const int col = sh.from * E::kVec + sh.lane;
        const bool other = col < sh.end && !(E::up(sh.x[min(col, sh.end - 1)]) > -INFINITY);
        const int at = count + __popcll(__ballot(other) & lower);
        if (other && at < k) best[at] = rank_key(-INFINITY, col);
      } else if (count < k) {
        // those that equal the bound follow, in the order of their columns
        int at = count, last = -1;
        for (int i = 0; i < notes && at < k; ++i) {
          const int what = __builtin_amdgcn_readfirstlane(s.note[i]);
          if (what < 0) {
            const bool equal = sh.tail_col >= 0 && sh.tail == bound;
            const int slot = at + __popcll(__ballot(equal) & lower);
            if (equal && slot < k) best[slot] = rank_key(bound, sh.tail_col);
            break;
          }
          if (what / 64 == last) continue;
          last = what / 64;
          for (int j = 0; j < kBatch && at < k; ++j) {
            float v[E::kVec];
            E::unpack(sh.read(sh.piece(last, j)), v);
            int slot = at;
#pragma unroll
            for (int e = 0; e < E::kVec; ++e) {
              const unsigned long long hit = __ballot(v[e] == bound);
              slot += __popcll(hit & lower);
              at += __popcll(hit);
            }
#pragma unroll
            for (int e = 0; e < E::kVec; ++e)
              if (v[e] == bound) {
                if (slot < k) best[slot] = rank_key(bound, sh.piece(last, j) * E::kVec + e);
                ++slot;
              }
          }
        }
      }
    } else {
      // more elements over the bound than fit: a round for each, over the noted batches or,
      // if those did not fit either, over the share
      unsigned long long below = ~0ull;
      for (int r = 0; r < k; ++r) {
        unsigned long long key = 0;
        auto look = [&](float v, int col) {
          const unsigned long long q = rank_key(v, col);
          if (v >= bound && q < below && q > key) key = q;
        };
        if (!full) each_noted(look);
        else
          for (int col = sh.from * E::kVec + sh.lane; col < sh.end; col += 64) look(E::up(sh.x[col]), col);
        for (int d = 32; d > 0; d >>= 1) key = max(key, (unsigned long long)__shfl_xor(key, d, 64));
        below = key;
        if (sh.lane == 0) best[r] = key;
        if (key == 0) break;
      }
    }
  }
  return a;
}

// P waves to a row, 4 / P rows to a workgroup (P = 1, 2) or one (P = 4, 8).  The waves of a row
// meet once, when each has its share's statistics and its k best columns in LDS; the first joins
// them.  Rows alone in a wave wait for nobody.
//
// Bound by one read of the logits: 10240 rows of 10000 in fp32, a quarter of them padding, 53 us (5.8
// TB/s), 2560 rows of 50001 in bf16 with 16 alternatives 57 us (4.5 TB/s; without alternatives 49 us,
// the bound and the notes are vector instructions).  Rows that are masked but for a few columns
// cost the same within a fifth (few of 50001 bf16 columns left over the lowest value 67 us, nothing
// but equal logits 62); those whose every logit is past 2^24 are read twice (111 us).
template <int DTYPE, int P, bool TOP, bool STREAM>
__global__ __launch_bounds__((P < 4 ? 4 : P) * 64, 8) void token_log_probs_kernel(ScoreArgs p) {
  typedef Elem<DTYPE> E;
  constexpr int WAVES = P < 4 ? 4 : P;
  __shared__ RowStats s_part[WAVES];
  __shared__ TopScratch s_top[TOP ? WAVES : 1];
  __shared__ unsigned long long s_best[TOP ? WAVES : 1][ICAP_MAX_ALTERNATIVES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int part = wave % P;
  const int row = (blockIdx.y * gridDim.x + blockIdx.x) * (WAVES / P) + wave / P;
  const bool live = row < p.N;
  const int token = live ? p.tokens[row] : p.pad;
  RowStats a = row_stats_empty();
  const typename E::type* x = (const typename E::type*)p.logits + p.view.at(live ? row : 0);
  const bool scored = live && token != p.pad;
  if (scored) {
    const int pieces = p.V / E::kVec;
    // shares of whole waves' pieces
    const int each = ((pieces + P - 1) / P + 63) / 64 * 64;
    Share<DTYPE, STREAM> sh;
    sh.x = x;
    sh.from = min(pieces, part * each);
    sh.to = min(pieces, sh.from + each);
    sh.lane = lane;
    sh.end = part == P - 1 ? p.V : sh.to * E::kVec;
    const int tail_col = pieces * E::kVec + lane;
    sh.tail_col = part == P - 1 && tail_col < p.V ? tail_col : -1;
    sh.tail = sh.tail_col >= 0 ? E::up(x[tail_col]) : -INFINITY;
    a = row_stats_lanes<64>(share_scan<DTYPE, TOP, STREAM>(sh, kLog2e, p.k, s_top[TOP ? wave : 0], s_best[TOP ? wave : 0]), kLog2e);
  }
  if constexpr (P > 1) {
    if (lane == 0) s_part[wave] = a;
    __syncthreads();
    if (part != 0) return;
    a = lane < P ? s_part[wave + lane] : row_stats_empty();
    a = row_stats_lanes<64>(a, kLog2e);
  } else if constexpr (TOP) {
    wave_sync();
  }
  if (!live) return;
  if (!scored) {
    if (lane == 0) {
      p.log_probs[row] = p.entropy[row] = 0.f;
      p.stats[2 * (size_t)row] = p.stats[2 * (size_t)row + 1] = 0.f;
    }
    if (TOP && lane < p.k) {
      p.top_ids[(size_t)row * p.k + lane] = -1;
      p.top_log_probs[(size_t)row * p.k + lane] = 0.f;
    }
    return;
  }
  const RowResult r = row_result(a, kLog2e, [&](float m) {
    RowStats f = {m, 0.f, 0.f};
    const int pieces = p.V / E::kVec;
#pragma unroll 4
    for (int i = lane; i < pieces; i += 64) {
      float v[E::kVec];
      E::unpack(load16<false>(x + (size_t)i * E::kVec), v);
#pragma unroll
      for (int e = 0; e < E::kVec; ++e) row_stats_add_far(f, v[e], kLog2e);
    }
    const int tail = pieces * E::kVec + lane;
    if (tail < p.V) row_stats_add_far(f, E::up(x[tail]), kLog2e);
    return row_stats_lanes<64>(f, kLog2e);
  });
  if (lane == 0) {
    const bool inside = token >= 0 && token < p.V;
    const float x_t = inside ? E::up(x[token]) : NAN;
    p.log_probs[row] = inside && r.none ? -INFINITY : (x_t - r.m) - r.log_s;
    p.entropy[row] = r.entropy;
    p.stats[2 * (size_t)row] = r.m;
    p.stats[2 * (size_t)row + 1] = r.log_s;
  }
  if constexpr (TOP) {
    unsigned long long mine = 0;
    if constexpr (P == 1) {
      if (lane < p.k) mine = s_best[wave][lane];
    } else {
      // lane i at the head of share i's list; the best head goes out and its list moves up
      int at = 0;
      unsigned long long head = lane < P ? s_best[wave + lane][0] : 0;
      for (int i = 0; i < p.k; ++i) {
        unsigned long long key = head;
        for (int d = P / 2; d > 0; d >>= 1) key = max(key, (unsigned long long)__shfl_xor(key, d, 64));
        key = __shfl(key, 0, 64);
        if (lane == i) mine = key;
        if (head == key && lane < P) head = ++at < p.k ? s_best[wave + lane][at] : 0;
      }
    }
    if (lane < p.k) {
      const int col = rank_col(mine);
      p.top_ids[(size_t)row * p.k + lane] = col;
      p.top_log_probs[(size_t)row * p.k + lane] = r.none ? -INFINITY : (E::up(x[col]) - r.m) - r.log_s;
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
  int shares;      // of a row
};

// d log p_t / d x_j = [j = t] - p_j,   d H / d x_j = -p_j (log p_j + H)
// Element by element, so a row is cut into shares of kGradPieces pieces a thread.  Bound by one read
// and one write: 10240 rows of 10000 in fp32 124 us (5.8 TB/s of both, a quarter padding that is not read), 1271 of
// 50001 in fp16 44 us (5.5 TB/s).
constexpr int kGradPieces = 4;

template <int DTYPE, bool STREAM>
__global__ __launch_bounds__(NT) void token_log_probs_grad_kernel(ScoreGradArgs p) {
  typedef Elem<DTYPE> E;
  typedef typename E::type type;
  const long long block = (long long)blockIdx.y * gridDim.x + blockIdx.x;
  const int row = (int)(block / p.shares), share = (int)(block % p.shares), tid = threadIdx.x;
  if (row >= p.N) return;
  const int token = p.tokens[row];
  const type* x = (const type*)p.logits + p.view.at(row);
  type* g = (type*)p.out + p.out_view.at(row);
  float g_lp = p.g_lp ? p.g_lp[row] : 0.f;
  const float g_h = p.g_h ? p.g_h[row] : 0.f;
  const float m = p.stats[2 * (size_t)row], log_s = p.stats[2 * (size_t)row + 1], h = p.entropy[row];
  const int pieces = p.V / E::kVec, first = share * NT * kGradPieces + tid;
  const int tail = pieces * E::kVec + tid;
  const bool has_tail = share == p.shares - 1 && tail < p.V;
  const bool none = m == -INFINITY && log_s == log_s;      // (a row of NaN and -inf has that maximum too)
  if (token == p.pad || none || (g_lp == 0.f && g_h == 0.f)) {
    const float zero[E::kVec] = {};
#pragma unroll
    for (int j = 0; j < kGradPieces; ++j)
      if (first + j * NT < pieces)
        Piece<DTYPE, E::kVec>::template store<STREAM>(g + (size_t)(first + j * NT) * E::kVec, zero);
    if (has_tail) g[tail] = E::down(0.f);
    return;
  }
  if ((token < 0 || token >= p.V) && g_lp != 0.f) g_lp = NAN;
  const float inv_s = __builtin_amdgcn_exp2f(-log_s * kLog2e);
  // (e u before g_h: where e is 0 - a masked logit - g_h u may pass fp32's range, and 0 inf is NaN)
  auto grad = [&](float v, int c) {
    const float d = v - m;
    const float e = __builtin_amdgcn_exp2f(d * kLog2e) * inv_s;
    const float u = fmaxf(d, kFarBelow) - log_s + h;
    return (c == token ? g_lp : 0.f) - __builtin_fmaf(g_h, e * u, e * g_lp);
  };
  u32x4 raw[kGradPieces];
  float t = 0.f;
  if (has_tail) t = E::up(x[tail]);
#pragma unroll
  for (int j = 0; j < kGradPieces; ++j)
    if (pieces > 0)
      raw[j] = load16<STREAM>(x + (size_t)min(first + j * NT, pieces - 1) * E::kVec);
#pragma unroll
  for (int j = 0; j < kGradPieces; ++j) {
    const int i = first + j * NT;
    if (i >= pieces) break;
    float v[E::kVec];
    E::unpack(raw[j], v);
#pragma unroll
    for (int e = 0; e < E::kVec; ++e) v[e] = grad(v[e], i * E::kVec + e);
    Piece<DTYPE, E::kVec>::template store<STREAM>(g + (size_t)i * E::kVec, v);
  }
  if (has_tail) g[tail] = E::down(grad(t, tail));
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

// An element's bits, and what they stand for: apart, so that a load can stay in flight meanwhile.
__device__ __forceinline__ uint32_t load_bits(const void* p, int dtype, size_t i) {
  return dtype == ICAP_DTYPE_F32 ? ((const uint32_t*)p)[i] : ((const uint16_t*)p)[i];
}
__device__ __forceinline__ float bits_value(uint32_t bits, int dtype) {
  if (dtype == ICAP_DTYPE_F32) return __uint_as_float(bits);
  if (dtype == ICAP_DTYPE_BF16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// Only what goes through LDS is ordered: loads and stores of device memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// loss = tau^2 sum_k q_k (log q_k - log p[id_k]),  q = soft-max of the teacher's K logits at tau,
// p = soft-max of the row at tau;   d loss / d x_j = tau (p_j - sum over k with id_k = j of q_k)
//
// A workgroup reads a row into registers, sums it, and writes the gradient from there; one barrier
// hands the waves' sums and the teacher's q round.  Bound by one read and one write: 10240 rows of
// 10000 in fp32 135 us with a quarter padding.  2048 of 50000 in bf16 take 97 us (4.0 TB/s): three
// such rows fit a compute unit, and reading, summing and writing overlap only between them.  (A
// workgroup that goes through several rows and reads the next one into a second set of registers was
// slower, 158 against 122 us for 2560 rows: the registers cost it half of its neighbours, which
// hide the same latency.)
//
// The second launch bound holds a thread to the registers that 8 waves a SIMD leave (7 and 6 for 10 and
// 13 pieces); without it 4000 rows of 20000 in fp32 take 161 instead of 120 us.
template <int DTYPE, int WAVES, int NV, bool STREAM>
__global__ __launch_bounds__(WAVES * 64, NV == 13 ? 6 : NV == 10 ? 7 : 8) void distill_loss_kernel(DistillArgs p) {
  typedef Elem<DTYPE> E;
  typedef typename E::type type;
  __shared__ RowStats s_part[WAVES];
  __shared__ int s_id[kMaxTeacher];
  __shared__ float s_q[kMaxTeacher], s_log_q[kMaxTeacher], s_x[kMaxTeacher];
  __shared__ int s_state;                    // 1: entries there, 2: an id outside the vocabulary
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.y * gridDim.x + blockIdx.x;
  if (row >= p.N) return;
  const float inv_tau = 1.f / p.tau, rate = kLog2e * inv_tau;
  type* g = p.out ? (type*)p.out + p.out_view.at(row) : nullptr;
  // every wave looks for itself whether the teacher has an entry
  const int32_t* ids = p.t_ids + (size_t)row * p.K;
  const int id0 = lane < p.K ? ids[lane] : -1;
  bool any = id0 != -1;
  for (int k = lane + 64; k < p.K; k += 64) any |= ids[k] != -1;
  if (!__any(any)) {
    if (tid == 0) p.loss[row] = 0.f;
    if (g) write_zeros<DTYPE, WAVES, STREAM>(g, p.V);
    return;
  }
  // The last wave (its share of the row is the shortest) sees to the teacher's entries.  It asks for
  // the first 64 before the row, whose sums they then do not delay.
  const type* x = (const type*)p.logits + p.view.at(row);
  const bool teaches = wave == WAVES - 1;
  uint32_t t0 = 0, x0 = 0;
  if (teaches && id0 != -1) {
    t0 = load_bits(p.t_logits, p.t_dtype, (size_t)row * p.K + lane);
    if ((unsigned)id0 < (unsigned)p.V) x0 = load_bits(x, DTYPE, id0);
  }
  Row<DTYPE, WAVES, NV, STREAM> data;
  data.open(x, p.V);
  const float coef = g ? p.g_loss[row] * p.tau : 0.f;
  RowStats part = row_stats_lanes<64>(data.sums(rate), rate);
  if (lane == 0) s_part[wave] = part;
  if (teaches) {        // (a lane reads back only what it wrote itself)
    bool bad = false, entries = false;
    float top = -INFINITY;
#pragma unroll 1
    for (int k = lane; k < p.K; k += 64) {
      const int id = k < 64 ? id0 : ids[k];
      const bool in = (unsigned)id < (unsigned)p.V;
      float t = -INFINITY, xk = 0.f;
      if (id != -1) t = bits_value(k < 64 ? t0 : load_bits(p.t_logits, p.t_dtype, (size_t)row * p.K + k), p.t_dtype);
      if (in) xk = bits_value(k < 64 ? x0 : load_bits(x, DTYPE, id), DTYPE);
      bad |= id != -1 && !in && !(t == -INFINITY);      // (an absent entry's id says nothing)
      entries |= !(t == -INFINITY);
      top = fmaxf(top, t);
      s_id[k] = in ? id : -1;
      s_x[k] = xk;
      s_log_q[k] = t;
    }
    bad = __any(bad);
    entries = __any(entries);
    top = wave_max(top);
    float sum = 0.f;
#pragma unroll 1
    for (int k = lane; k < p.K; k += 64) {
      const float t = s_log_q[k];
      const float q = t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((t - top) * rate);
      s_q[k] = q;
      sum += q;
    }
    sum = wave_sum(sum);
    const float log_sum = logf(sum), inv = 1.f / sum;
#pragma unroll 1
    for (int k = lane; k < p.K; k += 64) {
      s_log_q[k] = (s_log_q[k] - top) * inv_tau - log_sum;
      s_q[k] *= inv;
    }
    if (lane == 0) s_state = (entries ? 1 : 0) | (bad ? 2 : 0);
  }
  lds_barrier();
  const RowResult r =
      row_result(row_stats_lanes<WAVES>(s_part[lane & (WAVES - 1)], rate), rate, [&](float m) {
        RowStats f = {m, 0.f, 0.f};
        for (int i = tid; i < p.V; i += WAVES * 64) row_stats_add_far(f, E::up(data.x[i]), rate);
        f = row_stats_lanes<64>(f, rate);
        __syncthreads();
        if (lane == 0) s_part[wave] = f;
        __syncthreads();
        return row_stats_lanes<WAVES>(s_part[lane & (WAVES - 1)], rate);
      });
  const bool bad = s_state & 2, entries = s_state;
  if (teaches) {
    float sum = 0.f;
#pragma unroll 1
    for (int k = lane; k < p.K; k += 64) {
      const float q = s_q[k];
      const float lp = r.none ? -INFINITY : (s_x[k] - r.m) * inv_tau - r.log_s;
      if (!(q == 0.f)) sum += q * (s_log_q[k] - lp);
    }
    sum = wave_sum(sum) * p.tau * p.tau;
    if (lane == 0) p.loss[row] = bad ? NAN : entries ? sum : 0.f;
  }
  if (!g) return;
  if (!entries || coef == 0.f || (r.none && !bad)) {
    write_zeros<DTYPE, WAVES, STREAM>(g, p.V);
    return;
  }
  const float c0 = bad ? NAN : coef;
  data.write_softmax(g, r, rate, c0);
  if (bad) return;
  __syncthreads();      // the columns' first values are stored
  // the teacher's columns again, the first of several entries with the same id for all of them
  const float inv_s = __builtin_amdgcn_exp2f(-r.log_s * kLog2e);
  for (int k = tid; k < p.K; k += WAVES * 64) {
    const int id = s_id[k];
    bool first = id >= 0;
    float sum = 0.f;
    for (int j = 0; j < p.K; ++j) {
      const bool same = s_id[j] == id;
      sum += same ? s_q[j] : 0.f;
      if (same && j < k) first = false;
    }
    if (first) g[id] = E::down(c0 * (__builtin_amdgcn_exp2f((s_x[k] - r.m) * rate) * inv_s - sum));
  }
}

constexpr int kMostRows = 1 << 30;      // workgroup numbers stay within 31 bits, the last row of them unfilled

dim3 row_grid(int N) {
  const int x = N < 65536 ? N : 65536;
  return dim3((unsigned)x, (unsigned)ceil_div(N, x));
}

size_t row_bytes(int dtype, int N, int V) { return (size_t)N * V * (dtype == ICAP_DTYPE_F32 ? 4 : 2); }

int check_rows(const char* what, int dtype, int N, int V, const RowView& v) {
  ICAP_REQUIRE(dtype == ICAP_DTYPE_F32 || dtype == ICAP_DTYPE_BF16 || dtype == ICAP_DTYPE_F16,
               "%s: unknown dtype %d", what, dtype);
  ICAP_REQUIRE(N > 0 && V > 0, "%s: bad shape", what);
  if (N > kMostRows || V > kMostRows)
    return fail(ICAP_ERR_UNSUPPORTED, "%s: N and V go up to %d", what, kMostRows);
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

// Waves for a row of scores: as few as give the card some ten waves a compute unit, as long as each
// has 256 pieces and more to read.  Measured with 16 alternatives, us at 1 / 2 / 4 / 8 waves: 2560 rows of
// 50000 in bf16 65 / 58 / 66 / 68, 10240 of 10000 in bf16 51 / 60 / 76 / 121, 700 of 131072 in fp32
// 130 / 85 / 81 / 88, 300 of 50000 in bf16 41 / 28 / 22 / 21.
int waves_per_row(int dtype, int N, int V) {
  const int pieces = V / (dtype == ICAP_DTYPE_F32 ? 4 : 8);
  int P = 1;
  while (P < 8 && (long long)N * P < 2700 && pieces > P * 256) P *= 2;
  return P;
}

// Waves for a row and pieces a thread holds: as few waves as keep some 10 pieces a thread or less, more
// where two or three such rows still fit a compute unit's registers, and longer rows read twice.
// Few rows go to large workgroups: their time is that of one row.  Measured, us, with one read and one
// write of the logits at the rate of a copy in brackets: 40000 rows of 2000 in fp32 130 (121) by 2
// waves of 4, and before the teacher's entries were asked for ahead of the row 140 against 156 by 1 of 8
// and 162 by 4 of 4; 10240 of 10000 in fp32 149 (155) by 8 of 5, 161 then against 166 by 4 of 10; in bf16
// 81 (77) by 4 of 10, 87 then against 117 by 8 of 5; 2560 of 50000 in bf16 112 (97) by 8 of 13, 108 then
// against 115 by 16 of 7 and 113 by 4 of 25; 4000 of 20000 in fp32 120 (121) by 16 of 7, 121 then against
// 128 by 8 of 13; 2048 of 50000 in fp32 189 (155) read twice, 201 then by 16 of 13.
struct RowShape {
  int waves, held;
};
RowShape row_shape(int dtype, int N, int V) {
  const int pieces = V / (dtype == ICAP_DTYPE_F32 ? 4 : 8);
  const bool many = N > 512;      // two rows a compute unit
  if (pieces <= 64 * (many ? 4 : 1)) return {1, 4};
  if (many && pieces <= 128 * 4) return {2, 4};
  if (pieces <= 256 * (many ? 4 : 2)) return {4, 4};
  if (many && pieces <= 512 * 5) return dtype == ICAP_DTYPE_F32 ? RowShape{8, 5} : RowShape{4, 10};
  if (many && pieces <= 512 * 13 && dtype != ICAP_DTYPE_F32) return {8, 13};
  if (pieces <= 1024 * 7) return {16, 7};
  return {16, 0};
}

#define ICAP_BY_SHAPE(D, shape, call)              \
  do {                                             \
    if ((shape).waves == 1) call(D, 1, 4);         \
    else if ((shape).waves == 2) call(D, 2, 4);    \
    else if ((shape).waves == 4) { if ((shape).held == 4) call(D, 4, 4); else call(D, 4, 10); } \
    else if ((shape).waves == 8) { if ((shape).held == 5) call(D, 8, 5); else call(D, 8, 13); } \
    else if ((shape).held == 7) call(D, 16, 7);    \
    else call(D, 16, 0);                           \
  } while (0)
#define ICAP_BY_ROWS(dtype, shape, call)                                           \
  do {                                                                             \
    if ((dtype) == ICAP_DTYPE_F32) ICAP_BY_SHAPE(ICAP_DTYPE_F32, shape, call);     \
    else if ((dtype) == ICAP_DTYPE_BF16) ICAP_BY_SHAPE(ICAP_DTYPE_BF16, shape, call); \
    else ICAP_BY_SHAPE(ICAP_DTYPE_F16, shape, call);                               \
  } while (0)
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
  const int P = waves_per_row(dtype, N, V);
  const dim3 grid = row_grid(ceil_div(N, P < 4 ? 4 / P : 1)), block((P < 4 ? 4 : P) * 64);
  const bool streamed = stream_reads(row_bytes(dtype, N, V));
#define LAUNCH_P(D, P)                                                                       \
  do {                                                                                       \
    if (top_k && streamed) LAUNCH_4(D, P, true, true);                                       \
    else if (top_k) LAUNCH_4(D, P, true, false);                                             \
    else if (streamed) LAUNCH_4(D, P, false, true);                                          \
    else LAUNCH_4(D, P, false, false);                                                       \
  } while (0)
#define LAUNCH_4(D, P, TOP, S)                                                               \
  hipLaunchKernelGGL((token_log_probs_kernel<D, P, TOP, S>), grid, block, 0, (hipStream_t)stream, a)
#define LAUNCH(D)               \
  do {                          \
    if (P == 1) LAUNCH_P(D, 1);      \
    else if (P == 2) LAUNCH_P(D, 2); \
    else if (P == 4) LAUNCH_P(D, 4); \
    else LAUNCH_P(D, 8);             \
  } while (0)
  ICAP_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
#undef LAUNCH_4
#undef LAUNCH_P
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
  ScoreGradArgs a{logits, view, tokens, N, V, pad_token, stats, entropy, grad_log_probs, grad_entropy, dlogits, out,
                  std::max(1, ceil_div(V / (dtype == ICAP_DTYPE_F32 ? 4 : 8), NT * kGradPieces))};
  const long long blocks = (long long)N * a.shares;
  if (blocks > kMostRows)
    return fail(ICAP_ERR_UNSUPPORTED, "token_log_probs_grad: %d rows of %d are too many for one call", N, V);
  const bool streamed = stream_writes(row_bytes(dtype, N, V));
#define LAUNCH_S(D, S)                                                                          \
  hipLaunchKernelGGL((token_log_probs_grad_kernel<D, S>), row_grid((int)blocks), dim3(NT), 0,  \
                     (hipStream_t)stream, a)
#define LAUNCH(D) do { if (streamed) LAUNCH_S(D, true); else LAUNCH_S(D, false); } while (0)
  ICAP_BY_DTYPE(dtype, LAUNCH);
#undef LAUNCH
#undef LAUNCH_S
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
  const RowShape shape = row_shape(dtype, N, V);
  const bool streamed = dlogits && stream_writes(row_bytes(dtype, N, V));
#define LAUNCH_S(D, W, NV, S)                                                                         \
  hipLaunchKernelGGL((distill_loss_kernel<D, W, NV, S>), row_grid(N), dim3(W * 64), 0, (hipStream_t)stream, a)
#define LAUNCH(D, W, NV) do { if (streamed) LAUNCH_S(D, W, NV, true); else LAUNCH_S(D, W, NV, false); } while (0)
  ICAP_BY_ROWS(dtype, shape, LAUNCH);
#undef LAUNCH
#undef LAUNCH_S
  ICAP_LAUNCH_CHECK("distill_loss_kernel");
  return ICAP_OK;
}

}  // extern "C"
