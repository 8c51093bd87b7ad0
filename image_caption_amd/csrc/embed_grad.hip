// Scaled embedding lookup and its gradient by sorted tokens.
#include <algorithm>

#include "vocab_row.h"

namespace icap {
namespace {

// Rows of D elements as pieces of kVec (n = kVec), or one by one where D is shorter (n = 1).  The
// last piece of a row ends at its end: where D is no multiple of kVec it takes some columns a
// second time and writes the same values to them.
__device__ __forceinline__ int piece_col(int c, int n, int D) { return min(c, D - n); }

// One group of lanes per token, kLookupAhead tokens at a time.  Bound by the writes: 131072 rows of 512
// in bf16 take 28 us (4.8 TB/s written; the table stays in the caches).
constexpr int kLookupAhead = 4;

template <int DTYPE, int n, bool STREAM>
__global__ __launch_bounds__(256) void embedding_scaled_kernel(const void* table, const int32_t* ids,
                                                               void* out, int N, int V, int D, float scale,
                                                               int pad, int lanes) {
  typedef Piece<DTYPE, n> P;
  const int groups = 256 / lanes, lane = threadIdx.x & (lanes - 1);
  const int n0 = (blockIdx.x * groups + threadIdx.x / lanes) * kLookupAhead;
  if (n0 >= N) return;
  int id[kLookupAhead];
#pragma unroll
  for (int j = 0; j < kLookupAhead; ++j) {
    id[j] = ids[min(n0 + j, N - 1)];
    if ((unsigned)id[j] >= (unsigned)V || id[j] == pad) id[j] = -1;
  }
  for (int c0 = lane * n; c0 < D; c0 += lanes * n) {
    const int c = piece_col(c0, n, D);
    P x[kLookupAhead];
#pragma unroll
    for (int j = 0; j < kLookupAhead; ++j)
      x[j].load((const typename P::type*)table + (size_t)max(id[j], 0) * D + c);
#pragma unroll
    for (int j = 0; j < kLookupAhead; ++j) {
      if (n0 + j >= N) break;
      float v[n];
      x[j].unpack(v);
#pragma unroll
      for (int e = 0; e < n; ++e) v[e] = id[j] < 0 ? 0.f : v[e] * scale;
      P::template store<STREAM>((typename P::type*)out + (size_t)(n0 + j) * D + c, v);
    }
  }
}

// ---- gradient: tokens sorted by id, then one sum per row of the table -----------------------

constexpr int kSortWaves = 16;
constexpr int kSortRows = 512;      // table rows of one sorting workgroup at most
constexpr int kSortAhead = 4;       // 16-byte loads in flight for each lane
constexpr int kSortList = 512;      // tokens that a wave notes in LDS

// Place of table row v in the sorted order: row v belongs to workgroup v mod 2^bits, so that the
// frequent words of a vocabulary (ids falling with frequency) spread over all workgroups instead
// of meeting in the first.  Slots of a workgroup lie side by side; 2^bits * rows of them in all.
struct Slots {
  int bits, rows;
  __host__ __device__ int of(int v) const { return (v & ((1 << bits) - 1)) * rows + (v >> bits); }
  __host__ __device__ int row(int slot) const { return ((slot % rows) << bits) + slot / rows; }
  __host__ __device__ int count() const { return rows << bits; }
};

struct SortArgs {
  const int32_t* ids;
  int N, V, pad;
  Slots slots;
  int32_t* row_start;
  int2* sorted;               // (position, token)
  int32_t* long_count;
  int2* split;                // embed_split_kernel's lists and where each workgroup's tokens begin in them
  int32_t* split_start;
  int split_lists;
};

__device__ __forceinline__ bool takes_part(int id, int V, int pad) {
  return (unsigned)id < (unsigned)V && id != pad;
}

// The lanes whose key has the same low bits, among those that take part.
__device__ __forceinline__ unsigned long long same_key(int key, int bits, bool part) {
  unsigned long long same = __ballot(part);
  for (int i = 0; i < bits; ++i) {
    const unsigned long long one = __ballot((key >> i) & 1);
    same &= (key >> i) & 1 ? one : ~one;
  }
  return same;
}

constexpr int kSplitTokens = 2048;      // of a list
constexpr int kSplitLists = 1024;

// Lists of kSplitTokens tokens in a row, each ordered by the workgroup of embed_sort_kernel that
// will take a token, positions ascending: that kernel then reads its own tokens only.
__global__ __launch_bounds__(kSortWaves * 64) void embed_split_kernel(SortArgs p) {
  __shared__ int s_cnt[kSortWaves][256];
  __shared__ int s_wave[4];
  constexpr int kSteps = kSplitTokens / (kSortWaves * 64);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned long long lower = (1ull << lane) - 1;
  for (int i = tid; i < kSortWaves * 256; i += kSortWaves * 64) (&s_cnt[0][0])[i] = 0;
  __syncthreads();
  const int from = blockIdx.x * kSplitTokens + wave * 64 * kSteps + lane;
  int id[kSteps], at[kSteps];
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    id[j] = p.ids[min(from + j * 64, p.N - 1)];
    if (from + j * 64 >= p.N || !takes_part(id[j], p.V, p.pad)) id[j] = -1;
  }
#pragma unroll
  for (int j = 0; j < kSteps; ++j) {
    const unsigned long long same = same_key(id[j], 8, id[j] >= 0);
    const int leader = __ffsll(same) - 1;
    int begin = 0;
    if (id[j] >= 0 && lane == leader) begin = atomicAdd(&s_cnt[wave][id[j] & 255], __popcll(same));
    at[j] = __shfl(begin, max(leader, 0), 64) + __popcll(same & lower);
  }
  __syncthreads();
  int total = 0, upto = 0;
  if (tid < 256) {
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = s_cnt[w][tid];
      s_cnt[w][tid] = total;
      total += c;
    }
    upto = total;      // inclusive scan over the 256 keys
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    if (lane == 63) s_wave[wave] = upto;
  }
  __syncthreads();
  if (tid < 256) {
    for (int w = 0; w < wave; ++w) upto += s_wave[w];
    const int begin = upto - total;
    for (int w = 0; w < kSortWaves; ++w) s_cnt[w][tid] += begin;
    p.split_start[blockIdx.x * 257 + tid] = begin;
    if (tid == 255) p.split_start[blockIdx.x * 257 + 256] = upto;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSteps; ++j)
    if (id[j] >= 0)
      p.split[(size_t)blockIdx.x * kSplitTokens + s_cnt[wave][id[j] & 255] + at[j]] = make_int2(from + j * 64, id[j]);
}

// Workgroup b goes through the tokens - 16 waves, a share of the positions each - and counts how many
// belong to earlier workgroups and, per wave and row, how many to this one; its own tokens it
// notes in LDS, in order.  Then it writes them behind those counts, in ascending order of their
// positions within a row.  A wave whose own tokens overflow its list (one word filling the
// batch) reads its share again instead.  Every count is an integer and every place follows from
// the counts, so nothing depends on timing, and no workgroup waits for another.
// SPLIT: its tokens come from the lists of embed_split_kernel.  Otherwise it reads all of them, 256 x N
// in all from the caches (2^bits x N for tables of more than 131072 rows), which for few tokens is
// less than a launch: 10240 take 8 us, 131071 took 34 us and take 18 by way of the lists, 6 of them
// the lists.
template <bool SPLIT>
__global__ __launch_bounds__(kSortWaves * 64) void embed_sort_kernel(SortArgs p) {
  __shared__ int s_cnt[kSortWaves][kSortRows];
  __shared__ int2 s_list[kSortWaves][kSortList];
  __shared__ int s_wave[kSortWaves];
  __shared__ int s_upto[SPLIT ? kSortWaves : 1][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x, mask = (1 << p.slots.bits) - 1, rows = p.slots.rows;
  for (int i = tid; i < kSortWaves * rows; i += kSortWaves * 64) s_cnt[i / rows][i % rows] = 0;
  if (b == 0 && tid == 0) *p.long_count = 0;
  __syncthreads();
  const unsigned long long lower = (1ull << lane) - 1;
  int below = 0, noted = 0;
  // all tokens: this wave's positions are [from, to)
  const int per = ((p.N + kSortWaves - 1) / kSortWaves + 255) / 256 * 256;
  const int from = min(p.N, wave * per), to = min(p.N, from + per);
  // lists: this wave's are [first, first + mine), lane i knows the i-th one's part for b
  const int lists = (p.split_lists + kSortWaves - 1) / kSortWaves;
  const int first = wave * lists;
  int part_begin = 0;
  auto from_lists = [&](int t) {      // the wave's t-th token
    int l = 0;                        // the first list that reaches past t
    for (int step = 32; step > 0; step >>= 1)
      if (s_upto[wave][l + step - 1] <= t) l += step;
    const int before = l ? s_upto[wave][l - 1] : 0;
    const int begin = __shfl(part_begin, l, 64);
    return p.split[(size_t)(first + l) * kSplitTokens + begin + t - before];
  };
  if constexpr (SPLIT) {
    const bool there = lane < lists && first + lane < p.split_lists;
    int size = 0;
    if (there) {
      const int32_t* at = p.split_start + (size_t)(first + lane) * 257 + b;
      part_begin = at[0];
      size = at[1] - part_begin;
      below = part_begin;
    }
    int upto = size;
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(upto, d, 64);
      if (lane >= d) upto += o;
    }
    s_upto[wave][lane] = upto;
    noted = __shfl(upto, 63, 64);
    __syncthreads();
    for (int t0 = 0; t0 < noted; t0 += 64) {
      const int2 x = from_lists(min(t0 + lane, noted - 1));
      if (t0 + lane < noted) {
        atomicAdd(&s_cnt[wave][x.y >> p.slots.bits], 1);
        if (t0 + lane < kSortList) s_list[wave][t0 + lane] = x;
      }
    }
  } else {
    // tokens i0 + lane * 4 + 0 .. 3
    auto read = [&](int i0, int (&id)[4]) {
      const int i = i0 + lane * 4;
      if (i0 + 256 <= to) {
        typedef int int4_any __attribute__((ext_vector_type(4), aligned(4)));
        const int4_any x = *reinterpret_cast<const int4_any*>(p.ids + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) id[e] = x[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) id[e] = i + e < to ? p.ids[min(i + e, p.N - 1)] : -1;
      }
    };
    auto count = [&](int i0, const int (&id)[4]) {
      unsigned long long m[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool ok = takes_part(id[e], p.V, p.pad);
        below += ok && (id[e] & mask) < b;
        m[e] = __ballot(ok && (id[e] & mask) == b);
      }
      if (!(m[0] | m[1] | m[2] | m[3])) return;
      int at = noted;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        at += __popcll(m[e] & lower);
        noted += __popcll(m[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((m[e] >> lane) & 1) {
          atomicAdd(&s_cnt[wave][id[e] >> p.slots.bits], 1);
          if (at < kSortList) s_list[wave][at] = make_int2(i0 + lane * 4 + e, id[e]);
          ++at;
        }
    };
    for (int i0 = from; i0 < to; i0 += 256 * kSortAhead) {
      int id[kSortAhead][4];
#pragma unroll
      for (int j = 0; j < kSortAhead; ++j) read(i0 + j * 256, id[j]);
#pragma unroll
      for (int j = 0; j < kSortAhead; ++j) count(i0 + j * 256, id[j]);
    }
  }
  for (int d = 32; d > 0; d >>= 1) below += __shfl_xor(below, d, 64);
  if (lane == 0) s_wave[wave] = below;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < kSortWaves; ++w) base += s_wave[w];
  __syncthreads();
  int total = 0;
  if (tid < rows)
    for (int w = 0; w < kSortWaves; ++w) total += s_cnt[w][tid];
  int upto = total;       // inclusive scan over the rows
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d, 64);
    if (lane >= d) upto += o;
  }
  if (lane == 63) s_wave[wave] = upto;
  __syncthreads();
  for (int w = 0; w < wave; ++w) base += s_wave[w];
  if (tid < rows) {
    int at = base + upto - total;
    p.row_start[b * rows + tid] = at;
    if (b == mask && tid == rows - 1) p.row_start[p.slots.count()] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = s_cnt[w][tid];
      s_cnt[w][tid] = at;
      at += c;
    }
  }
  __syncthreads();
  // 64 tokens of one wave, in the order of the lanes
  const int row_bits = 32 - __builtin_clz(rows);
  auto place = [&](int2 t, bool part) {
    const int r = t.y >> p.slots.bits;
    const unsigned long long same = same_key(r, row_bits, part);
    const int leader = __ffsll(same) - 1;
    int at = 0;
    if (part && lane == leader) at = atomicAdd(&s_cnt[wave][r], __popcll(same));
    at = __shfl(at, max(leader, 0), 64);
    if (part) p.sorted[at + __popcll(same & lower)] = t;
  };
  if (noted <= kSortList) {
    for (int k = 0; k < noted; k += 64) place(s_list[wave][min(k + lane, noted - 1)], k + lane < noted);
  } else if constexpr (SPLIT) {
    for (int k = 0; k < noted; k += 64) place(from_lists(min(k + lane, noted - 1)), k + lane < noted);
  } else {
    for (int i = from; i < to; i += 64) {
      const int id = p.ids[min(i + lane, to - 1)];
      place(make_int2(i + lane, id), i + lane < to && takes_part(id, p.V, p.pad) && (id & mask) == b);
    }
  }
}

// The sums.  The sorted list is cut into chunks of equal length, one group of lanes for each chunk
// and block of columns (kVec of them a lane): the rows of `grad` are read in batches of kSumAhead
// whatever row of the table they belong to, so that frequent and rare words cost the same.  A row
// of up to `chunk` tokens is summed where it starts, past the chunk's end if need be.  A longer one
// (of 131072 tokens over 50000 words the most frequent word has 4000) is summed in shares, one in
// `part` for each chunk it reaches (slot 0: the row of the chunk's first token, slot 1: the row of
// its last one, if another); the chunk where it starts puts it on the list of long rows, and
// embed_join_kernel adds its shares up in the chunks' order.  Rows without tokens get their zeros
// from further waves, kZeroSlots of them each.  131071 rows of 512 in bf16 into 50000 take 39 us (4.5
// TB/s): rows of 1 kB in the order of the words, and the latency of where a chunk begins.
struct SumArgs {
  const void* grad;
  void* dtable;
  const int32_t* row_start;
  const int2* sorted;
  int32_t *long_count, *long_rows;
  float* part;
  Slots slots;
  int V, D, chunk, chunks;
  int lanes, col_blocks;      // lanes of a group (a power of two up to 64), groups side by side over D
  float scale;
};

constexpr int kSumAhead = 8;
constexpr int kZeroSlots = 16;       // rows that a wave looks over for ones without tokens

template <int DTYPE, int n, bool STREAM>
__global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs p) {
  typedef Piece<DTYPE, n> P;
  const int groups = 256 / p.lanes;
  const int lane = threadIdx.x & (p.lanes - 1);
  const int sums = p.chunks * p.col_blocks, sum_blocks = (sums + groups - 1) / groups;
  typename P::type* table = (typename P::type*)p.dtable;
  if ((int)blockIdx.x >= sum_blocks) {
    const int slot0 = (((int)blockIdx.x - sum_blocks) * 4 + (threadIdx.x >> 6)) * kZeroSlots;
    const int slot = slot0 + (threadIdx.x & 63);
    const bool empty = slot < p.slots.count() && p.row_start[slot] == p.row_start[slot + 1];
    const unsigned long long mask = __ballot(empty);
    const float zero[n] = {};
    for (int r = (threadIdx.x & 63) / p.lanes; r < kZeroSlots; r += 64 / p.lanes) {
      const int v = p.slots.row(slot0 + r);
      if (!((mask >> r) & 1) || v >= p.V) continue;
      for (int c = lane * n; c < p.D; c += p.lanes * n)
        P::store(table + (size_t)v * p.D + piece_col(c, n, p.D), zero);
    }
    return;
  }
  const int group = blockIdx.x * groups + threadIdx.x / p.lanes;
  if (group >= sums) return;
  const int unit = group / p.col_blocks, block = group % p.col_blocks;
  const int c0 = (block * p.lanes + lane) * n, c = piece_col(c0, n, p.D);
  const int total = p.row_start[p.slots.count()];
  const int lo = unit * p.chunk, hi = min(total, lo + p.chunk);
  if (lo >= hi || c0 >= p.D) return;
  const int first = p.sorted[lo].y, last = p.sorted[hi - 1].y;
  const int sa = p.slots.of(first), sb = p.slots.of(last);
  const int a0 = p.row_start[sa], a1 = p.row_start[sa + 1];
  const int b0 = p.row_start[sb], b1 = p.row_start[sb + 1];
  const bool long_a = a1 - a0 > p.chunk, long_b = b1 - b0 > p.chunk;
  // a short row that began in the chunk before was summed there; a short last one is ours to its end
  const int from = a0 < lo && !long_a ? a1 : lo, to = long_b ? hi : b1;
  if (from >= hi) return;
  if (block == 0 && lane == 0 && long_b && b0 >= lo) p.long_rows[atomicAdd(p.long_count, 1)] = last;
  float* part = p.part + (size_t)unit * 2 * p.D + c;
  const typename P::type* grad = (const typename P::type*)p.grad + c;
  float acc[n] = {};
  int2 at[kSumAhead];
#pragma unroll
  for (int j = 0; j < kSumAhead; ++j) at[j] = p.sorted[min(from + j, to - 1)];
  int row = at[0].y;
  auto flush = [&]() {
    if ((long_a && row == first) || (long_b && row == last)) {
      float* dst = part + (row == first ? 0 : p.D);
#pragma unroll
      for (int e = 0; e < n; ++e) dst[e] = acc[e];
    } else {
#pragma unroll
      for (int e = 0; e < n; ++e) acc[e] *= p.scale;
      P::store(table + (size_t)row * p.D + c, acc);
    }
#pragma unroll
    for (int e = 0; e < n; ++e) acc[e] = 0.f;
  };
  for (int i = from; i < to; i += kSumAhead) {
    P x[kSumAhead];
    int tok[kSumAhead];
#pragma unroll
    for (int j = 0; j < kSumAhead; ++j) {
      x[j].template load<STREAM>(grad + (size_t)at[j].x * p.D);
      tok[j] = at[j].y;
    }
#pragma unroll
    for (int j = 0; j < kSumAhead; ++j) at[j] = p.sorted[min(i + kSumAhead + j, to - 1)];
#pragma unroll
    for (int j = 0; j < kSumAhead; ++j) {
      if (i + j >= to) break;
      if (tok[j] != row) {
        flush();
        row = tok[j];
      }
      float v[n];
      x[j].unpack(v);
#pragma unroll
      for (int e = 0; e < n; ++e) acc[e] += v[e];
    }
  }
  flush();
}

constexpr int kJoinWaves = 4;

// The long rows, one workgroup each in turn; its waves take the shares in turn, 64 columns at a
// time.  The order of the list depends on timing, the sum of a row does not.  6 us for 131071 tokens,
// most of it a launch and one pass of the most frequent word's shares.
template <int DTYPE>
__global__ __launch_bounds__(kJoinWaves * 64) void embed_join_kernel(SumArgs p) {
  typedef Elem<DTYPE> E;
  __shared__ float s_acc[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int blocks = (p.D + 63) / 64, todo = *p.long_count * blocks;
  for (int i = blockIdx.x; i < todo; i += gridDim.x) {
    const int v = p.long_rows[i / blocks], c = i % blocks * 64 + lane;
    const int from = p.row_start[p.slots.of(v)], to = p.row_start[p.slots.of(v) + 1];
    const int begin = from / p.chunk, end = (to - 1) / p.chunk;        // chunks with a share
    float acc = 0.f;
    if (c < p.D) {
      if (wave == 0) acc = p.part[((size_t)begin * 2 + (from > begin * p.chunk ? 1 : 0)) * p.D + c];
      int k = begin + 1 + wave;
      for (; k + 7 * kJoinWaves <= end; k += 8 * kJoinWaves) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = p.part[(size_t)(k + j * kJoinWaves) * 2 * p.D + c];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc += x[j];
      }
      for (; k <= end; k += kJoinWaves) acc += p.part[(size_t)k * 2 * p.D + c];
    }
    __syncthreads();
    s_acc[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < p.D) {
      for (int w = 1; w < kJoinWaves; ++w) acc += s_acc[w][lane];
      ((typename E::type*)p.dtable)[(size_t)v * p.D + c] = E::down(acc * p.scale);
    }
  }
}

// Tokens of a chunk: 4096 chunks fill the card with 16 waves a compute unit; below 16 tokens a wave's
// fixed costs (where its chunk begins and ends) outweigh its sums.
int chunk_of(int N) { return std::max(16, ceil_div(N, 4096)); }

Slots slots_of(int V) {
  Slots s{8, 0};          // 256 workgroups, one for each compute unit, and more for large tables
  while (((long long)kSortRows << s.bits) < V) ++s.bits;
  s.rows = (int)(((long long)V + (1LL << s.bits) - 1) >> s.bits);
  return s;
}

struct Workspace {
  size_t row_start, sorted, long_rows, part, split, split_start, bytes;
};

// Whether the tokens go through lists: from where reading all of them 256 times costs more than a
// launch, as long as the lists' part for a workgroup fits the lanes that look it up (2097152 tokens)
// and the lists' 256 keys are the sorting workgroups (131072 rows of the table).  Past either every
// workgroup reads all tokens: 131071 tokens x 512 in bf16 take 89 us with 131072 rows and 168 with
// 131073, rows of 8 into 50000 take 0.68 ms for 2097152 tokens and 2.4 ms for one more.
bool splits(int N, int V) {
  return N > 24576 && ceil_div(N, kSplitTokens) <= kSplitLists && slots_of(V).bits == 8;
}

Workspace workspace_of(int N, int V, int D) {
  const size_t chunks = (size_t)ceil_div(N, chunk_of(N));
  auto pad16 = [](size_t n) { return (n + 15) / 16 * 16; };
  Workspace w;
  w.row_start = 0;
  w.sorted = w.row_start + pad16(((size_t)slots_of(V).count() + 1) * sizeof(int32_t));
  w.long_rows = w.sorted + pad16((size_t)N * sizeof(int2));
  w.part = w.long_rows + pad16((chunks + 1) * sizeof(int32_t));      // their number, then the rows
  w.split = w.part + pad16(chunks * 2 * (size_t)D * sizeof(float));
  w.split_start = w.split + (splits(N, V) ? (size_t)ceil_div(N, kSplitTokens) * kSplitTokens * sizeof(int2) : 0);
  w.bytes = w.split_start + (splits(N, V) ? (size_t)ceil_div(N, kSplitTokens) * 257 * sizeof(int32_t) : 0);
  return w;
}

constexpr int kMost = 1 << 25;      // a launch counts at most 2^32 lanes, 64 for each token or table row

int check(const char* what, int dtype, int N, int V, int D) {
  ICAP_REQUIRE(dtype == ICAP_DTYPE_F32 || dtype == ICAP_DTYPE_BF16 || dtype == ICAP_DTYPE_F16,
               "%s: unknown dtype %d", what, dtype);
  ICAP_REQUIRE(N >= 0 && V > 0 && D > 0, "%s: bad shape", what);
  if (N > kMost || V > kMost || D > kMost)
    return fail(ICAP_ERR_UNSUPPORTED, "%s: N, V and D go up to %d", what, kMost);
  return ICAP_OK;
}

// Elements of a piece, and lanes side by side on a row (a power of two up to a wave).
int vec_of(int dtype, int D) {
  const int vec = dtype == ICAP_DTYPE_F32 ? 4 : 8;
  return D < vec ? 1 : vec;
}
int lanes_of(int D, int vec) {
  int lanes = 1;
  while (lanes < 64 && lanes * vec < D) lanes *= 2;
  return lanes;
}

#define ICAP_BY_TYPE_AND_VEC(dtype, vec, call)                          \
  do {                                                                  \
    if ((dtype) == ICAP_DTYPE_F32) {                                    \
      if ((vec) == 1) call(ICAP_DTYPE_F32, 1); else call(ICAP_DTYPE_F32, 4);   \
    } else if ((dtype) == ICAP_DTYPE_BF16) {                            \
      if ((vec) == 1) call(ICAP_DTYPE_BF16, 1); else call(ICAP_DTYPE_BF16, 8); \
    } else {                                                            \
      if ((vec) == 1) call(ICAP_DTYPE_F16, 1); else call(ICAP_DTYPE_F16, 8);   \
    }                                                                   \
  } while (0)

}  // namespace
}  // namespace icap

using namespace icap;

extern "C" {

int icap_embedding_scaled(const void* table, int dtype, const int32_t* ids, void* out, int N, int V,
                          int D, float scale, int pad_token, icap_stream_t stream) {
  ICAP_REQUIRE(table && ids && out, "embedding_scaled: null pointer");
  if (int rc = check("embedding_scaled", dtype, N, V, D)) return rc;
  if (N == 0) return ICAP_OK;
  const int vec = vec_of(dtype, D), lanes = lanes_of(D, vec);
  const dim3 grid(ceil_div(ceil_div(N, kLookupAhead), 256 / lanes));
  const bool streamed = stream_writes((size_t)N * D * (dtype == ICAP_DTYPE_F32 ? 4 : 2));
#define LAUNCH_S(T, n, S)                                                                             \
  hipLaunchKernelGGL((embedding_scaled_kernel<T, n, S>), grid, dim3(256), 0, (hipStream_t)stream, table, \
                     ids, out, N, V, D, scale, pad_token, lanes)
#define LAUNCH(T, n) do { if (streamed) LAUNCH_S(T, n, true); else LAUNCH_S(T, n, false); } while (0)
  ICAP_BY_TYPE_AND_VEC(dtype, vec, LAUNCH);
#undef LAUNCH
#undef LAUNCH_S
  ICAP_LAUNCH_CHECK("embedding_scaled_kernel");
  return ICAP_OK;
}

size_t icap_embedding_grad_workspace_bytes(int N, int V, int D) {
  if (N < 0 || V <= 0 || D <= 0) return 0;
  return workspace_of(N, V, D).bytes;
}

int icap_embedding_grad(const void* grad, int dtype, const int32_t* ids, void* dtable, int N, int V,
                        int D, float scale, int pad_token, void* workspace, size_t workspace_bytes,
                        icap_stream_t stream) {
  ICAP_REQUIRE(grad && ids && dtable && workspace, "embedding_grad: null pointer");
  if (int rc = check("embedding_grad", dtype, N, V, D)) return rc;
  const Workspace w = workspace_of(N, V, D);
  ICAP_REQUIRE(aligned16(workspace) && workspace_bytes >= w.bytes,
               "embedding_grad: workspace too small or not aligned");
  char* ws = (char*)workspace;
  int32_t* row_start = (int32_t*)(ws + w.row_start);
  int2* sorted = (int2*)(ws + w.sorted);
  int32_t* long_count = (int32_t*)(ws + w.long_rows);
  hipStream_t s = (hipStream_t)stream;
  const Slots slots = slots_of(V);
  const bool split = splits(N, V);
  SortArgs sort{ids, N, V, pad_token, slots, row_start, sorted, long_count, (int2*)(ws + w.split),
                (int32_t*)(ws + w.split_start), split ? ceil_div(N, kSplitTokens) : 0};
  const dim3 sort_grid(1u << slots.bits), sort_block(kSortWaves * 64);
  if (split) {
    hipLaunchKernelGGL(embed_split_kernel, dim3(sort.split_lists), sort_block, 0, s, sort);
    ICAP_LAUNCH_CHECK("embed_split_kernel");
    hipLaunchKernelGGL(embed_sort_kernel<true>, sort_grid, sort_block, 0, s, sort);
  } else {
    hipLaunchKernelGGL(embed_sort_kernel<false>, sort_grid, sort_block, 0, s, sort);
  }
  ICAP_LAUNCH_CHECK("embed_sort_kernel");
  const int vec = vec_of(dtype, D), lanes = lanes_of(D, vec);
  const int chunk = chunk_of(N), chunks = ceil_div(N, chunk);
  SumArgs a{grad, dtable, row_start, sorted, long_count, long_count + 1, (float*)(ws + w.part),
            slots, V, D, chunk, chunks, lanes, ceil_div(D, lanes * vec), scale};
  const int groups = 256 / lanes;
  const dim3 grid((unsigned)(((long long)chunks * a.col_blocks + groups - 1) / groups +
                             ceil_div(slots.count(), 4 * kZeroSlots)));
  const dim3 join((unsigned)std::max(1LL, std::min(2048LL, (long long)chunks * ceil_div(D, 64))));
  // (a gradient is read for the last time here: past 96 MB it leaves the caches to others, 40 -> 36 us
  // for 131071 tokens)
  const bool streamed = stream_writes((size_t)N * D * (dtype == ICAP_DTYPE_F32 ? 4 : 2));
#define LAUNCH(T, n)                                                                   \
  do {                                                                                 \
    if (streamed) hipLaunchKernelGGL((embed_sum_kernel<T, n, true>), grid, dim3(256), 0, s, a);  \
    else hipLaunchKernelGGL((embed_sum_kernel<T, n, false>), grid, dim3(256), 0, s, a);          \
    hipLaunchKernelGGL(embed_join_kernel<T>, join, dim3(kJoinWaves * 64), 0, s, a);    \
  } while (0)
  ICAP_BY_TYPE_AND_VEC(dtype, vec, LAUNCH);
#undef LAUNCH
  ICAP_LAUNCH_CHECK("embed_sum_kernel");
  return ICAP_OK;
}

}  // extern "C"
