// raf.op.embedding and raf.op.embedding_dx: rows of a table by token, and the table's gradient.
#include <algorithm>

#include "model_io.cuh"

namespace rafb200 {

// ---- lookup -----------------------------------------------------------------------
//   out[n, :] = scale * x[id_n, :], a row of zeros where id_n is outside [0, rows)
// Bound: HBM, the rows read and the rows written.  A warp takes kLookupRows rows and has four accesses of 32 lanes in
// flight, at 32 to 48 registers a thread.  65536 rows of 1024 (bf16, 20000 different ones): 29.5 us, 5.7 TB/s of what has to
// be read and written, where a copy of as many bytes takes 5.5 TB/s.  Rows of 1023: 40 us; from fp32 into bf16, 20011 rows of
// 1023 20.4 us (3.2 TB/s).
constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 2;

template <typename T, typename O, int VEC, int COUNT>
__device__ __forceinline__ void lookup_groups(const T* from, O* to, int64_t left, float scale) {
  typename Group<T, VEC>::W w[COUNT];
  // without a condition, or the loads would wait for one another: behind the row's end its last group again
#pragma unroll
  for (int u = 0; u < COUNT; ++u)
    w[u] = *reinterpret_cast<const typename Group<T, VEC>::W*>(from + min((int64_t)u * 32 * VEC, left));
#pragma unroll
  for (int u = 0; u < COUNT; ++u) {
    Group<O, VEC> o;
    Group<T, VEC>::unpack(w[u], o.x);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.x[j] *= scale;
    if (u * 32 * VEC <= left) o.store(to + u * 32 * VEC);
  }
}

// Rows that begin anywhere: kPiece elements at a time, written to aligned addresses out of the aligned 16-byte groups that
// hold them, the first 4 Q + 0 or 2 bytes behind a boundary (Q < 0: at one).
template <typename T, typename O>
constexpr int kPiece = sizeof(T) == 4 && sizeof(O) == 4 ? 4 : 8;

template <typename T, typename O, int Q>
__device__ __forceinline__ void lookup_pieces(const T* from, O* to, int pieces, float scale, int lane) {
  constexpr int kPer = 16 / sizeof(T), kParts = kPiece<T, O> / kPer, kUnroll = 4 / kParts;
  const char* source = reinterpret_cast<const char*>(from);
  const uint32_t bits = (reinterpret_cast<uintptr_t>(source) & 3) * 8;
  for (int i = lane; i < pieces; i += 32 * kUnroll) {
    uint4 w[kUnroll][kParts];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int q = 0; q < kParts; ++q)
        w[u][q] = load_shifted<Q>(source + ((int64_t)min(i + u * 32, pieces - 1) * kParts + q) * 16, bits);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      Group<O, kPiece<T, O>> o;
#pragma unroll
      for (int q = 0; q < kParts; ++q) Group<T, kPer>::unpack(w[u][q], o.x + q * kPer);
#pragma unroll
      for (int j = 0; j < kPiece<T, O>; ++j) o.x[j] *= scale;
      if (i + u * 32 < pieces) o.store(to + (int64_t)(i + u * 32) * kPiece<T, O>);
    }
  }
}
// A row by one warp; 24 elements at least.
template <typename T, typename O>
__device__ __forceinline__ void lookup_anywhere(const T* from, O* to, int width, float scale, int lane) {
  int at = (int)((-(intptr_t)to & 15) / sizeof(O)), pieces = (width - at) / kPiece<T, O>;
  const uint32_t shift = reinterpret_cast<uintptr_t>(from + at) & 15;
  if (shift) {  // the first and the last piece element by element: the groups that hold the others lie inside the row
    at += kPiece<T, O>;
    pieces -= 2;
    switch (shift >> 2) {
      case 0: lookup_pieces<T, O, 0>(from + at, to + at, pieces, scale, lane); break;
      case 1: lookup_pieces<T, O, 1>(from + at, to + at, pieces, scale, lane); break;
      case 2: lookup_pieces<T, O, 2>(from + at, to + at, pieces, scale, lane); break;
      default: lookup_pieces<T, O, 3>(from + at, to + at, pieces, scale, lane); break;
    }
  } else {
    lookup_pieces<T, O, -1>(from + at, to + at, pieces, scale, lane);
  }
  const int j = lane < at ? lane : lane + pieces * kPiece<T, O>;  // 30 elements at most
  if (j < width) to[j] = Elem<O>::from_f32(Elem<T>::to_f32(from[j]) * scale);
}

template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kLookupThreads)
    embedding_kernel(const T* x, Ids ids, int64_t n, int64_t rows, int64_t width, float scale, O* out) {
  constexpr int kUnroll = VEC == 1 ? 8 : 4;
  grid_dependency_trigger();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t first = ((int64_t)blockIdx.x * (kLookupThreads / 32) + (threadIdx.x >> 5)) * kLookupRows;
  int64_t id[kLookupRows];
#pragma unroll
  for (int r = 0; r < kLookupRows; ++r) id[r] = first + r < n ? ids[first + r] : -1;
#pragma unroll
  for (int r = 0; r < kLookupRows; ++r) {
    if (first + r >= n) return;
    O* to = out + (first + r) * width;
    if ((uint64_t)id[r] < (uint64_t)rows) {
      const T* from = x + id[r] * width;
      if constexpr (VEC < 16 / (int)sizeof(T)) {
        if (width >= 256 && width < ((int64_t)1 << 31)) {  // shorter rows leave lanes without a piece
          lookup_anywhere<T, O>(from, to, (int)width, scale, lane);
          continue;
        }
      }
      for (int64_t c = (int64_t)lane * VEC; c < width; c += 32 * VEC * kUnroll)
        lookup_groups<T, O, VEC, kUnroll>(from + c, to + c, width - VEC - c, scale);
    } else {
      Group<O, VEC> zero{};
      for (int64_t c = (int64_t)lane * VEC; c < width; c += 32 * VEC) zero.store(to + c);
    }
  }
}

// ---- gradient ---------------------------------------------------------------------
//   dx[r, :] (+)= scale * sum over the n with id_n = r of dy[n, :]
// Two launches, every sum in an order that the tokens alone fix:
//   1. the tokens are sorted, stably, while other blocks write the zeros of rows without a token;
//   2. a warp walks `run` sorted tokens for 32 * VEC columns and keeps the sum of the present row in registers.  A row whose
//      tokens all lie there is written there; a row cut by the border between two warps of a block is put together in shared
//      memory, one cut by the border of a block (a chunk of tokens) leaves partial sums, which the last of its blocks to
//      come adds up, chunk after chunk.
struct SortArgs {
  Ids ids;
  int64_t n;
  int64_t rows;        // valid ids are [0, rows); every other id sorts as `rows`, behind them
  int64_t padding;
  uint2* a;            // (id, position) pairs: the last pass leaves them in a
  uint2* b;
  int passes, bits;    // digits and bits of each
  unsigned char* fill; // bytes to zero
  int64_t fill_bytes;
  uint32_t* counters;  // to be zeroed too: of the blocks that have left their part of a row
  int n_counters;
  __device__ __forceinline__ uint32_t key(int64_t id) const {
    return (uint64_t)id < (uint64_t)rows && id != padding ? (uint32_t)id : (uint32_t)rows;
  }
};

__device__ void zero_bytes(unsigned char* p, int64_t bytes, int64_t worker, int64_t workers) {
  const int64_t head = min((int64_t)(-(intptr_t)p & 15), bytes);
  const int64_t vecs = (bytes - head) >> 4, tail = head + (vecs << 4);
  uint4* q = reinterpret_cast<uint4*>(p + head);
  for (int64_t i = worker; i < vecs; i += workers) q[i] = make_uint4(0, 0, 0, 0);
  if (worker < head) p[worker] = 0;
  if (worker < bytes - tail) p[tail + worker] = 0;
}

// Few tokens: each warp finds the rank of its tokens by comparing them with all, which need no more than one block's shared
// memory.  No block waits for another.  The launch alone, without zeros to write: 1024 tokens take 3.4 us where the cluster's passes
// take 11.7 us, 2048 4.7 and 12.2 us, 4096 10.9 and 12.4 us.  Whole calls with a result to zero (30522 rows of 1024, bf16), ranked and
// sorted: 1000 tokens 20.1 and 22.3 us, 2048 21.7 and 23.2 us, 3000 24.6 and 23.6 us, 4096 28.5 and 24.6 us one behind the other;
// with cold caches, from 512 tokens on, 18.5 and 22.5, 20.5 and 26.6 (1000), 22.5 and 26.6 (2048), 26.6 and 26.6 (3000), 28.7 and 28.7 us: the
// border.
constexpr int kRankTokens = 4096;
constexpr int kRankThreads = 256;
constexpr int kRankLoads = 8;
__global__ void __launch_bounds__(kRankThreads) embedding_rank_kernel(SortArgs a) {
  __shared__ uint32_t keys[kRankTokens];
  grid_dependency_trigger();
  grid_dependency_wait();
  const int n = (int)a.n, tid = threadIdx.x, lane = tid & 31, warps = gridDim.x * (kRankThreads / 32);
  const int mine = blockIdx.x * (kRankThreads / 32) + (tid >> 5);
  if (blockIdx.x == gridDim.x - 1)
    for (int i = tid; i < a.n_counters; i += kRankThreads) a.counters[i] = 0;
  if (blockIdx.x * (kRankThreads / 32) < n) {
    for (int i0 = tid; i0 < n; i0 += kRankThreads * kRankLoads) {
      int64_t id[kRankLoads];  // all of them asked for before the first is looked at
#pragma unroll
      for (int u = 0; u < kRankLoads; ++u) id[u] = a.ids[min(i0 + u * kRankThreads, n - 1)];
#pragma unroll
      for (int u = 0; u < kRankLoads; ++u)
        if (i0 + u * kRankThreads < n) keys[i0 + u * kRankThreads] = a.key(id[u]);
    }
    __syncthreads();
    for (int i = mine; i < n; i += warps) {
      const uint32_t key = keys[i];
      int rank = 0;
#pragma unroll 4
      for (int j = lane; j < n; j += 32) rank += keys[j] < key + (j < i);  // key is below 2^32 - 1
      rank = __reduce_add_sync(0xffffffffu, rank);
      if (lane == 0) a.a[rank] = make_uint2(key, (uint32_t)i);
    }
  }
  zero_bytes(a.fill, a.fill_bytes, (int64_t)blockIdx.x * kRankThreads + tid, (int64_t)gridDim.x * kRankThreads);
}

// Many tokens: digits from the lowest up, by one cluster of 16 blocks.  Each of its 512 warps owns a contiguous range of the pairs:
// it counts its digits, equal ones of a group of 32 ranked by lane; the counts are summed over warps, blocks (through
// distributed shared memory) and digits, and the warp then moves its pairs in order.
// Bound: the latency of a pass's two cluster barriers and of its loads and stores, and the counting, which 16 SMs share: 16384
// tokens take 13 us, 65536 22 us; eight blocks took 37 us for these.
constexpr int kSortBlocks = 16;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;  // pairs of a lane in registers
constexpr int kDigitBits = 9;  // two passes for tables of up to 2^18 - 1 rows; the counters of 32 warps take 64 KB
constexpr int kDigits = 1 << kDigitBits;
constexpr int kFillClusters = 15;
constexpr size_t kSortSmem = sizeof(uint32_t) * (kSortWarps * kDigits + (kSortBlocks + 2) * kDigits + 32);

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(SortArgs a) {
  extern __shared__ uint32_t counts[];  // [warp][digit]
  uint32_t* totals = counts + kSortWarps * kDigits;  // [block][digit]
  uint32_t* halves = totals + kSortBlocks * kDigits;  // [half of the warps][digit]
  uint32_t* scan = halves + 2 * kDigits;
  grid_dependency_trigger();
  grid_dependency_wait();
  if (blockIdx.x >= kSortBlocks) {
    zero_bytes(a.fill, a.fill_bytes, (int64_t)(blockIdx.x - kSortBlocks) * kSortThreads + threadIdx.x,
               (int64_t)(gridDim.x - kSortBlocks) * kSortThreads);
    return;
  }
  cluster_arrive_relaxed();  // all blocks of the cluster run before one stores into another's shared memory
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cluster_rank(), n = (uint32_t)a.n;
  const uint32_t each = ((n + kSortBlocks * kSortWarps - 1) / (kSortBlocks * kSortWarps) + 31) & ~31u;
  const uint32_t from = (uint32_t)min((uint64_t)(rank * kSortWarps + warp) * each, (uint64_t)n), to = min(n - from, each) + from;
  for (int i = rank * kSortThreads + tid; i < a.n_counters; i += kSortBlocks * kSortThreads) a.counters[i] = 0;
  uint32_t* mine = counts + warp * kDigits;
  const uint32_t digits = 1u << a.bits, lower_lanes = (1u << lane) - 1u;
  const bool kept = each <= 32 * kSortItems;  // a warp's pairs stay in registers from counting to moving
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    // the passes end in a
    const uint2* src = ((a.passes - pass) & 1) ? a.b : a.a;
    uint2* dst = ((a.passes - pass) & 1) ? a.a : a.b;
    uint2 pair[kSortItems];
    uint32_t place[kSortItems];  // the digit, and the rank among the warp's pairs of this digit << kDigitBits
    auto load = [&](uint32_t i0) {  // of every 32 pairs from i0 on this lane's; all loads before the first is looked at
      const uint32_t last = to - 1;
      if (pass) {
#pragma unroll
        for (int u = 0; u < kSortItems; ++u) pair[u] = __ldcg(src + min(i0 + u * 32 + lane, last));
      } else {
        int64_t id[kSortItems];
#pragma unroll
        for (int u = 0; u < kSortItems; ++u) id[u] = a.ids[min(i0 + u * 32 + lane, last)];
#pragma unroll
        for (int u = 0; u < kSortItems; ++u) pair[u] = make_uint2(a.key(id[u]), i0 + u * 32 + lane);
      }
    };
    // The lanes whose digit is this lane's, from one vote for each bit: 30 instructions, where __match_any_sync took 150 cycles
    // of a warp's time with 32 different digits.  Lanes without a pair have a digit of their own.
    auto equals = [&](uint32_t d) {
      uint32_t same = 0xffffffffu;
#pragma unroll
      for (int b = 0; b <= kDigitBits; ++b) {
        if (b > a.bits) break;
        const uint32_t vote = __ballot_sync(0xffffffffu, d >> b & 1);
        same &= d >> b & 1 ? vote : ~vote;
      }
      return same;
    };
    auto count = [&](uint32_t i0) {  // ranks below 2^23: a warp's range, 2^31 / 512 pairs at most
      uint32_t same[kSortItems];
#pragma unroll
      for (int u = 0; u < kSortItems; ++u) {
        if (i0 + u * 32 >= to) break;
        place[u] = i0 + u * 32 + lane < to ? (pair[u].x >> shift) & (digits - 1) : digits;
        same[u] = equals(place[u]);
      }
#pragma unroll
      for (int u = 0; u < kSortItems; ++u) {
        if (i0 + u * 32 >= to) break;
        const uint32_t d = place[u], below = __popc(same[u] & lower_lanes);
        uint32_t old = 0;
        if (d < digits) old = mine[d];
        __syncwarp();
        if (d < digits && below == 0) mine[d] = old + __popc(same[u]);
        __syncwarp();
        place[u] = d | (old + below) << kDigitBits;
      }
    };
    auto move = [&](uint32_t i0) {  // to the ranks, and to where the warp's pairs of a digit begin
#pragma unroll
      for (int u = 0; u < kSortItems; ++u)
        if (i0 + u * 32 + lane < to) __stcg(dst + mine[place[u] & (kDigits - 1)] + (place[u] >> kDigitBits), pair[u]);
    };
    if (from < to) load(from);
    for (uint32_t d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    for (uint32_t i0 = from; i0 < to; i0 += 32 * kSortItems) {
      if (i0 != from) load(i0);
      count(i0);
    }
    __syncthreads();
    if (pass == 0) cluster_wait();
    // two threads a digit, each for half of the warps
    const uint32_t digit = tid & (kDigits - 1), half = tid / kDigits;
    uint32_t* column = counts + half * (kSortWarps / 2) * kDigits + digit;
    uint32_t sum = 0, c[kSortWarps / 2];
    if (digit < digits) {
#pragma unroll
      for (int w = 0; w < kSortWarps / 2; ++w) c[w] = column[w * kDigits];
#pragma unroll
      for (int w = 0; w < kSortWarps / 2; ++w) sum += c[w];
      halves[half * kDigits + digit] = sum;
    }
    __syncthreads();
    if (digit < digits) {
      const uint32_t all = halves[digit] + halves[kDigits + digit];
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks / 2; ++r) cluster_store(totals + rank * kDigits + digit, half * (kSortBlocks / 2) + r, all);
    }
    cluster_sync();
    uint32_t before = 0, all = 0;  // of this thread's digit: in the blocks before this one, in all of them
    if (digit < digits) {
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks; ++r) {
        const uint32_t t = totals[r * kDigits + digit];
        if (r < rank) before += t;
        all += t;
      }
    }
    uint32_t incl = all;  // exclusive sums over the digits
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    if (digit < digits) {
      uint32_t at = incl - all + before + (half ? halves[digit] : 0);
#pragma unroll
      for (uint32_t w = 0; w < kDigits / 32; ++w)
        if (w < warp % (kDigits / 32)) at += scan[w];
#pragma unroll
      for (int w = 0; w < kSortWarps / 2; ++w) {
        column[w * kDigits] = at;
        at += c[w];
      }
    }
    __syncthreads();
    if (kept) {
      move(from);
    } else {
      for (uint32_t i0 = from; i0 < to; i0 += 32 * kSortItems) {
        load(i0);
#pragma unroll
        for (int u = 0; u < kSortItems; ++u) {
          if (i0 + u * 32 >= to) break;
          const bool in = i0 + u * 32 + lane < to;
          const uint32_t d = in ? (pair[u].x >> shift) & (digits - 1) : digits, same = equals(d);
          const uint32_t below = __popc(same & lower_lanes);
          uint32_t old = 0;
          if (in) old = mine[d];
          __syncwarp();
          if (in && below == 0) mine[d] = old + __popc(same);
          __syncwarp();
          if (in) __stcg(dst + old + below, pair[u]);
        }
      }
    }
    // the pairs are written for all, and no block stores totals before all have read theirs
    if (pass + 1 < a.passes) cluster_sync();
  }
}

struct SumArgs {
  const void* dy;
  const uint2* sorted;
  int64_t n, rows, width;
  float scale;
  int accumulate;
  void* dx;
  float* partial;        // [chunk][2][stride]: sums of a row that began before the chunk, or goes on behind it
  int64_t stride;
  uint32_t* counters;    // [chunk in which the row begins][tile]
  int run;               // tokens of a warp
  uint32_t tiles;        // column tiles of 32 * VEC
};

constexpr int kSumWarps = 8;  // of a chunk
constexpr int kSumThreads = 32 * kSumWarps;
constexpr int kSumBatch = 4;                  // rows asked for together
constexpr int kSumAhead = 3;                  // batches on their way
constexpr int kSumRing = kSumBatch * kSumAhead;
constexpr int kMostRun = 128;                 // tokens of a warp, at most

// Copies BYTES (16, 8 or 4) of one lane to shared memory, asynchronously.
template <int BYTES>
__device__ __forceinline__ void copy_lane(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}
// The 4 bytes at `from`, as far as they lie in [begin, end), both multiples of 2.
__device__ __forceinline__ void copy_word(uint32_t* to, const char* from, const char* begin, const char* end) {
  if (from >= begin && from + 4 <= end) {
    copy_lane<4>(to, from);
  } else {  // the array's first or last element, half of a word
    if (from >= begin && from < end) reinterpret_cast<unsigned short*>(to)[0] = *reinterpret_cast<const unsigned short*>(from);
    if (from + 2 >= begin && from + 2 < end) reinterpret_cast<unsigned short*>(to)[1] = *reinterpret_cast<const unsigned short*>(from + 2);
  }
}

// VEC running sums, two an instruction.
template <int VEC>
struct Sums {
  Two s[VEC / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) s[j] = Two(0.f, 0.f);
  }
  template <typename Get>
  __device__ __forceinline__ void add(const Get& get) {
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) s[j] = s[j] + Two(get(2 * j), get(2 * j + 1));
  }
  __device__ __forceinline__ float at(int j) const { return j & 1 ? s[j / 2].hi() : s[j / 2].lo(); }
};
template <>
struct Sums<1> {
  float s;
  __device__ __forceinline__ void clear() { s = 0.f; }
  template <typename Get>
  __device__ __forceinline__ void add(const Get& get) {
    s += get(0);
  }
  __device__ __forceinline__ float at(int) const { return s; }
};

template <typename W, int VEC, bool ANY>
struct SumShared {
  W ring[kSumWarps][kSumRing][ANY ? 33 : 32];
  float parts[kSumWarps][32 * VEC];  // the warp's part of a row that began before it
  uint2 tokens[kSumWarps][kMostRun + 1];
  int through[kSumWarps];            // that row takes all of the warp's tokens and goes on behind it
  struct {
    int64_t begins, ends;            // chunks [begins, ends) have left their parts of the row, this one as the last; or 0, 0
    uint32_t row;
  } joins[2];                        // of the row that began before the chunk, and of the one that goes on behind it
};

// Bound: HBM, the gathered rows of dy.  Rows come through shared memory by asynchronous copies, kSumRing of them on their
// way for a lane, which alone reads what it has asked for; what accumulated rows hold already is asked for together for those
// that end in a batch.  The sums of cut rows, in a launch of their own, took 2 to 5 us more.  65536 tokens of 1024 (bf16), from
// the end of the sort on: into two rows 34 us with cold caches (3.9 TB/s), 28 us among calls that leave a part of dy in the L2 (4.8 TB/s);
// 54 us added to 20000 rows of fp32 (5.5 TB/s of dy and of the rows read and written).  Rows of 1023, two columns a lane: 127 us for
// the whole call, where rows of 1024 take 59 us into 30522 rows of bf16.
// ANY: 16-bit rows that begin at any element (VEC 2).  A lane's two elements are its word of the row's aligned ones, or, where
// the row begins in the middle of one, that word's second half and the next word's first.
template <typename T, typename O, int VEC, bool ANY>
__global__ void __launch_bounds__(kSumThreads, 3) embedding_sum_kernel(SumArgs a) {
  using W = typename Group<T, VEC>::W;
  constexpr int OUT = ANY ? 1 : VEC, ROW = ANY ? 33 : 32;  // elements of an access to dx; words of a row's place
  extern __shared__ uint4 shared[];
  auto& [ring, parts, tokens, through, joins] = *reinterpret_cast<SumShared<W, VEC, ANY>*>(shared);
  grid_dependency_trigger();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunk = blockIdx.x / a.tiles, col = (int64_t)((blockIdx.x - (uint32_t)chunk * a.tiles) * 32 + lane) * VEC;
  const int64_t from = (chunk * kSumWarps + warp) * a.run, to = min(from + a.run, a.n);
  const bool here = col < a.width;  // lanes behind the last column see to the tokens alone
  const uint32_t rows = (uint32_t)a.rows;
  const T* dy = static_cast<const T*>(a.dy) + (here || ANY ? col : 0);
  const char *begin = static_cast<const char*>(a.dy), *end = begin + a.n * a.width * (int64_t)sizeof(T);
  O* dx = static_cast<O*>(a.dx) + col;
  uint32_t row = rows, before = rows, behind = rows, first = rows;
  Sums<VEC> sum;
  sum.clear();
  auto keep = [&] {
#pragma unroll
    for (int j = 0; j < VEC; ++j) parts[warp][j * 32 + lane] = sum.at(j);
  };
  struct Held {
    Group<O, OUT> g[VEC / OUT];
  };
  auto look = [&](Held& old, uint32_t r) {
#pragma unroll
    for (int q = 0; q < VEC / OUT; ++q) old.g[q].load(dx + (int64_t)r * a.width + (col + q * OUT < a.width ? q * OUT : 0));
  };
  auto put = [&](const Held& old) {
#pragma unroll
    for (int q = 0; q < VEC / OUT; ++q) {
      if (col + q * OUT >= a.width) continue;
      Group<O, OUT> o;
#pragma unroll
      for (int j = 0; j < OUT; ++j) o.x[j] = a.accumulate ? fmaf(sum.at(q * OUT + j), a.scale, old.g[q].x[j]) : sum.at(q * OUT + j) * a.scale;
      o.store(dx + (int64_t)row * a.width + q * OUT);
    }
  };
  auto put_late = [&] {  // where what the row holds has not been asked for
    Held old{};
    if (a.accumulate && here) look(old, row);
    put(old);
  };
  if (from < a.n) {
    if (from) before = a.sorted[from - 1].x;
    if (to < a.n) behind = a.sorted[to].x;
    int count = 0;  // tokens that count: those that do not are behind all others
    for (int i0 = 0; i0 < a.run; i0 += 32) {
      const uint2 t = from + i0 + lane < to ? a.sorted[from + i0 + lane] : make_uint2(rows, 0);
      if (i0 + lane < a.run) tokens[warp][i0 + lane] = t;
      count += __popc(__ballot_sync(0xffffffffu, t.x < rows));
    }
    if (lane == 0) tokens[warp][a.run] = make_uint2(behind, 0);
    __syncwarp();
    first = tokens[warp][0].x;
    auto ask = [&](int i, W* at) {
#pragma unroll
      for (int u = 0; u < kSumBatch; ++u) {
        if (i + u >= count) break;
        const T* p = dy + (int64_t)tokens[warp][i + u].y * a.width;
        if constexpr (ANY) {
          const char* word = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(3));
          if (col <= a.width) copy_word(at + u * ROW, word, begin, end);
          if (lane == 31 && col + 1 < a.width) copy_word(at + u * ROW + 1, word + 4, begin, end);
        } else {
          copy_lane<sizeof(W)>(at + u * ROW, p);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    W* place = &ring[warp][0][lane];
#pragma unroll
    for (int b = 0; b < kSumAhead; ++b) ask(b * kSumBatch, place + b * kSumBatch * ROW);
    for (int i = 0; i < count; i += kSumBatch) {
      uint32_t r[kSumBatch + 1];
      Held old[kSumBatch];
#pragma unroll
      for (int u = 0; u <= kSumBatch; ++u) r[u] = i + u <= count ? tokens[warp][i + u].x : rows;
      if (a.accumulate && here) {  // what the rows that end in this batch hold, all of it asked for together
#pragma unroll
        for (int u = 0; u < kSumBatch; ++u) look(old[u], min(r[u], rows - 1));
      }
      asm volatile("cp.async.wait_group %0;" ::"n"(kSumAhead - 1) : "memory");
#pragma unroll
      for (int u = 0; u < kSumBatch; ++u) {
        if (i + u >= count) break;
        row = r[u];
        float x[VEC];
        W w = place[u * ROW];
        if constexpr (ANY) {
          const uint32_t own = w, next = __shfl_down_sync(0xffffffffu, own, 1);
          if (reinterpret_cast<uintptr_t>(dy + (int64_t)tokens[warp][i + u].y * a.width) & 2)
            w = __funnelshift_r(own, lane == 31 ? place[u * ROW + 1] : next, 16);
        }
        Group<T, VEC>::unpack(w, x);
        sum.add([&](int j) { return x[j]; });
        if (r[u + 1] != row) {  // the row ends here
          if (row == before) keep();
          else put(old[u]);
          sum.clear();
        }
      }
      ask(i + kSumRing, place);
      place = place == &ring[warp][kSumRing - kSumBatch][lane] ? &ring[warp][0][lane] : place + kSumBatch * ROW;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (row < rows && row == behind && row == before) keep();  // the whole of it between the two borders
  }
  if (threadIdx.x < 2) joins[threadIdx.x].ends = 0;
  if (lane == 0) through[warp] = row < rows && row == before && row == behind && row == first;
  const bool starts = row < rows && row != before && row == behind;  // a row goes on behind this warp
  const bool enters = warp == 0 && first < rows && first == before;  // a row began before this chunk
  __syncthreads();
  auto follow = [&](int w) {  // adds the parts of warps w, w + 1, ... as far as the row goes on; whether it leaves the chunk
    for (; w < kSumWarps; ++w) {
      sum.add([&](int j) { return parts[w][j * 32 + lane]; });
      if (!through[w]) return false;
    }
    return true;
  };
  auto put_partial = [&](int slot) {
    if (!here) return;
    Group<float, VEC> g;
#pragma unroll
    for (int j = 0; j < VEC; ++j) g.x[j] = sum.at(j);
    g.store(a.partial + (chunk * 2 + slot) * a.stride + col);
  };
  // This warp has left the chunk's part of `row`: is it the last to do so?
  const int64_t length = (int64_t)kSumWarps * a.run;
  auto left = [&](int which, int64_t begins, bool leaves) {
    for (bool go = begins < chunk; go;) {  // the chunk in which the row begins: it goes on before that chunk's first token otherwise
      const int64_t c = begins - lane;
      const uint32_t on = __ballot_sync(0xffffffffu, c > 0 && a.sorted[c * length - 1].x == row);
      go = on == 0xffffffffu;
      begins -= go ? 32 : __ffs(~on) - 1;
    }
    int64_t ends = chunk + 1;  // the first chunk that does not begin with the row
    for (bool go = leaves; go;) {
      const int64_t c = ends + lane;
      const uint32_t on = __ballot_sync(0xffffffffu, c * length < a.n && a.sorted[c * length].x == row);
      go = on == 0xffffffffu;
      ends += go ? 32 : __ffs(~on) - 1;
    }
    __threadfence();
    __syncwarp();
    if (lane == 0 && atomicAdd(a.counters + begins * a.tiles + (blockIdx.x - (uint32_t)chunk * a.tiles), 1u) + 1 == (uint32_t)(ends - begins)) {
      joins[which].begins = begins;
      joins[which].ends = ends;
      joins[which].row = row;
    }
  };
  if (starts) {
    if (follow(warp + 1)) {
      put_partial(1);
      left(1, chunk, true);
    } else {
      put_late();
    }
  }
  if (enters) {  // warp 0 may see to this row and to another one that begins with it
    row = first;
    sum.clear();
    const bool leaves = follow(0);
    put_partial(0);
    left(0, chunk - 1, leaves);
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {  // each warp takes every eighth part; their sums in the order of the warps
    const int64_t begins = joins[which].begins, ends = joins[which].ends;
    if (!ends) continue;
    __threadfence();
    sum.clear();
    if (here) {
      constexpr int kParts = 4;
      const float* part = a.partial + col;
      for (int64_t c0 = begins + warp; c0 < ends; c0 += kParts * kSumWarps) {
        Group<float, VEC> g[kParts];
#pragma unroll
        for (int u = 0; u < kParts; ++u) {  // all of them asked for before the first is looked at
          const int64_t c = min(c0 + u * kSumWarps, ends - 1);
          g[u].load_coherent(part + (c * 2 + (c == begins)) * a.stride);
        }
#pragma unroll
        for (int u = 0; u < kParts; ++u)
          if (c0 + u * kSumWarps < ends) sum.add([&](int j) { return g[u].x[j]; });
      }
    }
    keep();
    __syncthreads();
    if (warp == 0) {
      row = joins[which].row;
      sum.clear();
      for (int w = 0; w < kSumWarps; ++w) sum.add([&](int j) { return parts[w][j * 32 + lane]; });
      put_late();
    }
    __syncthreads();
  }
}

// Elements of an access that every row of both arrays allows: 16 bytes of the first array's, 2, or 1.
static int group_width(const void* p, int size_p, const void* q, int size_q, int64_t width) {
  auto fits = [&](int vec) {
    return width % vec == 0 && reinterpret_cast<uintptr_t>(p) % std::min(vec * size_p, 16) == 0 &&
           reinterpret_cast<uintptr_t>(q) % std::min(vec * size_q, 16) == 0;
  };
  return fits(16 / size_p) ? 16 / size_p : fits(2) ? 2 : 1;
}

template <typename T, typename F>
static int with_width(int vec, const F& f) {
  switch (vec) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 16 / (int)sizeof(T)>{});
  }
}

static bool range_overflows(int64_t a, int64_t b) {
  int64_t r;
  return __builtin_mul_overflow(a, b, &r) || r > ((int64_t)1 << 60);
}

// Tokens of a warp: as many as give every SM its three blocks once.  Many of them cut fewer rows.
static int warp_tokens(int64_t n, int64_t width) {
  const int64_t tiles = (width + 255) / 256, warps = 148 * 3 * kSumWarps;
  const int64_t want = (n * tiles + warps * kSumBatch - 1) / (warps * kSumBatch) * kSumBatch;
  return (int)std::min<int64_t>(std::max<int64_t>(want, 2 * kSumBatch), kMostRun);
}

static size_t round_up(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace rafb200

using namespace rafb200;

extern "C" {

int rafb200_embedding(const void* x, int x_dtype, int64_t rows, int64_t width, const void* indices, int index_dtype,
                      int64_t n, float scale, void* out, int out_dtype, void* stream) {
  RAFB200_REQUIRE(dtype_valid(x_dtype) && dtype_valid(out_dtype), "rafb200_embedding: bad dtype");
  RAFB200_REQUIRE(index_dtype_valid(index_dtype), "rafb200_embedding: indices are int32 or int64");
  RAFB200_REQUIRE(rows >= 0 && width >= 0 && n >= 0 && !range_overflows(rows, width) && !range_overflows(n, width),
                  "rafb200_embedding: bad sizes");
  if (n == 0 || width == 0) return RAFB200_OK;
  RAFB200_REQUIRE(indices && out && (x || rows == 0), "rafb200_embedding: NULL argument");
  const int vec = group_width(x, dtype_size(x_dtype), out, dtype_size(out_dtype), width);
  const int64_t per_block = kLookupThreads / 32 * kLookupRows, grid = (n + per_block - 1) / per_block;
  RAFB200_REQUIRE(grid < ((int64_t)1 << 31), "rafb200_embedding: too many indices");
  const Ids ids{indices, index_dtype == RAFB200_I64};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_type(x_dtype, [&](auto t) {
    return with_type(out_dtype, [&](auto o) {
      return with_width<decltype(t)>(vec, [&](auto w) {
        using T = decltype(t);
        using O = decltype(o);
        RAFB200_CUDA(launch_dependent(embedding_kernel<T, O, decltype(w)::value>, dim3((unsigned)grid), kLookupThreads, 0, s,
                                      static_cast<const T*>(x), ids, n, rows, width, scale, static_cast<O*>(out)));
        return (int)RAFB200_OK;
      });
    });
  });
}

// The workspace holds the pairs twice, then the partial sums of the chunks and their counters.
size_t rafb200_embedding_dx_workspace_bytes(int64_t n, int64_t width) {
  if (n <= 0 || width <= 0 || n >= ((int64_t)1 << 31) || range_overflows(n, width)) return 0;
  const int64_t tokens = (int64_t)kSumWarps * warp_tokens(n, width), chunks = (n + tokens - 1) / tokens;
  return 2 * round_up((size_t)n * sizeof(uint2)) + round_up((size_t)chunks * 2 * ((width + 7) & ~int64_t(7)) * sizeof(float)) +
         (size_t)chunks * ((width + 31) / 32) * sizeof(uint32_t);  // a tile has 32 columns at least
}

int rafb200_embedding_dx(const void* dy, int dy_dtype, const void* indices, int index_dtype, int64_t n, int64_t rows,
                         int64_t width, float scale, int64_t padding_idx, int accumulate, void* dx, int dx_dtype,
                         void* workspace, size_t workspace_bytes, void* stream) {
  RAFB200_REQUIRE(dtype_valid(dy_dtype) && dtype_valid(dx_dtype), "rafb200_embedding_dx: bad dtype");
  RAFB200_REQUIRE(index_dtype_valid(index_dtype), "rafb200_embedding_dx: indices are int32 or int64");
  RAFB200_REQUIRE(rows >= 0 && width >= 0 && n >= 0 && !range_overflows(rows, width) && !range_overflows(n, width),
                  "rafb200_embedding_dx: bad sizes");
  RAFB200_REQUIRE(n < ((int64_t)1 << 31) && rows < ((int64_t)1 << 31), "rafb200_embedding_dx: 2^31 indices or rows and more");
  if (rows == 0 || width == 0 || (n == 0 && accumulate)) return RAFB200_OK;
  RAFB200_REQUIRE(dx && (n == 0 || (dy && indices)), "rafb200_embedding_dx: NULL argument");
  RAFB200_REQUIRE(n == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                             workspace_bytes >= rafb200_embedding_dx_workspace_bytes(n, width)),
                  "rafb200_embedding_dx: workspace smaller than rafb200_embedding_dx_workspace_bytes, or not aligned");
  cudaStream_t s = static_cast<cudaStream_t>(stream);

  const int vec = group_width(dy, dtype_size(dy_dtype), dx, dtype_size(dx_dtype), width);
  const int lane_width = vec == 1 ? 4 / dtype_size(dy_dtype) : vec;  // 16-bit rows at odd addresses: words, shifted
  const int64_t tiles = (width + 32 * lane_width - 1) / (32 * lane_width);
  SortArgs so{};
  so.ids = Ids{indices, index_dtype == RAFB200_I64};
  so.n = n;
  so.rows = rows;
  so.padding = padding_idx;
  so.a = static_cast<uint2*>(workspace);
  so.b = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + round_up((size_t)n * sizeof(uint2)));
  const int run = n ? warp_tokens(n, width) : 1;
  const int64_t tokens = (int64_t)kSumWarps * run, chunks = (n + tokens - 1) / tokens, grid = chunks * tiles;
  const int64_t stride = (width + 7) & ~int64_t(7);
  float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * round_up((size_t)n * sizeof(uint2)));
  RAFB200_REQUIRE(grid < ((int64_t)1 << 31), "rafb200_embedding_dx: rows too wide");
  so.counters = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(partial) + round_up((size_t)chunks * 2 * stride * sizeof(float)));
  so.n_counters = (int)grid;
  int bits = 1;
  while (rows >> bits) ++bits;
  so.passes = (bits + kDigitBits - 1) / kDigitBits;
  so.bits = (bits + so.passes - 1) / so.passes;
  if (!accumulate) {
    so.fill = static_cast<unsigned char*>(dx);
    so.fill_bytes = rows * width * dtype_size(dx_dtype);
  }
  if (n <= kRankTokens) {
    const int64_t ranks = (n + kRankThreads / 32 - 1) / (kRankThreads / 32), fills = so.fill_bytes / (kRankThreads * 64);
    const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>({ranks, fills, 1}), 148 * 4);
    RAFB200_CUDA(launch_dependent(embedding_rank_kernel, dim3(grid), kRankThreads, 0, s, so));
  } else {
    const int64_t each = (int64_t)kSortBlocks * kSortThreads * 64;  // four stores a thread
    const unsigned clusters = 1 + (unsigned)std::min<int64_t>((so.fill_bytes + each - 1) / each, kFillClusters);
    if (const int rc = allow_smem<embedding_sort_kernel>(kSortSmem, kSortSmem)) return rc;
    if (const int rc = allow_large_cluster<embedding_sort_kernel>()) return rc;
    RAFB200_CUDA(launch_cluster(embedding_sort_kernel, kSortBlocks, clusters * kSortBlocks, kSortThreads, kSortSmem, s, so));
  }
  if (n == 0) return RAFB200_OK;

  SumArgs a{};
  a.dy = dy;
  a.sorted = so.a;
  a.n = n;
  a.rows = rows;
  a.width = width;
  a.scale = scale;
  a.accumulate = accumulate;
  a.dx = dx;
  a.partial = partial;
  a.stride = stride;
  a.counters = so.counters;
  a.tiles = (uint32_t)tiles;
  a.run = run;
  return with_type(dx_dtype, [&](auto o) {
    using O = decltype(o);
    return with_type(dy_dtype, [&](auto t) {
      return with_width<decltype(t)>(vec, [&](auto w) {
        using T = decltype(t);
        constexpr bool kAny = sizeof(T) == 2 && decltype(w)::value == 1;
        constexpr int kVec = kAny ? 2 : decltype(w)::value;
        constexpr size_t smem = sizeof(SumShared<typename Group<T, kVec>::W, kVec, kAny>);
        if (const int rc = allow_smem<embedding_sum_kernel<T, O, kVec, kAny>>(smem, smem)) return rc;
        RAFB200_CUDA(launch_dependent(embedding_sum_kernel<T, O, kVec, kAny>, dim3((unsigned)grid), kSumThreads, smem, s, a));
        return (int)RAFB200_OK;
      });
    });
  });
}

}  // extern "C"
