// raf.op.embedding and raf.op.embedding_dx: rows of a table by token, and the table's gradient.
#include <algorithm>

#include "model_io.cuh"

namespace rafb200 {

// ---- lookup -----------------------------------------------------------------------
//   out[n, :] = scale * x[id_n, :], a row of zeros where id_n is outside [0, rows)
// Bound: HBM, the rows read and the rows written.  2^tpr_log threads share a row, so that no element needs a division,
// and a thread has kLookupRows rows in flight: the load of a row waits for that of its id.
constexpr int kLookupThreads = 256;
constexpr int kLookupRows = 4;

template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kLookupThreads)
    embedding_kernel(const T* x, Ids ids, int64_t n, int64_t rows, int64_t width, float scale, O* out,
                     int tpr_log) {
  grid_dependency_trigger();
  grid_dependency_wait();
  const int tpr = 1 << tpr_log, per = kLookupThreads >> tpr_log;
  const int64_t row0 = (int64_t)blockIdx.x * per * kLookupRows + (threadIdx.x >> tpr_log);
  int64_t id[kLookupRows];
#pragma unroll
  for (int u = 0; u < kLookupRows; ++u) {
    const int64_t row = row0 + u * per;
    id[u] = row < n ? ids[row] : -1;
  }
  for (int64_t c = (int64_t)(threadIdx.x & (tpr - 1)) * VEC; c < width; c += (int64_t)tpr * VEC) {
    Group<T, VEC> g[kLookupRows];
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      if ((uint64_t)id[u] < (uint64_t)rows) {
        g[u].load(x + id[u] * width + c);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) g[u].x[j] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < kLookupRows; ++u) {
      const int64_t row = row0 + u * per;
      if (row < n) {
        Group<O, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.x[j] = g[u].x[j] * scale;
        o.store(out + row * width + c);
      }
    }
  }
}

// ---- gradient ---------------------------------------------------------------------
//   dx[r, :] (+)= scale * sum over the n with id_n = r of dy[n, :]
// Three launches, every sum in an order that the tokens alone fix:
//   1. the tokens are sorted, stably, while other blocks write the zeros of rows without a token;
//   2. a warp walks `run` sorted tokens for 32 * VEC columns and keeps the sum of the present row in registers.  A row whose
//      tokens all lie there is written there; a row cut by the border between two warps of a block is put together in shared
//      memory, one cut by the border of a block (a chunk of tokens) leaves partial sums;
//   3. the rows that were cut by chunks are joined, chunk after chunk.
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
// memory.  No block waits for another.
constexpr int kRankTokens = 4096;
constexpr int kRankThreads = 256;
__global__ void __launch_bounds__(kRankThreads) embedding_rank_kernel(SortArgs a) {
  __shared__ uint32_t keys[kRankTokens];
  grid_dependency_trigger();
  grid_dependency_wait();
  const int n = (int)a.n, tid = threadIdx.x, lane = tid & 31, warps = gridDim.x * (kRankThreads / 32);
  const int mine = blockIdx.x * (kRankThreads / 32) + (tid >> 5);
  if (blockIdx.x * (kRankThreads / 32) < n) {
    for (int i = tid; i < n; i += kRankThreads) keys[i] = a.key(a.ids[i]);
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

// Many tokens: digits from the lowest up, by one cluster.  Each of its 256 warps owns a contiguous range of the pairs: it counts
// its digits, the counts are summed over warps, blocks (through distributed shared memory) and digits, and
// the warp then moves its pairs in order, equal digits of a group of 32 ranked by lane.
// 65536 tokens take XXX us, 16384 take XXX us.
constexpr int kSortBlocks = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortItems = 8;  // pairs of a lane in registers
constexpr int kDigitBits = 9;  // two passes for tables of up to 2^18 - 1 rows; the counters of 32 warps take 64 KB
constexpr int kDigits = 1 << kDigitBits;
constexpr int kFillClusters = 17;  // with the sorting one 144 blocks of 148 SMs
constexpr size_t kSortSmem = sizeof(uint32_t) * (kSortWarps * kDigits + kSortBlocks * kDigits + kDigits + 32);

__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(SortArgs a) {
  extern __shared__ uint32_t counts[];  // [warp][digit]
  uint32_t* totals = counts + kSortWarps * kDigits;  // [block][digit]
  uint32_t* base = totals + kSortBlocks * kDigits;
  uint32_t* scan = base + kDigits;
  grid_dependency_trigger();
  grid_dependency_wait();
  if (blockIdx.x >= kSortBlocks) {
    zero_bytes(a.fill, a.fill_bytes, (int64_t)(blockIdx.x - kSortBlocks) * kSortThreads + threadIdx.x,
               (int64_t)(gridDim.x - kSortBlocks) * kSortThreads);
    return;
  }
  cluster_arrive();  // all blocks of the cluster run before one stores into another's shared memory
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  const int64_t each = ((a.n + kSortBlocks * kSortWarps - 1) / (kSortBlocks * kSortWarps) + 31) & ~int64_t(31);
  const int64_t from = min(((int64_t)rank * kSortWarps + warp) * each, a.n), to = min(from + each, a.n);
  uint32_t* mine = counts + warp * kDigits;
  const int digits = 1 << a.bits;
  const bool kept = each <= 32 * kSortItems;  // a warp's pairs stay in registers from counting to moving
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    // the passes end in a
    const uint2* src = ((a.passes - pass) & 1) ? a.b : a.a;
    uint2* dst = ((a.passes - pass) & 1) ? a.a : a.b;
    uint2 pair[kSortItems];
    auto load = [&](int64_t i0) {  // of every 32 pairs from i0 on this lane's
#pragma unroll
      for (int u = 0; u < kSortItems; ++u) {
        const int64_t i = i0 + u * 32 + lane;
        if (i < to) pair[u] = pass ? __ldcg(src + i) : make_uint2(a.key(a.ids[i]), (uint32_t)i);
      }
    };
    auto digit = [&](int64_t i0, int u) { return i0 + u * 32 + lane < to ? (pair[u].x >> shift) & (digits - 1) : digits; };
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    for (int64_t i0 = from; i0 < to; i0 += 32 * kSortItems) {
      load(i0);
#pragma unroll
      for (int u = 0; u < kSortItems; ++u) {
        if (i0 + u * 32 >= to) break;
        const uint32_t d = digit(i0, u), same = __match_any_sync(0xffffffffu, d);
        if (d < digits && lane == __ffs(same) - 1) mine[d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    if (pass == 0) cluster_wait();
    if (tid < digits) {
      uint32_t c[kSortWarps], sum = 0;
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) c[w] = counts[w * kDigits + tid];
#pragma unroll
      for (int w = 0; w < kSortWarps; ++w) {
        counts[w * kDigits + tid] = sum;
        sum += c[w];
      }
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks; ++r) cluster_store(totals + rank * kDigits + tid, r, sum);
    }
    cluster_sync();
    uint32_t before = 0, all = 0;  // of this thread's digit: in the blocks before this one, in all of them
    if (tid < digits) {
#pragma unroll
      for (uint32_t r = 0; r < kSortBlocks; ++r) {
        const uint32_t c = totals[r * kDigits + tid];
        if (r < rank) before += c;
        all += c;
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
    if (tid < digits) {
      uint32_t lower = incl - all;
#pragma unroll
      for (int w = 0; w < kDigits / 32; ++w)
        if (w < warp) lower += scan[w];
      base[tid] = lower + before;
    }
    __syncthreads();
    for (int64_t i0 = from; i0 < to; i0 += 32 * kSortItems) {
      if (!kept) load(i0);
#pragma unroll
      for (int u = 0; u < kSortItems; ++u) {
        if (i0 + u * 32 >= to) break;
        const uint32_t d = digit(i0, u), same = __match_any_sync(0xffffffffu, d);
        uint32_t old = 0;
        if (d < digits) old = mine[d];
        __syncwarp();
        if (d < digits && lane == __ffs(same) - 1) mine[d] = old + __popc(same);
        __syncwarp();
        if (d < digits) __stcg(dst + base[d] + old + __popc(same & ((1u << lane) - 1u)), pair[u]);
      }
    }
    cluster_sync();  // the pairs are written for all, and no block stores totals or counts before all have read theirs
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
  int run;               // tokens of a warp
  int64_t tiles;         // column tiles of 32 * VEC
};

constexpr int kSumWarps = 8;  // of a chunk
constexpr int kSumThreads = 32 * kSumWarps;
constexpr int kSumUnroll = 8;

// Bound: HBM, the gathered rows of dy.  kSumUnroll rows are in flight per lane, and what an accumulated row holds already is
// asked for when its first token is met.
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kSumThreads) embedding_sum_kernel(SumArgs a) {
  __shared__ float parts[kSumWarps][32 * VEC];  // the warp's part of a row that began before it
  __shared__ int through[kSumWarps];            // that row takes all of the warp's tokens and goes on behind it
  grid_dependency_trigger();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t chunk = blockIdx.x / a.tiles, col = (blockIdx.x % a.tiles * 32 + lane) * VEC;
  const int64_t from = (chunk * kSumWarps + warp) * a.run, to = min(from + a.run, a.n);
  const bool here = col < a.width;  // lanes behind the last column see to the tokens alone
  const uint32_t rows = (uint32_t)a.rows;
  const T* dy = static_cast<const T*>(a.dy) + (here ? col : 0);
  O* dx = static_cast<O*>(a.dx) + col;
  uint32_t row = rows, before = rows, behind = rows;
  float sum[VEC];
  Group<O, VEC> old;
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  auto begin = [&](uint32_t r) {
    row = r;
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
    if (a.accumulate && here && r < rows && r != before) old.load(dx + (int64_t)r * a.width);
  };
  auto put = [&](const float* s, const Group<O, VEC>& was, uint32_t r) {
    if (!here) return;
    Group<O, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.x[j] = a.accumulate ? fmaf(s[j], a.scale, was.x[j]) : s[j] * a.scale;
    o.store(dx + (int64_t)r * a.width);
  };
  auto keep = [&] {
#pragma unroll
    for (int j = 0; j < VEC; ++j) parts[warp][j * 32 + lane] = sum[j];
  };
  bool through_w = false;
  if (from < a.n) {
    before = from ? a.sorted[from - 1].x : rows;
    behind = to < a.n ? a.sorted[to].x : rows;
    bool first = true;
    for (int64_t i0 = from; i0 < to; i0 += 32) {
      const uint2 mine = i0 + lane < to ? a.sorted[i0 + lane] : make_uint2(rows, 0);
      const int count = (int)min((int64_t)32, to - i0);
      for (int q0 = 0; q0 < count; q0 += kSumUnroll) {
        if (__shfl_sync(0xffffffffu, mine.x, q0) >= rows) break;
        uint32_t r[kSumUnroll];
        typename Group<T, VEC>::W g[kSumUnroll];
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
          r[u] = __shfl_sync(0xffffffffu, mine.x, q0 + u);
          const uint32_t at = __shfl_sync(0xffffffffu, mine.y, q0 + u);
          // without a condition, or the loads would wait for one another: what does not count is loaded all the same
          g[u] = *reinterpret_cast<const typename Group<T, VEC>::W*>(dy + (int64_t)at * a.width);
        }
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
          if (r[u] >= rows) break;  // behind the last token that counts
          if (first) {
            begin(r[u]);
            first = false;
          } else if (r[u] != row) {
            if (row == before) keep();
            else put(sum, old, row);
            begin(r[u]);
          }
          float x[VEC];
          Group<T, VEC>::unpack(g[u], x);
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum[j] += x[j];
        }
      }
    }
    // the last row: of this warp alone, begun before it, or going on behind it
    if (row < rows) {
      through_w = row == before && row == behind && row == a.sorted[from].x;
      if (row == before) keep();
      else if (row != behind) put(sum, old, row);
    }
  }
  if (lane == 0) through[warp] = through_w;
  const bool starts = row < rows && row != before && row == behind;   // a row goes on behind this warp
  const uint32_t head = warp == 0 && from < a.n ? a.sorted[from].x : rows;
  const bool enters = head < rows && head == before;                  // a row began before this chunk
  __syncthreads();
  if (!(starts || enters)) return;
  // warp 0 may see to two rows: the one that began before the chunk, and one that begins with it
  auto follow = [&](int w) {  // adds the parts of warps w, w + 1, ... as far as the row goes on; whether it leaves the chunk
    for (; w < kSumWarps; ++w) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] += parts[w][j * 32 + lane];
      if (!through[w]) return false;
    }
    return true;
  };
  auto put_partial = [&](int slot) {
    if (!here) return;
    Group<float, VEC> g;
#pragma unroll
    for (int j = 0; j < VEC; ++j) g.x[j] = sum[j];
    g.store(a.partial + (chunk * 2 + slot) * a.stride + col);
  };
  if (starts) {
    if (warp == kSumWarps - 1 || follow(warp + 1)) put_partial(1);
    else put(sum, old, row);
  }
  if (enters) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
    follow(0);
    put_partial(0);
  }
}

// The rows that chunks have cut: the block of the chunk in which a row begins adds up its parts.  Eight warps take
// every eighth part, and their sums are added in the order of the warps.
constexpr int kJoinThreads = 256;
constexpr int kJoinCols = 128;

template <typename O>
__global__ void __launch_bounds__(kJoinThreads) embedding_join_kernel(SumArgs a) {
  __shared__ float4 part[kJoinThreads / 32][32];
  grid_dependency_trigger();
  grid_dependency_wait();
  const int64_t tokens = (int64_t)kSumWarps * a.run, chunk = blockIdx.x, from = chunk * tokens, to = from + tokens;
  if (to >= a.n) return;
  const uint32_t row = a.sorted[to].x, last = a.sorted[to - 1].x, before = from ? a.sorted[from - 1].x : (uint32_t)a.rows;
  if (row >= (uint32_t)a.rows || last != row || before == row) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.y * kJoinCols + lane * 4;
  const float* at = a.partial + col;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < a.width) {
    if (warp == 0) sum = *reinterpret_cast<const float4*>(at + (chunk * 2 + 1) * a.stride);
#pragma unroll 4
    for (int64_t c = chunk + 1 + warp; c * tokens < a.n && a.sorted[c * tokens].x == row; c += kJoinThreads / 32) {
      const float4 p = *reinterpret_cast<const float4*>(at + c * 2 * a.stride);
      sum.x += p.x;
      sum.y += p.y;
      sum.z += p.z;
      sum.w += p.w;
    }
  }
  part[warp][lane] = sum;
  __syncthreads();
  if (warp || col >= a.width) return;
#pragma unroll
  for (int w = 1; w < kJoinThreads / 32; ++w) {
    sum.x += part[w][lane].x;
    sum.y += part[w][lane].y;
    sum.z += part[w][lane].z;
    sum.w += part[w][lane].w;
  }
  const float s[4] = {sum.x, sum.y, sum.z, sum.w};
  O* dx = static_cast<O*>(a.dx) + (int64_t)row * a.width + col;
  for (int j = 0; j < 4 && col + j < a.width; ++j)
    dx[j] = Elem<O>::from_f32(a.accumulate ? fmaf(s[j], a.scale, Elem<O>::to_f32(dx[j])) : s[j] * a.scale);
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

// Tokens of a warp: many of them cut fewer rows, few of them give every SM four blocks.
static int warp_tokens(int64_t n, int64_t width) {
  const int64_t tiles = (width + 255) / 256, want = n * tiles / (148 * 4 * kSumWarps) / kSumUnroll * kSumUnroll;
  return (int)std::min<int64_t>(std::max<int64_t>(want, kSumUnroll), 128);
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
  int tpr_log = 5;
  while (tpr_log < 8 && ((int64_t)1 << tpr_log) * vec < width) ++tpr_log;
  const int64_t per_block = (int64_t)(kLookupThreads >> tpr_log) * kLookupRows, grid = (n + per_block - 1) / per_block;
  RAFB200_REQUIRE(grid < ((int64_t)1 << 31), "rafb200_embedding: too many indices");
  const Ids ids{indices, index_dtype == RAFB200_I64};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_type(x_dtype, [&](auto t) {
    return with_type(out_dtype, [&](auto o) {
      return with_width<decltype(t)>(vec, [&](auto w) {
        using T = decltype(t);
        using O = decltype(o);
        RAFB200_CUDA(launch_dependent(embedding_kernel<T, O, decltype(w)::value>, dim3((unsigned)grid), kLookupThreads, 0, s,
                                      static_cast<const T*>(x), ids, n, rows, width, scale, static_cast<O*>(out), tpr_log));
        return (int)RAFB200_OK;
      });
    });
  });
}

// The workspace holds the pairs twice, then the partial sums of the chunks.
size_t rafb200_embedding_dx_workspace_bytes(int64_t n, int64_t width) {
  if (n <= 0 || width <= 0 || n >= ((int64_t)1 << 31) || range_overflows(n, width)) return 0;
  const int64_t tokens = (int64_t)kSumWarps * warp_tokens(n, width), chunks = (n + tokens - 1) / tokens;
  return 2 * round_up((size_t)n * sizeof(uint2)) + (size_t)chunks * 2 * ((width + 7) & ~int64_t(7)) * sizeof(float);
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

  SortArgs so{};
  so.ids = Ids{indices, index_dtype == RAFB200_I64};
  so.n = n;
  so.rows = rows;
  so.padding = padding_idx;
  so.a = static_cast<uint2*>(workspace);
  so.b = reinterpret_cast<uint2*>(static_cast<char*>(workspace) + round_up((size_t)n * sizeof(uint2)));
  int bits = 1;
  while (rows >> bits) ++bits;
  so.passes = (bits + kDigitBits - 1) / kDigitBits;
  so.bits = (bits + so.passes - 1) / so.passes;
  if (!accumulate) {
    so.fill = static_cast<unsigned char*>(dx);
    so.fill_bytes = rows * width * dtype_size(dx_dtype);
  }
  // three to six times as fast as the cluster's passes where a warp has one token to compare, and no slower at the border:
  // XXX
  if (n <= kRankTokens) {
    const int64_t ranks = (n + kRankThreads / 32 - 1) / (kRankThreads / 32), fills = so.fill_bytes / (kRankThreads * 64);
    const unsigned grid = (unsigned)std::min<int64_t>(std::max<int64_t>({ranks, fills, 1}), 148 * 4);
    RAFB200_CUDA(launch_dependent(embedding_rank_kernel, dim3(grid), kRankThreads, 0, s, so));
  } else {
    const int64_t each = (int64_t)kSortBlocks * kSortThreads * 64;  // four stores a thread
    const unsigned clusters = 1 + (unsigned)std::min<int64_t>((so.fill_bytes + each - 1) / each, kFillClusters);
    if (const int rc = allow_smem<embedding_sort_kernel>(kSortSmem)) return rc;
    RAFB200_CUDA(launch_cluster(embedding_sort_kernel, kSortBlocks, clusters * kSortBlocks, kSortThreads, kSortSmem, s, so));
  }
  if (n == 0) return RAFB200_OK;

  const int vec = group_width(dy, dtype_size(dy_dtype), dx, dtype_size(dx_dtype), width);
  SumArgs a{};
  a.dy = dy;
  a.sorted = so.a;
  a.n = n;
  a.rows = rows;
  a.width = width;
  a.scale = scale;
  a.accumulate = accumulate;
  a.dx = dx;
  a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + 2 * round_up((size_t)n * sizeof(uint2)));
  a.stride = (width + 7) & ~int64_t(7);
  a.tiles = (width + 32 * vec - 1) / (32 * vec);
  a.run = warp_tokens(n, width);
  const int64_t tokens = (int64_t)kSumWarps * a.run, chunks = (n + tokens - 1) / tokens;
  const int64_t grid = chunks * a.tiles, cols = (width + kJoinCols - 1) / kJoinCols;
  RAFB200_REQUIRE(grid < ((int64_t)1 << 31) && cols < 65536, "rafb200_embedding_dx: rows too wide");
  return with_type(dx_dtype, [&](auto o) {
    using O = decltype(o);
    const int rc = with_type(dy_dtype, [&](auto t) {
      return with_width<decltype(t)>(vec, [&](auto w) {
        RAFB200_CUDA(launch_dependent(embedding_sum_kernel<decltype(t), O, decltype(w)::value>, dim3((unsigned)grid), kSumThreads,
                                      0, s, a));
        return (int)RAFB200_OK;
      });
    });
    if (rc != RAFB200_OK || chunks == 1) return rc;
    RAFB200_CUDA(launch_dependent(embedding_join_kernel<O>, dim3((unsigned)(chunks - 1), (unsigned)cols), kJoinThreads, 0, s, a));
    return (int)RAFB200_OK;
  });
}

}  // extern "C"
