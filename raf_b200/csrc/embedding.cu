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
//   1. the tokens are sorted, stably, by one cluster of eight blocks, while the other clusters write the zeros of rows
//      without a token;
//   2. a warp walks a chunk of the sorted tokens for 32 * VEC columns and keeps the sum of the present row in registers.
//      A row whose tokens all lie in one chunk is written here; a row cut by a chunk's border leaves partial sums;
//   3. the rows that were cut are joined, chunk after chunk.
constexpr int kSortBlocks = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigitBits = 9;  // two passes for tables of up to 2^18 - 1 rows; the counters of 32 warps take 64 KB
constexpr int kDigits = 1 << kDigitBits;
constexpr int kFillClusters = 17;  // with the sorting one 144 blocks of 148 SMs
constexpr size_t kSortSmem = sizeof(uint32_t) * (kSortWarps * kDigits + 2 * kDigits + 32);

struct SortArgs {
  Ids ids;
  int64_t n;
  int64_t rows;        // valid ids are [0, rows); every other id sorts as `rows`, behind them
  int64_t padding;
  uint2* a;            // (id, position) pairs: the last pass leaves them in a
  uint2* b;
  int passes, bits;    // digits and bits of each
  unsigned char* fill; // bytes to zero, or nullptr
  int64_t fill_bytes;
};

__device__ void zero_bytes(unsigned char* p, int64_t bytes, int64_t worker, int64_t workers) {
  const int64_t head = min((int64_t)(-(intptr_t)p & 15), bytes);
  const int64_t vecs = (bytes - head) >> 4, tail = head + (vecs << 4);
  uint4* q = reinterpret_cast<uint4*>(p + head);
  for (int64_t i = worker; i < vecs; i += workers) q[i] = make_uint4(0, 0, 0, 0);
  if (worker < head) p[worker] = 0;
  if (worker < bytes - tail) p[tail + worker] = 0;
}

// Digits from the lowest up.  Each of the cluster's 256 warps owns a contiguous range of the pairs: it counts
// its digits, the counts are summed over warps, blocks (through distributed shared memory) and digits, and
// the warp then moves its pairs in order, equal digits of a group of 32 ranked by lane.
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(SortArgs a) {
  extern __shared__ uint32_t counts[];  // [warp][digit]
  uint32_t* totals = counts + kSortWarps * kDigits;
  uint32_t* base = totals + kDigits;
  uint32_t* scan = base + kDigits;
  grid_dependency_trigger();
  grid_dependency_wait();
  if (blockIdx.x >= kSortBlocks) {
    zero_bytes(a.fill, a.fill_bytes, (int64_t)(blockIdx.x - kSortBlocks) * kSortThreads + threadIdx.x,
               (int64_t)(gridDim.x - kSortBlocks) * kSortThreads);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cluster_rank();
  const int64_t each = ((a.n + kSortBlocks * kSortWarps - 1) / (kSortBlocks * kSortWarps) + 31) & ~int64_t(31);
  const int64_t from = min(((int64_t)rank * kSortWarps + warp) * each, a.n), to = min(from + each, a.n);
  uint32_t* mine = counts + warp * kDigits;
  const int digits = 1 << a.bits;
  for (int pass = 0; pass < a.passes; ++pass) {
    const int shift = pass * a.bits;
    // the passes end in a
    const uint2* src = ((a.passes - pass) & 1) ? a.b : a.a;
    uint2* dst = ((a.passes - pass) & 1) ? a.a : a.b;
    auto pair_at = [&](int64_t i) {
      if (pass) return __ldcg(src + i);
      const int64_t id = a.ids[i];
      const bool counts_in = (uint64_t)id < (uint64_t)a.rows && id != a.padding;
      return make_uint2(counts_in ? (uint32_t)id : (uint32_t)a.rows, (uint32_t)i);
    };
    for (int d = lane; d < digits; d += 32) mine[d] = 0;
    __syncwarp();
    for (int64_t i0 = from; i0 < to; i0 += 32) {
      const bool in = i0 + lane < to;
      const uint32_t d = in ? (pair_at(i0 + lane).x >> shift) & (digits - 1) : digits;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (in && lane == __ffs(same) - 1) mine[d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    for (int d = tid; d < digits; d += kSortThreads) {
      uint32_t sum = 0;
      for (int w = 0; w < kSortWarps; ++w) {
        const uint32_t c = counts[w * kDigits + d];
        counts[w * kDigits + d] = sum;
        sum += c;
      }
      totals[d] = sum;
    }
    cluster_sync();
    uint32_t before = 0, all = 0;  // of this thread's digit: in the blocks before this one, in all of them
    if (tid < digits) {
      for (uint32_t r = 0; r < kSortBlocks; ++r) {
        const uint32_t c = cluster_load(totals + tid, r);
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
      for (int w = 0; w < warp; ++w) lower += scan[w];
      base[tid] = lower + before;
    }
    __syncthreads();
    for (int64_t i0 = from; i0 < to; i0 += 32) {
      const bool in = i0 + lane < to;
      uint2 pair = make_uint2(0, 0);
      uint32_t d = digits;
      if (in) {
        pair = pair_at(i0 + lane);
        d = (pair.x >> shift) & (digits - 1);
      }
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      uint32_t old = 0;
      if (in) old = mine[d];
      __syncwarp();
      if (in && lane == __ffs(same) - 1) mine[d] = old + __popc(same);
      __syncwarp();
      if (in) __stcg(dst + base[d] + old + __popc(same & ((1u << lane) - 1u)), pair);
    }
    cluster_sync();  // the pairs are written for all, and no block reads the totals any more
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
  int chunk;             // tokens of a chunk
  int64_t tiles;         // column tiles of 32 * VEC
};

constexpr int kSumThreads = 256;
constexpr int kSumUnroll = 4;

template <typename O, int VEC>
__device__ __forceinline__ void put_row(const SumArgs& a, uint32_t row, int64_t col, const float* sum) {
  O* at = static_cast<O*>(a.dx) + (int64_t)row * a.width + col;
  Group<O, VEC> o;
  if (a.accumulate) {
    o.load(at);
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.x[j] = fmaf(sum[j], a.scale, o.x[j]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.x[j] = sum[j] * a.scale;
  }
  o.store(at);
}

// Bound: HBM, the gathered rows of dy.  kSumUnroll rows are in flight per lane.
template <typename T, typename O, int VEC>
__global__ void __launch_bounds__(kSumThreads) embedding_sum_kernel(SumArgs a) {
  grid_dependency_trigger();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * (kSumThreads / 32) + (threadIdx.x >> 5);
  const int64_t chunk = unit / a.tiles, col = (unit % a.tiles * 32 + lane) * VEC;
  const int64_t from = chunk * a.chunk, to = min(from + a.chunk, a.n);
  if (from >= a.n || col >= a.width) return;
  const T* dy = static_cast<const T*>(a.dy) + col;
  const uint32_t before = from ? a.sorted[from - 1].x : 0xffffffffu;
  const uint32_t behind = to < a.n ? a.sorted[to].x : 0xffffffffu;
  uint32_t row = a.sorted[from].x;
  float sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  auto put_partial = [&](int slot) {
    float* at = a.partial + (chunk * 2 + slot) * a.stride + col;
    if constexpr (VEC == 8) {
      reinterpret_cast<float4*>(at)[0] = make_float4(sum[0], sum[1], sum[2], sum[3]);
      reinterpret_cast<float4*>(at)[1] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) at[j] = sum[j];
    }
  };
  for (int64_t i0 = from; i0 < to; i0 += kSumUnroll) {
    uint2 pair[kSumUnroll];
    Group<T, VEC> g[kSumUnroll];
#pragma unroll
    for (int u = 0; u < kSumUnroll; ++u) pair[u] = i0 + u < to ? a.sorted[i0 + u] : make_uint2(0xffffffffu, 0);
#pragma unroll
    for (int u = 0; u < kSumUnroll; ++u)
      if (pair[u].x < (uint32_t)a.rows) g[u].load(dy + (int64_t)pair[u].y * a.width);
#pragma unroll
    for (int u = 0; u < kSumUnroll; ++u) {
      if (pair[u].x >= (uint32_t)a.rows) continue;
      if (pair[u].x != row) {
        if (row == before) put_partial(0);
        else put_row<O, VEC>(a, row, col, sum);
        row = pair[u].x;
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] += g[u].x[j];
    }
  }
  if (row >= (uint32_t)a.rows) return;
  if (row == before) put_partial(0);
  else if (row == behind) put_partial(1);
  else put_row<O, VEC>(a, row, col, sum);
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
  const int64_t chunk = blockIdx.x, from = chunk * a.chunk, to = from + a.chunk;
  if (to >= a.n) return;
  const uint32_t row = a.sorted[to].x;
  if (row >= (uint32_t)a.rows || a.sorted[to - 1].x != row || (from && a.sorted[from - 1].x == row)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t col = (int64_t)blockIdx.y * kJoinCols + lane * 4;
  const float* at = a.partial + col;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < a.width) {
    if (warp == 0) sum = *reinterpret_cast<const float4*>(at + (chunk * 2 + 1) * a.stride);
    for (int64_t c = chunk + 1 + warp; c * a.chunk < a.n && a.sorted[c * a.chunk].x == row; c += kJoinThreads / 32) {
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
  for (int j = 0; j < 4 && col + j < a.width; ++j) put_row<O, 1>(a, row, col + j, s + j);
}

// Elements of a vector access that every row of both arrays allows.
static int group_width(const void* p, int size_p, const void* q, int size_q, int64_t width) {
  auto fits = [&](int vec, int bytes_p, int bytes_q) {
    return width % vec == 0 && reinterpret_cast<uintptr_t>(p) % bytes_p == 0 && reinterpret_cast<uintptr_t>(q) % bytes_q == 0;
  };
  if (fits(8, 16, 16)) return 8;
  return fits(2, 2 * size_p, 2 * size_q) ? 2 : 1;
}

template <typename F>
static int with_width(int vec, const F& f) {
  switch (vec) {
    case 8: return f(std::integral_constant<int, 8>{});
    case 2: return f(std::integral_constant<int, 2>{});
    default: return f(std::integral_constant<int, 1>{});
  }
}

static bool range_overflows(int64_t a, int64_t b) {
  int64_t r;
  return __builtin_mul_overflow(a, b, &r) || r > ((int64_t)1 << 60);
}

// Tokens of a chunk: long chunks cut fewer rows, and short ones give every SM 32 warps.
static int chunk_tokens(int64_t n, int64_t tiles) {
  const int64_t want = n * tiles / (148 * 32) / kSumUnroll * kSumUnroll;
  return (int)std::min<int64_t>(std::max<int64_t>(want, 2 * kSumUnroll), 256);
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
      return with_width(vec, [&](auto w) {
        using T = decltype(t);
        using O = decltype(o);
        RAFB200_CUDA(launch_dependent(embedding_kernel<T, O, decltype(w)::value>, dim3((unsigned)grid), kLookupThreads, 0, s,
                                      static_cast<const T*>(x), ids, n, rows, width, scale, static_cast<O*>(out), tpr_log));
        return (int)RAFB200_OK;
      });
    });
  });
}

// Layout of the workspace: the pairs twice, then the partial sums.  It does not go by the widths of accesses,
// which depend on addresses: the partial sums are those of the narrowest chunks there can be.
size_t rafb200_embedding_dx_workspace_bytes(int64_t n, int64_t width) {
  if (n <= 0 || width <= 0 || n >= ((int64_t)1 << 31) || range_overflows(n, width)) return 0;
  const int64_t chunks = (n + chunk_tokens(n, (width + 255) / 256) - 1) / chunk_tokens(n, (width + 255) / 256);
  return 2 * round_up((size_t)n * sizeof(uint2)) + (size_t)chunks * 2 * ((width + 7) & ~7) * sizeof(float);
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
  unsigned clusters = 1;
  if (!accumulate) {
    so.fill = static_cast<unsigned char*>(dx);
    so.fill_bytes = rows * width * dtype_size(dx_dtype);
    const int64_t each = (int64_t)kSortBlocks * kSortThreads * 64;  // four stores a thread
    clusters += (unsigned)std::min<int64_t>((so.fill_bytes + each - 1) / each, kFillClusters);
  }
  if (const int rc = allow_smem<embedding_sort_kernel>(kSortSmem)) return rc;
  RAFB200_CUDA(launch_cluster(embedding_sort_kernel, kSortBlocks, clusters * kSortBlocks, kSortThreads, kSortSmem, s, so));
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
  a.chunk = chunk_tokens(n, (width + 255) / 256);
  const int64_t chunks = (n + a.chunk - 1) / a.chunk;
  const int64_t grid = (chunks * a.tiles + kSumThreads / 32 - 1) / (kSumThreads / 32), cols = (width + kJoinCols - 1) / kJoinCols;
  RAFB200_REQUIRE(grid < ((int64_t)1 << 31) && cols < 65536, "rafb200_embedding_dx: rows too wide");
  return with_type(dx_dtype, [&](auto o) {
    using O = decltype(o);
    const int rc = with_type(dy_dtype, [&](auto t) {
      return with_width(vec, [&](auto w) {
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
