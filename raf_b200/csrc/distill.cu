// Distillation loss against a teacher's top logits, and its gradient.
//
// A row has student logits z (v of them), and k teacher entries (class j_i, logit t_i); entries whose class is outside
// [0, v) are absent.  With
//   p = softmax of the present t_i / T,  q = softmax(z / T),  r = softmax(z),  S = sum p (1, or 0 without a teacher)
//   loss   = alpha T^2 sum_i p_i (log p_i - log q_{j_i}) + (1 - alpha) (-log r_label)
//   dz_j   = alpha T (S q_j - sum over i with j_i = j of p_i) + (1 - alpha) (r_j - [j = label])
// The second terms only with labels; a row whose label is ignore_index or outside [0, v) has loss and gradient 0
// whatever its logits.
//
// Exponentials are those of base 2 of (z - m) c with m the row's maximum and c = log2(e) / T: the difference first, so that
// neither the product overflows at a type's lowest values (masks) nor logits far from zero lose digits.  Sums are fp32,
// in a fixed order.
#include <cmath>

#include "model_io.cuh"

namespace rafb200 {

constexpr int kDistillThreads = 512;
constexpr int kDistillWarps = kDistillThreads / 32;
constexpr int kDistillUnroll = 4;
constexpr int kMaxTeacher = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DistillArgs {
  const void* pred;
  const void* teacher;
  Ids ids;
  Ids labels;       // p == nullptr: none
  const float* dy;  // one weight per row (dy_step 1), one for all (0), or nullptr: 1
  float* loss;
  float4* stats;    // per row: maximum, sum of exponentials at the temperature, the same at one, 0
  void* out;
  int64_t n, v, ld, ld_out, ignore;
  int k, teacher_type, dy_step;
  float c, soft_loss, soft_grad, hard, grad_scale;  // log2(e) / T, alpha T^2, alpha T, 1 - alpha
  int slices;       // blocks of a row
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float load_teacher(const DistillArgs& a, int64_t i) {
  if (a.teacher_type == RAFB200_F32) return static_cast<const float*>(a.teacher)[i];
  if (a.teacher_type == RAFB200_F16) return __half2float(static_cast<const __half*>(a.teacher)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher)[i]);
}

// Maximum and sums of exponentials seen so far.
struct Running {
  float top, soft, hard;
};
// What logits are taken relative to: of -infinity alone, 0, so that their exponentials are 0 and not those of NaN.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.f : top; }
__device__ __forceinline__ float power(float z, float base, float c) { return ex2((z - base) * c); }

template <bool TWO>
__device__ __forceinline__ Running merge(const Running& x, const Running& y, float c) {
  Running r;
  r.top = fmaxf(x.top, y.top);
  const float base = base_of(r.top), dx = base_of(x.top) - base, dy = base_of(y.top) - base;
  // sums over -infinity alone are 0, or NaN, and stay it, whatever the distance of the maxima
  r.soft = x.soft * (x.top == -INFINITY ? 1.f : ex2(dx * c)) + y.soft * (y.top == -INFINITY ? 1.f : ex2(dy * c));
  r.hard = 0.f;
  if (TWO)
    r.hard = x.hard * (x.top == -INFINITY ? 1.f : ex2(dx * kLog2e)) + y.hard * (y.top == -INFINITY ? 1.f : ex2(dy * kLog2e));
  return r;
}

// A block's part of a row: 16-byte groups [from, to) of the aligned middle; the elements in front of
// the middle are the first block's, those behind it the last one's.
template <typename T>
struct Slice {
  static constexpr int kPer = 16 / sizeof(T);
  int64_t head, from, to, body;  // elements in front; groups; first element behind the middle
  int edge;                      // elements of this block outside the middle: thread i < edge takes edge_at(i)
  int64_t v;
  int first;                     // of them in front

  __device__ __forceinline__ Slice(const T* row, int64_t v_, int slice, int slices) : v(v_) {
    head = min((int64_t)((-(intptr_t)row & 15) / sizeof(T)), v);
    const int64_t groups = (v - head) / kPer, each = (groups + slices - 1) / slices;
    from = min(slice * each, groups);
    to = min(from + each, groups);
    body = head + groups * kPer;
    first = slice == 0 ? (int)head : 0;
    edge = first + (slice == slices - 1 ? (int)(v - body) : 0);
  }
  __device__ __forceinline__ int64_t edge_at(int i) const { return i < first ? i : body + (i - first); }
  __device__ __forceinline__ bool owns(int64_t j, bool first_slice, bool last_slice) const {
    if (j < head) return first_slice;
    if (j >= body) return last_slice;
    const int64_t g = (j - head) / kPer;
    return g >= from && g < to;
  }
};

// The teacher's entries of a row in shared memory: class (-1: absent), weight p, student's logit there.
// Entry k is the label, with weight 0.
struct Entries {
  int* at;
  float* p;
  float* z;
  __device__ __forceinline__ Entries(void* smem, int k)
      : at(static_cast<int*>(smem)), p(reinterpret_cast<float*>(at + k + 1)), z(p + k + 1) {}
  static size_t bytes(int k) { return (size_t)(k + 1) * 12; }
};

// softmax over the present entries; the sum of the weights (1 or 0), and with `loss` sum p (log p - log q).  One warp.
__device__ __forceinline__ float weigh(const Entries& e, int k, float c, float base, float log2_soft, bool want, float* kl) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int i = lane; i < k; i += 32)
    if (e.at[i] >= 0) top = fmaxf(top, e.p[i]);
#pragma unroll
  for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  const float t_base = base_of(top);
  float sum = 0.f;
  for (int i = lane; i < k; i += 32)
    if (e.at[i] >= 0) sum += power(e.p[i], t_base, c);
  sum = warp_sum(sum);
  const bool some = sum != 0.f;  // false: no teacher, or all of it at -infinity
  const float inv = some ? 1.f / sum : 0.f, log2_sum = log2f(sum);
  float part = 0.f;
  for (int i = lane; i < k; i += 32) {
    const float t = (e.p[i] - t_base) * c;
    const float w = e.at[i] >= 0 && some ? ex2(t) * inv : 0.f;
    if (want && !(w == 0.f)) part = fmaf(w, (t - log2_sum) - ((e.z[i] - base) * c - log2_soft), part);  // log2 p - log2 q
    e.p[i] = w;
  }
  if (want) *kl = warp_sum(part) * kLn2;
  return isnan(sum) ? sum : some ? 1.f : 0.f;
}

template <typename T>
__device__ __forceinline__ void load_entries(const DistillArgs& a, const Entries& e, int64_t row, const T* z, int64_t label) {
  for (int i = threadIdx.x; i <= a.k; i += kDistillThreads) {
    const int64_t j = i < a.k ? a.ids[row * a.k + i] : label;
    const bool in = (uint64_t)j < (uint64_t)a.v;
    e.at[i] = in ? (int)j : -1;
    e.p[i] = i < a.k ? load_teacher(a, row * a.k + i) : 0.f;
    e.z[i] = in ? Elem<T>::to_f32(z[j]) : 0.f;
  }
}

// What a gradient is made of: dz = soft * 2^((z - base) c) + hard * 2^((z - base) log2e), at the entries minus
// teach * (sum of p), and minus hit at the label.
struct Coefficients {
  float c, base, soft, hard, teach, hit;
  template <bool TWO>
  __device__ __forceinline__ float at(float z) const {
    float g = soft * power(z, base, c);
    if (TWO) g = fmaf(hard, power(z, base, kLog2e), g);
    return g;
  }
};

template <bool TWO>
__device__ __forceinline__ Coefficients coefficients(const DistillArgs& a, int64_t row, float4 stats, float some, bool labels) {
  const float w = (a.dy ? a.dy[row * a.dy_step] : 1.f) * a.grad_scale;
  Coefficients co;
  co.c = a.c;
  co.base = base_of(stats.x);
  co.teach = w * a.soft_grad;
  co.hit = labels ? w * a.hard : 0.f;
  co.soft = co.teach * some / stats.y;
  co.hard = co.hit / stats.z;
  if (!TWO) {  // one exponential serves both terms, or there is one term only
    co.soft += labels ? co.hit / stats.y : 0.f;
    co.hard = 0.f;
  }
  return co;
}

// The gradient of a slice: `get(i)` is the group of 16 bytes i, `edge` this thread's element outside the middle.
template <typename T, bool TWO, typename Get>
__device__ __forceinline__ void write_slice(const Slice<T>& s, T* out, const Coefficients& co, float edge, const Get& get) {
  constexpr int per = Slice<T>::kPer;
  T* middle = out + s.head;
  const bool aligned = (reinterpret_cast<uintptr_t>(middle) & 15) == 0;
  for (int64_t i = s.from + threadIdx.x; i < s.to; i += kDistillThreads) {
    float z[per];
    Group<T, 8>::template unpack<T>(get(i), z);
#pragma unroll
    for (int j = 0; j < per; ++j) z[j] = co.at<TWO>(z[j]);
    if (aligned) {
      reinterpret_cast<uint4*>(middle)[i] = Group<T, 8>::template pack<T>(z);
    } else {
#pragma unroll
      for (int j = 0; j < per; ++j) middle[i * per + j] = Elem<T>::from_f32(z[j]);
    }
  }
  if ((int)threadIdx.x < s.edge) out[s.edge_at(threadIdx.x)] = Elem<T>::from_f32(co.at<TWO>(edge));
}

// The elements that the teacher or the label names, once each however often they are named.
template <typename T, bool TWO>
__device__ __forceinline__ void write_entries(const DistillArgs& a, const Entries& e, const Slice<T>& s, T* out, const Coefficients& co,
                                              bool first_slice, bool last_slice) {
  for (int i = threadIdx.x; i <= a.k; i += kDistillThreads) {
    const int j = e.at[i];
    if (j < 0 || !s.owns(j, first_slice, last_slice)) continue;
    bool again = false;
    float p = e.p[i];
    for (int q = 0; q <= a.k; ++q) {
      if (q == i || e.at[q] != j) continue;
      again |= q < i;
      p += e.p[q];
    }
    if (again) continue;
    float g = co.at<TWO>(e.z[i]) - co.teach * p;
    if (e.at[a.k] == j) g -= co.hit;
    out[j] = Elem<T>::from_f32(g);
  }
}

template <typename T>
__device__ __forceinline__ void zero_slice(const Slice<T>& s, T* out) {
  for (int64_t i = s.from * Slice<T>::kPer + threadIdx.x; i < s.to * Slice<T>::kPer; i += kDistillThreads)
    out[s.head + i] = Elem<T>::from_f32(0.f);
  if ((int)threadIdx.x < s.edge) out[s.edge_at(threadIdx.x)] = Elem<T>::from_f32(0.f);
}

// Loss, and with GRAD the gradient, of a row by a cluster of `slices` blocks: one pass with a running maximum and its
// sums, joined over threads, warps and blocks.
template <typename T, bool TWO, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads) distill_kernel(DistillArgs a) {
  constexpr int per = Slice<T>::kPer;
  extern __shared__ char smem[];
  __shared__ Running warps[kDistillWarps];
  __shared__ Running whole;
  __shared__ float some_s;
  const Entries e(smem, a.k);
  grid_dependency_trigger();
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  const Slice<T> s(z, a.v, slice, a.slices);
  T* out = GRAD ? static_cast<T*>(a.out) + row * a.ld_out : nullptr;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && (label == a.ignore || (uint64_t)label >= (uint64_t)a.v)) {  // the same for every block of the cluster
    if (slice == 0 && tid == 0) {
      a.loss[row] = 0.f;
      if (a.stats) a.stats[row] = make_float4(0.f, 1.f, 1.f, 0.f);
    }
    if (GRAD) zero_slice(s, out);
    return;
  }
  load_entries(a, e, row, z, label);

  Running run{-INFINITY, 0.f, 0.f};
  const uint4* middle = reinterpret_cast<const uint4*>(z + s.head);
  const T lowest = Elem<T>::from_f32(-INFINITY);
  const uint32_t pad = sizeof(T) == 4 ? __float_as_uint(-INFINITY) : (uint32_t)reinterpret_cast<const uint16_t&>(lowest) * 0x10001u;
  for (int64_t i0 = s.from + tid; i0 < s.to; i0 += kDistillThreads * kDistillUnroll) {
    uint4 raw[kDistillUnroll];
#pragma unroll
    for (int u = 0; u < kDistillUnroll; ++u) {
      const int64_t i = i0 + u * kDistillThreads;
      raw[u] = i < s.to ? middle[i] : make_uint4(pad, pad, pad, pad);
    }
    float f[kDistillUnroll * per];
    float top = run.top;
#pragma unroll
    for (int u = 0; u < kDistillUnroll; ++u) Group<T, 8>::template unpack<T>(raw[u], f + u * per);
#pragma unroll
    for (int j = 0; j < kDistillUnroll * per; ++j) top = fmaxf(top, f[j]);
    Running next = merge<TWO>(run, Running{top, 0.f, 0.f}, a.c);
    const float base = base_of(top);
#pragma unroll
    for (int j = 0; j < kDistillUnroll * per; ++j) {
      next.soft += power(f[j], base, a.c);
      if (TWO) next.hard += power(f[j], base, kLog2e);
    }
    run = next;
  }
  float edge = 0.f;
  if (tid < s.edge) {
    edge = Elem<T>::to_f32(z[s.edge_at(tid)]);
    const float base = base_of(edge);
    run = merge<TWO>(run, Running{edge, power(edge, base, a.c), TWO ? power(edge, base, kLog2e) : 0.f}, a.c);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const Running other{__shfl_xor_sync(0xffffffffu, run.top, d), __shfl_xor_sync(0xffffffffu, run.soft, d),
                        TWO ? __shfl_xor_sync(0xffffffffu, run.hard, d) : 0.f};
    // the lower lane's sums first, on both sides
    run = lane & d ? merge<TWO>(other, run, a.c) : merge<TWO>(run, other, a.c);
  }
  if (lane == 0) warps[warp] = run;
  __syncthreads();
  if (tid == 0) {
    run = warps[0];
    for (int w = 1; w < kDistillWarps; ++w) run = merge<TWO>(run, warps[w], a.c);
    whole = run;
  }
  if (a.slices > 1) {
    cluster_sync();
    if (tid < 32) {
      run = Running{-INFINITY, 0.f, 0.f};
      for (int r = 0; r < a.slices; ++r) {
        Running other;
        other.top = __uint_as_float(cluster_load(&whole.top, r));
        other.soft = __uint_as_float(cluster_load(&whole.soft, r));
        other.hard = __uint_as_float(cluster_load(&whole.hard, r));
        run = merge<TWO>(run, other, a.c);
      }
    }
    cluster_sync();  // read by all before one of them overwrites it or ends
    if (tid == 0) whole = run;
  }
  __syncthreads();
  run = whole;
  const float base = base_of(run.top);
  const float4 stats = make_float4(run.top, run.soft, TWO ? run.hard : run.soft, 0.f);
  if (warp == 0) {
    float kl = 0.f;
    const float some = weigh(e, a.k, a.c, base, log2f(run.soft), true, &kl);
    if (lane == 0) some_s = some;
    if (lane == 0 && slice == 0) {
      float loss = a.soft_loss > 0.f ? a.soft_loss * kl : 0.f;  // a term without weight counts nothing, infinite or not
      if (labels && a.hard > 0.f) loss += a.hard * kLn2 * (log2f(stats.z) - (e.z[a.k] - base) * kLog2e);
      a.loss[row] = loss;
      if (a.stats) a.stats[row] = stats;
    }
  }
  if (!GRAD) return;
  __syncthreads();
  const Coefficients co = coefficients<TWO>(a, row, stats, some_s, labels);
  write_slice<T, TWO>(s, out, co, edge, [&](int64_t i) { return middle[i]; });
  __syncthreads();
  write_entries<T, TWO>(a, e, s, out, co, slice == 0, slice == a.slices - 1);
}

// The gradient from the statistics that the forward pass has left.
template <typename T, bool TWO>
__global__ void __launch_bounds__(kDistillThreads) distill_dpred_kernel(DistillArgs a) {
  extern __shared__ char smem[];
  __shared__ float some_s;
  const Entries e(smem, a.k);
  grid_dependency_trigger();
  grid_dependency_wait();
  const int64_t row = blockIdx.x / a.slices;
  const int slice = blockIdx.x % a.slices;
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  const Slice<T> s(z, a.v, slice, a.slices);
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && (label == a.ignore || (uint64_t)label >= (uint64_t)a.v)) {
    zero_slice(s, out);
    return;
  }
  const float4 stats = a.stats[row];
  // in place another block may have overwritten what its own slice names: those entries are not used here
  load_entries(a, e, row, z, label);
  const float edge = (int)threadIdx.x < s.edge ? Elem<T>::to_f32(z[s.edge_at(threadIdx.x)]) : 0.f;
  __syncthreads();
  if (threadIdx.x < 32) {
    const float some = weigh(e, a.k, a.c, 0.f, 0.f, false, nullptr);
    if (threadIdx.x == 0) some_s = some;
  }
  __syncthreads();
  const Coefficients co = coefficients<TWO>(a, row, stats, some_s, labels);
  const uint4* middle = reinterpret_cast<const uint4*>(z + s.head);
  write_slice<T, TWO>(s, out, co, edge, [&](int64_t i) { return middle[i]; });
  __syncthreads();
  write_entries<T, TWO>(a, e, s, out, co, slice == 0, slice == a.slices - 1);
}

static int check_args(const rafb200_distill* d, const char* who) {
  RAFB200_REQUIRE(d, "%s: NULL arguments", who);
  RAFB200_REQUIRE(dtype_valid(d->pred_dtype) && dtype_valid(d->teacher_dtype), "%s: bad dtype", who);
  RAFB200_REQUIRE(index_dtype_valid(d->ids_dtype) && (!d->labels || index_dtype_valid(d->labels_dtype)),
                  "%s: classes are int32 or int64", who);
  RAFB200_REQUIRE(d->n >= 0 && d->n < ((int64_t)1 << 28) && d->v >= 1 && d->v < ((int64_t)1 << 31), "%s: bad sizes", who);
  RAFB200_REQUIRE(d->k >= 0 && d->k <= kMaxTeacher, "%s: a row takes 0 to %d teacher entries", who, kMaxTeacher);
  RAFB200_REQUIRE(d->ld >= d->v && d->ld < ((int64_t)1 << 32), "%s: rows overlap", who);
  RAFB200_REQUIRE(d->temperature >= 0x1p-20 && d->temperature <= 0x1p20, "%s: the temperature lies in [2^-20, 2^20]", who);
  RAFB200_REQUIRE(d->alpha >= 0.0 && d->alpha <= 1.0, "%s: alpha lies in [0, 1]", who);
  RAFB200_REQUIRE(d->labels || d->alpha == 1.0 || d->n == 0, "%s: alpha below 1 needs labels", who);
  RAFB200_REQUIRE(d->n == 0 || (d->pred && (d->k == 0 || (d->teacher_logits && d->teacher_ids))), "%s: NULL argument", who);
  return RAFB200_OK;
}

static DistillArgs device_args(const rafb200_distill* d) {
  DistillArgs a{};
  a.pred = d->pred;
  a.teacher = d->teacher_logits;
  a.ids = Ids{d->teacher_ids, d->ids_dtype == RAFB200_I64};
  a.labels = Ids{d->labels, d->labels_dtype == RAFB200_I64};
  a.n = d->n;
  a.v = d->v;
  a.ld = d->ld;
  a.ignore = d->ignore_index;
  a.k = d->k;
  a.teacher_type = d->teacher_dtype;
  a.c = (float)(M_LOG2E / d->temperature);
  a.soft_loss = (float)(d->alpha * d->temperature * d->temperature);
  a.soft_grad = (float)(d->alpha * d->temperature);
  a.hard = (float)(1.0 - d->alpha);
  a.slices = 1;
  return a;
}

// Two exponentials an element where both terms count and their temperatures differ.
static bool two_exps(const rafb200_distill* d) { return d->labels && d->alpha < 1.0 && d->temperature != 1.0; }

static int row_slices(const rafb200_distill* d) {
  int slices = 1;
  const int64_t groups = d->v * dtype_size(d->pred_dtype) / 16;
  while (slices < 8 && d->n * slices * 2 <= 148 * 2 && groups / (slices * 2) >= kDistillThreads) slices *= 2;
  return slices;
}

template <typename F>
static int with_case(const rafb200_distill* d, const F& f) {
  return with_type(d->pred_dtype, [&](auto t) {
    return two_exps(d) ? f(t, std::integral_constant<bool, true>{}) : f(t, std::integral_constant<bool, false>{});
  });
}

}  // namespace rafb200

using namespace rafb200;

extern "C" {

int rafb200_distill_loss(const rafb200_distill* d, float* loss, float* stats, void* stream) {
  if (const int rc = check_args(d, "rafb200_distill_loss")) return rc;
  if (d->n == 0) return RAFB200_OK;
  RAFB200_REQUIRE(loss && stats && reinterpret_cast<uintptr_t>(stats) % 16 == 0, "rafb200_distill_loss: NULL or misaligned output");
  DistillArgs a = device_args(d);
  a.loss = loss;
  a.stats = reinterpret_cast<float4*>(stats);
  a.slices = row_slices(d);
  return with_case(d, [&](auto t, auto two) {
    RAFB200_CUDA(launch_cluster(distill_kernel<decltype(t), decltype(two)::value, false>, a.slices, (unsigned)(d->n * a.slices),
                                kDistillThreads, Entries::bytes(d->k), static_cast<cudaStream_t>(stream), a));
    return (int)RAFB200_OK;
  });
}

static int check_gradient(const rafb200_distill* d, const void* dpred, int64_t ld_out, const char* who) {
  RAFB200_REQUIRE(dpred && ld_out >= d->v && ld_out < ((int64_t)1 << 32), "%s: NULL gradient, or its rows overlap", who);
  const uintptr_t p = reinterpret_cast<uintptr_t>(d->pred), q = reinterpret_cast<uintptr_t>(dpred);
  const uintptr_t size = (uintptr_t)dtype_size(d->pred_dtype);
  const uintptr_t p_end = p + ((uintptr_t)(d->n - 1) * d->ld + d->v) * size, q_end = q + ((uintptr_t)(d->n - 1) * ld_out + d->v) * size;
  RAFB200_REQUIRE((p == q && d->ld == ld_out) || p_end <= q || q_end <= p, "%s: the gradient overlaps pred without being it", who);
  return RAFB200_OK;
}

int rafb200_distill_loss_dpred(const rafb200_distill* d, const float* dy, int dy_step, float grad_scale, const float* stats,
                               void* dpred, int64_t ld_dpred, void* stream) {
  if (const int rc = check_args(d, "rafb200_distill_loss_dpred")) return rc;
  if (d->n == 0) return RAFB200_OK;
  if (const int rc = check_gradient(d, dpred, ld_dpred, "rafb200_distill_loss_dpred")) return rc;
  RAFB200_REQUIRE(stats && reinterpret_cast<uintptr_t>(stats) % 16 == 0, "rafb200_distill_loss_dpred: NULL or misaligned stats");
  DistillArgs a = device_args(d);
  a.dy = dy;
  a.dy_step = dy_step ? 1 : 0;
  a.grad_scale = grad_scale;
  a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  a.out = dpred;
  a.ld_out = ld_dpred;
  a.slices = row_slices(d);
  return with_case(d, [&](auto t, auto two) {
    RAFB200_CUDA(launch_dependent(distill_dpred_kernel<decltype(t), decltype(two)::value>, dim3((unsigned)(d->n * a.slices)),
                                  kDistillThreads, Entries::bytes(d->k), static_cast<cudaStream_t>(stream), a));
    return (int)RAFB200_OK;
  });
}

int rafb200_distill_loss_with_dpred(const rafb200_distill* d, const float* dy, int dy_step, float grad_scale, float* loss,
                                    void* dpred, int64_t ld_dpred, void* stream) {
  if (const int rc = check_args(d, "rafb200_distill_loss_with_dpred")) return rc;
  if (d->n == 0) return RAFB200_OK;
  if (const int rc = check_gradient(d, dpred, ld_dpred, "rafb200_distill_loss_with_dpred")) return rc;
  RAFB200_REQUIRE(loss, "rafb200_distill_loss_with_dpred: NULL loss");
  DistillArgs a = device_args(d);
  a.dy = dy;
  a.dy_step = dy_step ? 1 : 0;
  a.grad_scale = grad_scale;
  a.loss = loss;
  a.out = dpred;
  a.ld_out = ld_dpred;
  a.slices = row_slices(d);
  return with_case(d, [&](auto t, auto two) {
    RAFB200_CUDA(launch_cluster(distill_kernel<decltype(t), decltype(two)::value, true>, a.slices, (unsigned)(d->n * a.slices),
                                kDistillThreads, Entries::bytes(d->k), static_cast<cudaStream_t>(stream), a));
    return (int)RAFB200_OK;
  });
}

}  // extern "C"
