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
#include <algorithm>
#include <cmath>

#include "model_io.cuh"

namespace rafb200 {

// Bound: HBM in the sweeps over the logits, as long as an element takes few instructions: at 6.45 TB/s an SM has 22
// issue slots per 32 elements of 2 bytes read and written, and an exponential fills the special-function unit for 8 of
// them.  So two elements are computed by one instruction (f32x2), maxima are taken on the raw pairs, and where the second
// exponential is a small power of the first (T = 2 or 4) it is multiplied out.
constexpr int kDistillUnroll = 4;  // the rests of one to three groups are written out
constexpr int kDistillRing = 2 * kDistillUnroll;  // groups of a thread on their way in: a third batch leaves less L1 (328 -> 338 us)
constexpr int kSweepThreads = 1024;  // of an SM, at least
constexpr int kMaxTeacher = 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// How exp(z - m) follows from exp((z - m) / T): not needed (or T = 1), an exponential of its own, the square (T = 2),
// the fourth power (T = 4).
enum Second { kNone, kOwn, kSquare, kFourth };

struct DistillArgs {
  const void* pred;
  const void* teacher;
  Ids ids;
  Ids labels;       // p == nullptr: none
  const float* dy;  // one weight per row (dy_step 1), one for all (0), or nullptr: 1
  float* loss;
  float4* stats;    // per row: maximum, sum of exponentials at the temperature, the same at one (NaN if not summed up); the fourth is
                    // within a launch the sum of the teacher's weights - 1, which no other launch reads
  void* out;
  int64_t n, v, ld, ld_out, ignore;
  int k, teacher_type, dy_step;
  float c, soft_loss, soft_grad, hard, grad_scale;  // log2(e) / T, alpha T^2, alpha T, 1 - alpha
  int slices_log;   // a row has 2^slices_log blocks
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Two ex2(Two a) { return Two(ex2(a.lo()), ex2(a.hi())); }

// The elements of 16 bytes: their number, pair j of them, and the largest.
template <typename T>
struct Raw {
  static constexpr int kPer = 16 / sizeof(T);
  static __device__ __forceinline__ uint32_t word(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
  static __device__ __forceinline__ Two pair(const uint4& r, int j) {
    if constexpr (sizeof(T) == 4) {
      return Two(__uint_as_float(word(r, 2 * j)), __uint_as_float(word(r, 2 * j + 1)));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return Two(__uint_as_float(word(r, j) << 16), __uint_as_float(word(r, j) & 0xffff0000u));
    } else {
      const uint32_t w = word(r, j);
      __half2 h;
      memcpy(&h, &w, 4);
      const float2 f = __half22float2(h);
      return Two(f.x, f.y);
    }
  }
  // pairwise maxima of the raw words; NaN gives way to numbers (their exponentials carry it on)
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
      using P = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
      P x, y;
      memcpy(&x, &a, 4);
      memcpy(&y, &b, 4);
      x = __hmax2(x, y);
      memcpy(&a, &x, 4);
      return a;
    }
  }
  static __device__ __forceinline__ uint32_t max2(const uint4& r) { return max2(max2(r.x, r.y), max2(r.z, r.w)); }
  static __device__ __forceinline__ float max1(uint32_t w) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    const Two p = pair(make_uint4(w, w, w, w), 0);
    return fmaxf(p.lo(), p.hi());
  }
  static __device__ __forceinline__ uint32_t put(Two p) {  // 16-bit types: a pair rounded into a word
    uint32_t w;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(p.lo(), p.hi());
      memcpy(&w, &h, 4);
    } else {
      const __half2 h = __floats2half2_rn(p.lo(), p.hi());
      memcpy(&w, &h, 4);
    }
    return w;
  }
};

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

// The sums of `x`, relative to its maximum, relative to a maximum that is no smaller.
template <Second S>
__device__ __forceinline__ void rebase(Running& x, float top, float c) {
  if (x.top != -INFINITY) {  // sums over -infinity alone are 0, or NaN, and stay it
    const float d = x.top - top;
    x.soft *= ex2(d * c);
    if (S != kNone) x.hard *= ex2(d * kLog2e);
  }
  x.top = top;
}

// What the loss has not summed up is NaN in the statistics: a gradient that takes it (with other labels or another alpha) is NaN
// rather than one from another sum.
__device__ __forceinline__ float not_summed() { return __int_as_float(0x7fffffff); }
// The sum at one where a single one is kept, at the temperature.
__device__ __forceinline__ float sum_at_one(const DistillArgs& a, float soft) { return a.c == kLog2e ? soft : not_summed(); }

// Copies 16 bytes to shared memory without waiting; a thread waits for all but its last N batches of copies.
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The teacher's entries of a row in shared memory: class (-1: absent), weight p, its logarithm of base 2, student's logit
// there.  Entry k is the label, with weight 0.  Behind them a table of 2^table_log classes, more than there are entries.
struct Entries {
  int* at;
  float* p;
  float* log_p;
  float* z;
  int* table;
  __device__ __forceinline__ Entries(void* smem, int k)
      : at(static_cast<int*>(smem)), p(reinterpret_cast<float*>(at + k + 1)), log_p(p + k + 1), z(log_p + k + 1), table(reinterpret_cast<int*>(z + k + 1)) {}
  static __host__ __device__ __forceinline__ int table_log(int k) {
    int log = 5;
    while (1 << log < k + k / 4 + 2) ++log;
    return log;
  }
  static __host__ __device__ __forceinline__ size_t bytes(int k) { return (size_t)(k + 1) * 16 + ((size_t)4 << table_log(k)); }
};

// softmax over the present entries, whose logits p holds before; returns the sum of the weights, 1 or 0 (or NaN).  One warp.
__device__ __forceinline__ float weigh(const Entries& e, int k, float c) {
  const int lane = threadIdx.x & 31;
  float top = -INFINITY;
  for (int i = lane; i < k; i += 32)
    if (e.at[i] >= 0) top = fmaxf(top, e.p[i]);
#pragma unroll
  for (int s = 16; s; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
  const float base = base_of(top);
  float sum = 0.f;
  for (int i = lane; i < k; i += 32)
    if (e.at[i] >= 0) sum += power(e.p[i], base, c);
  sum = warp_sum(sum);
  const bool some = sum != 0.f;  // false: no teacher, or all of it at -infinity
  const float inv = some ? 1.f / sum : 0.f, log2_sum = log2f(sum);
  for (int i = lane; i < k; i += 32) {
    const float t = (e.p[i] - base) * c;
    e.log_p[i] = t - log2_sum;
    e.p[i] = e.at[i] >= 0 && some ? ex2(t) * inv : 0.f;
  }
  __syncwarp();
  return isnan(sum) ? sum : some ? 1.f : 0.f;
}

// sum p (log p - log q).  One warp.
__device__ __forceinline__ float divergence(const Entries& e, int k, float c, float base, float log2_soft) {
  float part = 0.f;
  for (int i = threadIdx.x & 31; i < k; i += 32)
    if (!(e.p[i] == 0.f)) part = fmaf(e.p[i], e.log_p[i] - ((e.z[i] - base) * c - log2_soft), part);
  return warp_sum(part) * kLn2;
}

// Fills in the entries of a row.  One warp.
template <typename T>
__device__ __forceinline__ void load_entries(const DistillArgs& a, const Entries& e, int64_t row, const T* z, int64_t label) {
  for (int i = threadIdx.x & 31; i <= a.k; i += 32) {
    const int64_t j = i < a.k ? a.ids[row * a.k + i] : label;
    const bool in = (uint64_t)j < (uint64_t)a.v;
    e.at[i] = in ? (int)j : -1;
    e.p[i] = i < a.k ? load_teacher(a, row * a.k + i) : 0.f;
    e.z[i] = in ? Elem<T>::to_f32(z[j]) : 0.f;
  }
  __syncwarp();
}

// What a gradient is made of: dz = soft * 2^((z - base) c) + hard * 2^((z - base) log2e), at the entries minus
// teach * (sum of p), and minus hit at the label.
struct Coefficients {
  float c, base, soft, hard, teach, hit;
  template <Second S>
  __device__ __forceinline__ float at(float z) const {
    const float e = power(z, base, c);
    if (S == kNone) return soft * e;
    if (S == kOwn) return fmaf(hard, power(z, base, kLog2e), soft * e);
    const float f = S == kFourth ? e * e * e : e;
    return fmaf(hard, f, soft) * e;
  }
  template <Second S>
  __device__ __forceinline__ Two at(Two z) const {
    const Two x = z + Two(-base, -base), e = ex2(x * Two(c, c)), w(soft, soft);
    if (S == kNone) return w * e;
    if (S == kOwn) return fma2(Two(hard, hard), ex2(x * Two(kLog2e, kLog2e)), w * e);
    const Two f = S == kFourth ? e * e * e : e;
    return fma2(Two(hard, hard), f, w) * e;
  }
};

template <Second S>
__device__ __forceinline__ Coefficients coefficients(const DistillArgs& a, float weight, float4 stats, bool labels) {
  const float w = weight * a.grad_scale;
  Coefficients co;
  co.c = a.c;
  co.base = base_of(stats.x);
  co.teach = w * a.soft_grad;
  co.hit = labels ? w * a.hard : 0.f;
  // a term that the row does not have is 0, whatever its sums are: those of nothing but -infinity are 0 themselves
  const bool taught = stats.w != -1.f, hit = labels && a.hard != 0.f;
  co.soft = taught ? co.teach * (stats.w + 1.f) / stats.y : 0.f;
  co.hard = hit ? co.hit / stats.z : 0.f;
  if (S == kNone) {  // one exponential serves both terms, or there is one term only
    co.soft += hit ? co.hit / stats.y : 0.f;
    co.hard = 0.f;
  }
  return co;
}

// The groups of a slice on their way through shared memory, kDistillRing places a thread that go round: each is read by the
// thread alone that asked for it, so no registers are bound by what is on its way, and no barrier is needed.
template <typename T, int NT>
struct Stream {
  static constexpr int kAhead = kDistillRing / kDistillUnroll, kStep = kDistillUnroll * NT, kPlaces = kDistillRing * NT;
  const uint4* source;
  uint4 *first, *place;
  int groups;
  __device__ __forceinline__ Stream(const Slice<T>& s, const T* z, uint4* image)
      : source(reinterpret_cast<const uint4*>(z + s.at)), first(image + threadIdx.x), place(first), groups(s.groups) {}
  __device__ __forceinline__ void ask(int i, uint4* to) {  // a batch, this thread's groups from i on
#pragma unroll
    for (int u = 0; u < kDistillUnroll; ++u)
      if (i + u * NT < groups) copy_async(to + u * NT, source + i + u * NT);
    copy_commit();
  }
  __device__ __forceinline__ void begin() {
#pragma unroll
    for (int b = 0; b < kAhead; ++b) ask(threadIdx.x + b * kStep, first + b * kStep);
  }
  // use(i, where group i lies, number of this thread's groups from i on) for every batch
  template <typename Use>
  __device__ __forceinline__ void run(const Use& use) {
    for (int i = threadIdx.x; i < groups; i += kStep) {
      copy_wait<kAhead - 1>();
      use(i, place, (groups - i + NT - 1) / NT);
      ask(i + kAhead * kStep, place);
      place = place == first + (kAhead - 1) * kStep ? first : place + kStep;
    }
    copy_wait<0>();
    place = first;
  }
};

template <typename T, Second S>
__device__ __forceinline__ uint4 gradient_of(const uint4& raw, const Coefficients& co) {
  if constexpr (sizeof(T) == 4) {
    const Two a = co.at<S>(Raw<T>::pair(raw, 0)), b = co.at<S>(Raw<T>::pair(raw, 1));
    return make_uint4(__float_as_uint(a.lo()), __float_as_uint(a.hi()), __float_as_uint(b.lo()), __float_as_uint(b.hi()));
  } else {
    return make_uint4(Raw<T>::put(co.at<S>(Raw<T>::pair(raw, 0))), Raw<T>::put(co.at<S>(Raw<T>::pair(raw, 1))),
                      Raw<T>::put(co.at<S>(Raw<T>::pair(raw, 2))), Raw<T>::put(co.at<S>(Raw<T>::pair(raw, 3))));
  }
}

// The gradient of COUNT groups, NT apart; `from` holds the bytes of the first.
template <typename T, Second S, int NT, int Q, int COUNT>
__device__ __forceinline__ void write_groups(const char* from, uint32_t bits, uint4* to, const Coefficients& co) {
  uint4 raw[COUNT];
#pragma unroll
  for (int u = 0; u < COUNT; ++u) raw[u] = load_shifted<Q>(from + u * NT * 16, bits);
#pragma unroll
  for (int u = 0; u < COUNT; ++u) to[u * NT] = gradient_of<T, S>(raw[u], co);
}
// A batch of them, `left` from the first on: the rest together, for one wait for memory.
template <typename T, Second S, int NT, int Q>
__device__ __forceinline__ void write_batch(const char* from, uint32_t bits, uint4* to, int left, const Coefficients& co) {
  if (left >= kDistillUnroll) write_groups<T, S, NT, Q, kDistillUnroll>(from, bits, to, co);
  else if (left == 1) write_groups<T, S, NT, Q, 1>(from, bits, to, co);
  else if (left == 2) write_groups<T, S, NT, Q, 2>(from, bits, to, co);
  else if (left == 3) write_groups<T, S, NT, Q, 3>(from, bits, to, co);
}

// The gradient of a slice of z.  `edge` is this thread's element outside the groups.
template <typename T, Second S, int NT, int Q>
__device__ __forceinline__ void write_batches(const Slice<T>& s, const T* z, T* out, const Coefficients& co, int tid) {
  const char* from = reinterpret_cast<const char*>(z + s.at);
  uint4* to = reinterpret_cast<uint4*>(out + s.at);
  const uint32_t bits = (reinterpret_cast<uintptr_t>(from) & 3) * 8;
  for (int i = tid; i < s.groups; i += kDistillUnroll * NT)
    write_batch<T, S, NT, Q>(from + (int64_t)i * 16, bits, to + i, (s.groups - i + NT - 1) / NT, co);
}
// The same where the gradient's groups are not those of z.
template <typename T, Second S, int NT>
__device__ __forceinline__ void write_shifted(const Slice<T>& in, const T* z, T* out, const Coefficients& co, int tid) {
  const Slice<T> s = in.aligned_at(out);
  switch ((reinterpret_cast<uintptr_t>(z + s.at) & 15) >> 2) {
    case 0: write_batches<T, S, NT, 0>(s, z, out, co, tid); break;
    case 1: write_batches<T, S, NT, 1>(s, z, out, co, tid); break;
    case 2: write_batches<T, S, NT, 2>(s, z, out, co, tid); break;
    default: write_batches<T, S, NT, 3>(s, z, out, co, tid); break;
  }
  if (tid < s.edges()) {
    const int j = s.edge_at(tid);
    out[j] = Elem<T>::from_f32(co.at<S>(Elem<T>::to_f32(z[j])));
  }
}
// By the stream, which has begun where z and out are alike, or by loads.
template <typename T, Second S, int NT, bool STREAMED>
__device__ __forceinline__ void write_slice(const Slice<T>& in, const T* z, float edge, T* out, const Coefficients& co, Stream<T, NT>& stream) {
  if (!alike(z, out)) {
    write_shifted<T, S, NT>(in, z, out, co, threadIdx.x);
    return;
  }
  if constexpr (STREAMED) {
    uint4* to = reinterpret_cast<uint4*>(out + in.at);
    stream.run([&](int i, const uint4* place, int left) {
      write_batch<T, S, NT, -1>(reinterpret_cast<const char*>(place), 0, to + i, left, co);
    });
  } else {
    write_batches<T, S, NT, -1>(in, z, out, co, threadIdx.x);
  }
  if ((int)threadIdx.x < in.edges()) out[in.edge_at(threadIdx.x)] = Elem<T>::from_f32(co.at<S>(edge));
}

// Whether it is known that no class is named twice: each is put into the table, whose places are tried one after the other.  For
// short lists write_entries() compares sooner than the table is filled (4096 rows of 1000 with 32 entries: 13.9 against
// 15.9 us for loss and gradient), for 64 entries it does not (8192 rows of 50257: 355 against 340 us).  One warp.
__device__ __forceinline__ bool all_different(const Entries& e, int k) {
  if (k < 64) return false;
  const int lane = threadIdx.x & 31, log = Entries::table_log(k), places = 1 << log;
  for (int i = lane; i < places; i += 32) e.table[i] = -1;
  __syncwarp();
  bool again = false;
  for (int i = lane; i <= k; i += 32) {
    const int j = e.at[i];
    if (j < 0) continue;
    uint32_t at = (uint32_t)j * 0x9E3779B1u >> (32 - log);
    for (int tries = 0; tries < places; ++tries, at = (at + 1) & (places - 1)) {
      const int old = atomicCAS(&e.table[at], -1, j);
      again |= old == j;
      if (old == -1 || old == j) break;
    }
  }
  return !__any_sync(0xffffffffu, again);
}

// The elements that the teacher or the label names, once each however often they are named.  One warp.
template <typename T, Second S>
__device__ __forceinline__ void write_entries(const DistillArgs& a, const Entries& e, const Slice<T>& s, T* out, const Coefficients& co,
                                              bool different) {
  for (int i = threadIdx.x & 31; i <= a.k; i += 32) {
    const int j = e.at[i];
    if (j < 0 || !s.owns(j)) continue;
    float p = e.p[i];
    bool hit = i == a.k, again = false;
    if (!different) {
      for (int q = 0; q <= a.k; ++q) {
        if (e.at[q] != j || q == i) continue;
        again |= q < i;
        p += e.p[q];
        hit |= q == a.k;
      }
    }
    if (again) continue;
    float g = co.at<S>(e.z[i]) - co.teach * p;
    if (hit) g -= co.hit;
    out[j] = Elem<T>::from_f32(g);
  }
}

template <typename T, int NT>
__device__ __forceinline__ void zero_slice(const Slice<T>& s, T* out, int tid) {
  uint4* to = reinterpret_cast<uint4*>(out + s.at);
  for (int i = tid; i < s.groups; i += NT) to[i] = make_uint4(0, 0, 0, 0);
  if (tid < s.edges()) out[s.edge_at(tid)] = Elem<T>::from_f32(0.f);
}

// Running maximum and sums of a thread's groups.
template <typename T, Second S>
struct Sweep {
  Running run{-INFINITY, 0.f, 0.f};
  Two soft{0.f, 0.f}, hard{0.f, 0.f};

  template <int COUNT>
  __device__ __forceinline__ void add(const uint4* from, int step, float c) {
    uint4 raw[COUNT];
#pragma unroll
    for (int u = 0; u < COUNT; ++u) raw[u] = from[u * step];
    uint32_t most = Raw<T>::max2(raw[0]);
#pragma unroll
    for (int u = 1; u < COUNT; ++u) most = Raw<T>::max2(most, Raw<T>::max2(raw[u]));
    const float top = fmaxf(run.top, Raw<T>::max1(most)), base = base_of(top);
    if (top != run.top) {
      const float d = run.top - top;  // -infinity at first: the sums are 0 and stay it, or NaN
      const float fs = run.top == -INFINITY ? 1.f : ex2(d * c), fh = run.top == -INFINITY ? 1.f : ex2(d * kLog2e);
      soft = soft * Two(fs, fs);
      if (S != kNone) hard = hard * Two(fh, fh);
      run.top = top;
    }
#pragma unroll
    for (int u = 0; u < COUNT; ++u) terms(raw[u], base, c);
  }
  // adds the exponentials of a group
  __device__ __forceinline__ void terms(const uint4& raw, float base, float c) {
    const Two nb(-base, -base), c2(c, c);
#pragma unroll
    for (int j = 0; j < Raw<T>::kPer / 2; ++j) {
      const Two x = Raw<T>::pair(raw, j) + nb, p = ex2(x * c2);
      soft = soft + p;
      if (S == kOwn) hard = hard + ex2(x * Two(kLog2e, kLog2e));
      if (S == kSquare) hard = fma2(p, p, hard);
      if (S == kFourth) hard = fma2(p * p, p * p, hard);
    }
  }
  // The groups of a batch that exist, `left` of them from the first on.
  __device__ __forceinline__ void batch(const uint4* from, int step, int left, float c) {
    if (left >= kDistillUnroll) add<kDistillUnroll>(from, step, c);
    else if (left == 1) add<1>(from, step, c);
    else if (left == 2) add<2>(from, step, c);
    else if (left == 3) add<3>(from, step, c);
  }
  __device__ __forceinline__ void edge(float z, float c) {
    rebase<S>(run, fmaxf(run.top, z), c);
    const float base = base_of(run.top);
    run.soft += power(z, base, c);
    if (S != kNone) run.hard += power(z, base, kLog2e);
  }
  __device__ __forceinline__ void finish() {
    run.soft = soft.lo() + soft.hi();
    run.hard = hard.lo() + hard.hi();
  }
};

// What the warps of a block, and the blocks of a cluster, tell one another about a row.
template <int WARPS>
struct Exchange {
  float tops[WARPS];
  float2 sums[WARPS];
  Running part[8];  // of the cluster's blocks
  float some;       // sum of the teacher's weights - 1
  float4 stats;
};

// A block is NT threads that sweep the logits, and a warp that sees to the teacher's entries meanwhile.
template <int N>
__device__ __forceinline__ void bar_sync(int id) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ void bar_arrive(int id) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(N) : "memory");
}
enum { kSweepers = 1, kWeighed = 2, kWritten = 3 };  // barriers

// Joins the sweeping threads' sums of a row: the block's maximum first and then sums relative to it.
template <Second S, int NT>
__device__ __forceinline__ float4 join(Exchange<NT / 32>& x, Running run, const DistillArgs& a) {
  constexpr int kWarps = NT / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = run.top;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) x.tops[warp] = top;
  bar_sync<NT>(kSweepers);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, x.tops[w]);
  rebase<S>(run, top, a.c);
  run.soft = warp_sum(run.soft);
  if (S != kNone) run.hard = warp_sum(run.hard);
  if (lane == 0) x.sums[warp] = make_float2(run.soft, run.hard);
  bar_sync<NT + 32>(kWeighed);
  run = Running{top, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    run.soft += x.sums[w].x;
    run.hard += x.sums[w].y;
  }
  if (a.slices_log) {
    cluster_wait();  // every block of the cluster runs
    if (threadIdx.x < 1u << a.slices_log) {
      Running* to = &x.part[blockIdx.x & ((1 << a.slices_log) - 1)];
      cluster_store(&to->top, threadIdx.x, __float_as_uint(run.top));
      cluster_store(&to->soft, threadIdx.x, __float_as_uint(run.soft));
      cluster_store(&to->hard, threadIdx.x, __float_as_uint(run.hard));
    }
    cluster_sync();  // nothing of another block is looked at from here on
    for (int r = 0; r >> a.slices_log == 0; ++r) top = fmaxf(top, x.part[r].top);
    run = Running{top, 0.f, 0.f};
    for (int r = 0; r >> a.slices_log == 0; ++r) {
      Running part = x.part[r];
      rebase<S>(part, top, a.c);
      run.soft += part.soft;
      run.hard += part.hard;
    }
  }
  return make_float4(run.top, run.soft, S != kNone ? run.hard : sum_at_one(a, run.soft), x.some);
}

// The loss of a row, by one warp.
__device__ __forceinline__ void put_loss(const DistillArgs& a, const Entries& e, int64_t row, const float4& stats, bool labels) {
  const float base = base_of(stats.x), kl = divergence(e, a.k, a.c, base, log2f(stats.y));
  if ((threadIdx.x & 31) != 0) return;
  float loss = a.soft_loss > 0.f ? a.soft_loss * kl : 0.f;  // a term without weight counts nothing, infinite or not
  if (labels && a.hard > 0.f) loss += a.hard * kLn2 * (log2f(stats.z) - (e.z[a.k] - base) * kLog2e);
  a.loss[row] = loss;
  if (a.stats) a.stats[row] = stats;
}

__device__ __forceinline__ bool left_out(const DistillArgs& a, int64_t label) {
  return label == a.ignore || (uint64_t)label >= (uint64_t)a.v;
}

template <typename T, int NT, bool GRAD>
__device__ __forceinline__ void leave_out(const DistillArgs& a, int64_t row, int slice, int tid) {
  if (slice == 0 && tid == 0) {
    a.loss[row] = 0.f;
    if (a.stats) a.stats[row] = make_float4(not_summed(), not_summed(), not_summed(), not_summed());
  }
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  if (GRAD) zero_slice<T, NT>(Slice<T>(out, (int)a.v, slice, a.slices_log), out, tid);
}

// Loss, and with GRAD the gradient, of a row by a cluster of 2^slices_log blocks: one pass with a running maximum and its
// sums, joined over threads, warps and blocks.
// GRAD reads the logits a second time, from the L2: the launch sees to it that it holds what the resident blocks work on.
// 8192 rows of 50257 (bf16, T = 2, labels), loss and gradient: 316 us (5.2 TB/s of what has to be read and written), with
// gradient rows that lie otherwise than the logits do.  Slices kept in shared memory instead, which
// leave room for two blocks an SM: 450 us, 590 us with the next row on its way meanwhile - 16 warps an SM are too few for
// the arithmetic.  The loss alone, 4096 rows of 30522: 55 us (4.6 TB/s), fp32 6.0 TB/s: 16-bit logits give every byte twice the
// arithmetic.
template <typename T, Second S, bool GRAD, int NT>
__global__ void __launch_bounds__(NT + 32, kSweepThreads / NT) distill_kernel(DistillArgs a) {
  extern __shared__ uint4 image[];
  __shared__ Exchange<NT / 32> exchange;
  grid_dependency_trigger();
  grid_dependency_wait();
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x >> a.slices_log;
  const int slice = blockIdx.x & ((1 << a.slices_log) - 1);
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && left_out(a, label)) {  // the same for every block of the cluster
    if (tid < NT) leave_out<T, NT, GRAD>(a, row, slice, tid);
    return;
  }
  if (a.slices_log) cluster_arrive_relaxed();
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const Slice<T> s(z, (int)a.v, slice, a.slices_log);

  if (tid >= NT) {  // the warp of the entries
    const Entries e(image + Stream<T, NT>::kPlaces, a.k);
    const float weight = GRAD && a.dy ? a.dy[row * a.dy_step] : 1.f;
    load_entries(a, e, row, z, label);
    const float some = weigh(e, a.k, a.c);
    if (tid == NT) exchange.some = some - 1.f;
    __syncwarp();
    bar_arrive<NT + 32>(kWeighed);
    if (a.slices_log) {
      cluster_wait();
      cluster_sync();
    }
    const bool different = GRAD && all_different(e, a.k);
    bar_sync<NT + 32>(kWritten);
    const float4 stats = exchange.stats;
    if (GRAD) write_entries<T, S>(a, e, s, out, coefficients<S>(a, weight, stats, labels), different);
    if (slice == 0) put_loss(a, e, row, stats, labels);
    return;
  }

  Stream<T, NT> stream(s, z, image);
  stream.begin();
  const float edge = tid < s.edges() ? Elem<T>::to_f32(z[s.edge_at(tid)]) : 0.f;
  const float weight = GRAD && a.dy ? a.dy[row * a.dy_step] : 1.f;
  Sweep<T, S> sweep;
  stream.run([&](int, const uint4* place, int left) { sweep.batch(place, NT, left, a.c); });
  // 32-bit logits stream a second time (4096 rows of 50304: 5.5 instead of 5.0 TB/s); 16-bit ones do better with loads (8192
  // rows of 50257 in bf16: 327 instead of 340 us)
  constexpr bool kStreamed = GRAD && sizeof(T) == 4;
  if (kStreamed && alike(z, out)) stream.begin();
  sweep.finish();
  if (tid < s.edges()) sweep.edge(edge, a.c);
  const float4 stats = join<S, NT>(exchange, sweep.run, a);
  if (tid == 0) exchange.stats = stats;
  if (GRAD) write_slice<T, S, NT, kStreamed>(s, z, edge, out, coefficients<S>(a, weight, stats, labels), stream);
  bar_arrive<NT + 32>(kWritten);
}

// The gradient from the maximum and the sums that the forward pass has left.  What the teacher's weights sum to (0 for a row
// without one) is taken from its entries, which are at hand.
constexpr int kDpredThreads = 128;
template <typename T, Second S>
__global__ void __launch_bounds__(kDpredThreads + 32, 6) distill_dpred_kernel(DistillArgs a) {
  constexpr int NT = kDpredThreads;
  extern __shared__ uint4 image[];
  grid_dependency_trigger();
  grid_dependency_wait();
  const int64_t row = blockIdx.x >> a.slices_log;
  const int slice = blockIdx.x & ((1 << a.slices_log) - 1), tid = threadIdx.x;
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && left_out(a, label)) {
    if (tid < NT) zero_slice<T, NT>(Slice<T>(out, (int)a.v, slice, a.slices_log), out, tid);
    return;
  }
  __shared__ float some;
  const Slice<T> s(z, (int)a.v, slice, a.slices_log);
  float4 stats = a.stats[row];
  const float weight = a.dy ? a.dy[row * a.dy_step] : 1.f;
  if (tid < NT) {
    const float edge = tid < s.edges() ? Elem<T>::to_f32(z[s.edge_at(tid)]) : 0.f;
    Stream<T, NT> stream(s, z, image);
    if (alike(z, out)) stream.begin();
    bar_sync<NT + 32>(kWeighed);  // out may be pred: the entries of this slice are read (those of others are not used here)
    stats.w = some;
    write_slice<T, S, NT, true>(s, z, edge, out, coefficients<S>(a, weight, stats, labels), stream);
    bar_arrive<NT + 32>(kWritten);
    return;
  }
  const Entries e(image + Stream<T, NT>::kPlaces, a.k);
  load_entries(a, e, row, z, label);
  stats.w = weigh(e, a.k, a.c) - 1.f;
  if (tid == NT) some = stats.w;
  __syncwarp();
  bar_arrive<NT + 32>(kWeighed);
  bool mine = false;
  for (int i = tid - NT; i <= a.k; i += 32) mine |= e.at[i] >= 0 && s.owns(e.at[i]);
  mine = __any_sync(0xffffffffu, mine);
  const bool different = mine && all_different(e, a.k);
  bar_sync<NT + 32>(kWritten);
  if (mine) write_entries<T, S>(a, e, s, out, coefficients<S>(a, weight, stats, labels), different);
}

// Short rows: a warp takes a row, which its registers hold from the first look to the gradient, and sees to the row's
// entries too.  Bound by the instructions and the latency of a row's entries, for which an SM has 24 rows on their way.
// Blocks that share a row took longer at every length that registers hold: 4096 rows of 1000 (bf16, 32 entries,
// T = 2, labels), loss 14.3 -> 8.0 us, gradient 21.5 -> 11.5 us, both 25 -> 13.9 us; rows of 2040: 14.7 -> 9.0, 21.9 -> 12.7,
// 26.6 -> 15.4 us.
constexpr int kShortGroups = 8;  // of a lane
constexpr int kShortWarps = 4;
enum Part { kLoss, kDpred, kBoth };
template <typename T, Second S, Part P>
__global__ void __launch_bounds__(32 * kShortWarps, 6) distill_short_kernel(DistillArgs a) {
  extern __shared__ uint4 image[];
  grid_dependency_trigger();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kShortWarps + warp;
  if (row >= a.n) return;
  const Entries e(reinterpret_cast<char*>(image) + warp * Entries::bytes(a.k), a.k);
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const Slice<T> s(z, (int)a.v, 0, 0);
  const uint4* source = reinterpret_cast<const uint4*>(z + s.at) + lane;
  const uint32_t low = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -infinity
  uint4 raw[kShortGroups];
#pragma unroll
  for (int u = 0; u < kShortGroups; ++u) {
    raw[u] = make_uint4(low, low, low, low);
    if (u * 32 + lane < s.groups) raw[u] = source[u * 32];
  }
  const float edge = lane < s.edges() ? Elem<T>::to_f32(z[s.edge_at(lane)]) : -INFINITY;
  const float weight = P != kLoss && a.dy ? a.dy[row * a.dy_step] : 1.f;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  float4 stats = P == kDpred ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
  load_entries(a, e, row, z, label);
  if (labels && left_out(a, label)) {
    if (P == kDpred) zero_slice<T, 32>(Slice<T>(out, (int)a.v, 0, 0), out, lane);
    else leave_out<T, 32, P == kBoth>(a, row, 0, lane);
    return;
  }
  const float some = weigh(e, a.k, a.c) - 1.f;
  if (P != kDpred) {
    uint32_t most = Raw<T>::max2(raw[0]);
#pragma unroll
    for (int u = 1; u < kShortGroups; ++u)
      if (u * 32 < s.groups) most = Raw<T>::max2(most, Raw<T>::max2(raw[u]));
    float top = fmaxf(edge, Raw<T>::max1(most));
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float base = base_of(top);
    Sweep<T, S> sweep;
#pragma unroll
    for (int u = 0; u < kShortGroups; ++u)
      if (u * 32 < s.groups) sweep.terms(raw[u], base, a.c);
    sweep.finish();
    float soft = sweep.run.soft, hard = sweep.run.hard;
    if (lane < s.edges()) {
      soft += power(edge, base, a.c);
      if (S != kNone) hard += power(edge, base, kLog2e);
    }
    soft = warp_sum(soft);
    if (S != kNone) hard = warp_sum(hard);
    stats = make_float4(top, soft, S != kNone ? hard : sum_at_one(a, soft), 0.f);
  }
  stats.w = some;
  if (P != kDpred) put_loss(a, e, row, stats, labels);
  if (P == kLoss) return;
  const Coefficients co = coefficients<S>(a, weight, stats, labels);
  if (alike(z, out)) {
    uint4* to = reinterpret_cast<uint4*>(out + s.at) + lane;
#pragma unroll
    for (int u = 0; u < kShortGroups; ++u)
      if (u * 32 + lane < s.groups) to[u * 32] = gradient_of<T, S>(raw[u], co);
    if (lane < s.edges()) out[s.edge_at(lane)] = Elem<T>::from_f32(co.at<S>(edge));
  } else {
    write_shifted<T, S, 32>(s, z, out, co, lane);
  }
  const bool different = all_different(e, a.k);
  __syncwarp();  // what other lanes have written is overwritten
  write_entries<T, S>(a, e, s, out, co, different);
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
  a.k = d->alpha == 0.0 ? 0 : d->k;  // a teacher without weight is not looked at: 0 times its NaN would be NaN
  a.teacher_type = d->teacher_dtype;
  a.c = (float)(M_LOG2E / d->temperature);
  a.soft_loss = (float)(d->alpha * d->temperature * d->temperature);
  a.soft_grad = (float)(d->alpha * d->temperature);
  a.hard = (float)(1.0 - d->alpha);
  return a;
}

static Second second_of(const rafb200_distill* d) {
  if (!d->labels || d->alpha == 1.0 || d->temperature == 1.0) return kNone;  // one term, or both at one temperature
  return d->temperature == 2.0 ? kSquare : d->temperature == 4.0 ? kFourth : kOwn;
}

constexpr int64_t kMostGroups = 110 * 1024 / 16;
static int64_t row_groups(const rafb200_distill* d) { return d->v * dtype_size(d->pred_dtype) / 16; }

template <typename T, Second S, bool GRAD, int NT>
static int launch_rows(const rafb200_distill* d, DistillArgs a, cudaStream_t s) {
  const size_t ring = (size_t)kDistillRing * NT * 16, smem = ring + Entries::bytes(d->k);
  // few rows are cut until every SM has work, while a thread keeps a group
  while (a.slices_log < 3 && (d->n << (a.slices_log + 1)) <= 148 * 2 && row_groups(d) >> (a.slices_log + 1) >= NT) ++a.slices_log;
  // what the resident blocks hold of the logits, to be read again, is to stay in the L2
  while (GRAD && a.slices_log < 3 && row_groups(d) >> a.slices_log > kMostGroups) ++a.slices_log;
  if (const int rc = allow_smem<distill_kernel<T, S, GRAD, NT>>(smem, ring + Entries::bytes(kMaxTeacher))) return rc;
  RAFB200_CUDA(launch_cluster(distill_kernel<T, S, GRAD, NT>, 1u << a.slices_log, (unsigned)(d->n << a.slices_log), NT + 32, smem, s, a));
  return RAFB200_OK;
}

// Rows of which a lane holds at most kShortGroups groups.
static bool short_rows(const rafb200_distill* d) { return row_groups(d) <= 32 * kShortGroups; }

template <typename T, Second S, Part P>
static int launch_short(const rafb200_distill* d, const DistillArgs& a, cudaStream_t s) {
  const size_t smem = kShortWarps * Entries::bytes(d->k);
  if (const int rc = allow_smem<distill_short_kernel<T, S, P>>(smem, kShortWarps * Entries::bytes(kMaxTeacher))) return rc;
  RAFB200_CUDA(launch_dependent(distill_short_kernel<T, S, P>, dim3((unsigned)((d->n + kShortWarps - 1) / kShortWarps)), 32 * kShortWarps, smem, s, a));
  return RAFB200_OK;
}

template <typename F>
static int with_case(const rafb200_distill* d, const F& f) {
  return with_type(d->pred_dtype, [&](auto t) {
    switch (second_of(d)) {
      case kNone: return f(t, std::integral_constant<Second, kNone>{});
      case kOwn: return f(t, std::integral_constant<Second, kOwn>{});
      case kSquare: return f(t, std::integral_constant<Second, kSquare>{});
      default: return f(t, std::integral_constant<Second, kFourth>{});
    }
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
  return with_case(d, [&](auto t, auto second) {
    if (short_rows(d)) return launch_short<decltype(t), decltype(second)::value, kLoss>(d, a, static_cast<cudaStream_t>(stream));
    // Blocks of 128 threads and of 256, 4096 rows, the loss alone: of 312 groups 18 and 29 us, of 2048 41 and 43, of 3000 and 3815 (16-bit)
    // 53 and 49, 59 and 59, of 4096 (fp32) 66 and 57, of 5000 78 and 70, of 10000 129 and 117 us.  300 rows take the same within 2 us
    // up to 3815 groups, then 14 and 12 us (5000), 21 and 16 us (10000).
    if (row_groups(d) >= 4096) return launch_rows<decltype(t), decltype(second)::value, false, 256>(d, a, static_cast<cudaStream_t>(stream));
    return launch_rows<decltype(t), decltype(second)::value, false, 128>(d, a, static_cast<cudaStream_t>(stream));
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
  // few rows are cut until every SM has its six blocks: blocks beyond that cost more than they even out (777 rows of 50257
  // in fp16: 37 us whole, 45 us in eight parts; 100 rows: 20 us whole, 12 us in eight)
  while (a.slices_log < 6 && d->n << (a.slices_log + 1) <= 148 * 6 && row_groups(d) >> (a.slices_log + 1) >= kDpredThreads * kDistillUnroll)
    ++a.slices_log;
  return with_case(d, [&](auto t, auto second) {
    using T = decltype(t);
    constexpr Second S = decltype(second)::value;
    if (short_rows(d)) return launch_short<T, S, kDpred>(d, a, static_cast<cudaStream_t>(stream));
    const size_t ring = Stream<T, kDpredThreads>::kPlaces * 16, smem = ring + Entries::bytes(d->k);
    if (const int rc = allow_smem<distill_dpred_kernel<T, S>>(smem, ring + Entries::bytes(kMaxTeacher))) return rc;
    RAFB200_CUDA(launch_dependent(distill_dpred_kernel<T, S>, dim3((unsigned)(d->n << a.slices_log)), kDpredThreads + 32, smem,
                                  static_cast<cudaStream_t>(stream), a));
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
  return with_case(d, [&](auto t, auto second) {
    if (short_rows(d)) return launch_short<decltype(t), decltype(second)::value, kBoth>(d, a, static_cast<cudaStream_t>(stream));
    // Blocks of 128 threads and of 256, 4096 rows: of 1125 groups 45 and 57 us, of 2048 (16-bit) 64 and 70, of 2250 (fp32) 72 and 70, of
    // 3000 90 and 88, of 3815 119 and 107, of 6282 207 and 168 us.  Fewer rows at a time leave the second look at them to the L2.
    if (row_groups(d) >= 2048) return launch_rows<decltype(t), decltype(second)::value, true, 256>(d, a, static_cast<cudaStream_t>(stream));
    return launch_rows<decltype(t), decltype(second)::value, true, 128>(d, a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
