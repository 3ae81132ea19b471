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

// Bound: HBM in the sweeps over the logits, as long as an element takes few instructions: at 6.45 TB/s an SM has 22
// issue slots per 32 elements of 2 bytes read and written, and an exponential fills the special-function unit for 8 of
// them.  So two elements are computed by one instruction (f32x2), maxima are taken on the raw pairs, and where the second
// exponential is a small power of the first (T = 2 or 4) it is multiplied out.
constexpr int kDistillThreads = 128;
constexpr int kDistillWarps = kDistillThreads / 32;
constexpr int kDistillUnroll = 4;
constexpr int kDistillBlocks = 8;  // resident blocks of an SM: 64 registers a thread
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
  float4* stats;    // per row: maximum, sum of exponentials at the temperature, the same at one, sum of the teacher's weights - 1
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

// Two fp32 numbers in a register pair.
struct Two {
  uint64_t r;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ float lo() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
    return a;
  }
  __device__ __forceinline__ float hi() const {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
    return b;
  }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two c;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(c.r) : "l"(a.r), "l"(b.r));
  return c;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two c;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(c.r) : "l"(a.r), "l"(b.r));
  return c;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two d) {
  Two c;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(c.r) : "l"(a.r), "l"(b.r), "l"(d.r));
  return c;
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

// A block's part of a row: groups [from, to) of 16 bytes of the part that is aligned at `p`; the elements in front of
// that part are the first block's, those behind it the last one's.  With `trim` the first and the last group
// count to those.
template <typename T>
struct Slice {
  static constexpr int kPer = Raw<T>::kPer;
  int head, from, to, body;  // elements in front; groups; first element behind
  int edge;                  // elements of this block outside the groups: thread i < edge takes edge_at(i)
  int first;                 // of them in front

  __device__ __forceinline__ Slice(const T* p, int v, int slice, int slices_log, bool trim) {
    head = min((int)((-(intptr_t)p & 15) / sizeof(T)), v);
    int groups = (v - head) / kPer;
    if (trim && groups > 0) {
      head += kPer;
      groups = max(groups - 2, 0);
    }
    const int each = (groups + (1 << slices_log) - 1) >> slices_log;
    from = min(slice * each, groups);
    to = min(from + each, groups);
    body = head + groups * kPer;
    first = slice == 0 ? head : 0;
    edge = first + (slice + 1 == 1 << slices_log ? v - body : 0);
  }
  __device__ __forceinline__ int edge_at(int i) const { return i < first ? i : body + (i - first); }
  __device__ __forceinline__ bool owns(int j, bool first_slice, bool last_slice) const {
    if (j < head) return first_slice;
    if (j >= body) return last_slice;
    const int g = (j - head) / kPer;
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

// softmax over the present entries; the sum of the weights (1 or 0), and with `kl` sum p (log p - log q).  One warp.
__device__ __forceinline__ float weigh(const Entries& e, int k, float c, float base, float log2_soft, float* kl) {
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
    if (kl && !(w == 0.f)) part = fmaf(w, (t - log2_sum) - ((e.z[i] - base) * c - log2_soft), part);  // log2 p - log2 q
    e.p[i] = w;
  }
  if (kl) *kl = warp_sum(part) * kLn2;
  return isnan(sum) ? sum : some ? 1.f : 0.f;
}

// A thread's first entry is asked for before the logits are swept (`begin`), and its logit is looked up behind them, when
// the caches hold it (`end`): neither keeps the sweep waiting.
template <typename T>
struct Fetch {
  int64_t at = -1;
  float t = 0.f;
  __device__ __forceinline__ void begin(const DistillArgs& a, int64_t row, int64_t label) {
    const int i = threadIdx.x;
    if (i < a.k) {
      at = a.ids[row * a.k + i];
      t = load_teacher(a, row * a.k + i);
    } else if (i == a.k) {
      at = label;
    }
  }
  __device__ __forceinline__ void end(const DistillArgs& a, const Entries& e, int64_t row, const T* z, int64_t label) {
    for (int i = threadIdx.x; i <= a.k; i += kDistillThreads) {
      if (i != (int)threadIdx.x) {
        at = i < a.k ? a.ids[row * a.k + i] : label;
        t = i < a.k ? load_teacher(a, row * a.k + i) : 0.f;
      }
      const bool in = (uint64_t)at < (uint64_t)a.v;
      e.at[i] = in ? (int)at : -1;
      e.p[i] = t;
      e.z[i] = in ? Elem<T>::to_f32(z[at]) : 0.f;
    }
  }
};

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
__device__ __forceinline__ Coefficients coefficients(const DistillArgs& a, int64_t row, float4 stats, bool labels) {
  const float w = (a.dy ? a.dy[row * a.dy_step] : 1.f) * a.grad_scale;
  Coefficients co;
  co.c = a.c;
  co.base = base_of(stats.x);
  co.teach = w * a.soft_grad;
  co.hit = labels ? w * a.hard : 0.f;
  co.soft = co.teach * (stats.w + 1.f) / stats.y;
  co.hard = co.hit / stats.z;
  if (S == kNone) {  // one exponential serves both terms, or there is one term only
    co.soft += labels ? co.hit / stats.y : 0.f;
    co.hard = 0.f;
  }
  return co;
}

// 16 bytes from an address that is 4 Q + r bytes (r = bits / 8, 0 or 2) behind a 16-byte boundary.
template <int Q>
__device__ __forceinline__ uint4 load_shifted(const char* p, uint32_t bits) {
  if constexpr (Q < 0) {
    return *reinterpret_cast<const uint4*>(p);
  } else {
    const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
    const uint4 a = q[0], b = q[1];
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return make_uint4(__funnelshift_r(w[Q], w[Q + 1], bits), __funnelshift_r(w[Q + 1], w[Q + 2], bits),
                      __funnelshift_r(w[Q + 2], w[Q + 3], bits), __funnelshift_r(w[Q + 3], w[(Q + 4) & 7], bits));
  }
}

// The gradient of the groups of a slice, which is aligned at `out`.
template <typename T, Second S, int Q>
__device__ __forceinline__ void write_groups(const Slice<T>& s, const T* z, T* out, const Coefficients& co) {
  constexpr int per = Slice<T>::kPer;
  const char* from = reinterpret_cast<const char*>(z + s.head);
  uint4* to = reinterpret_cast<uint4*>(out + s.head);
  const uint32_t bits = (reinterpret_cast<uintptr_t>(from) & 3) * 8;
  auto groups = [&](int i0, auto count) {
    uint4 raw[count.value];
#pragma unroll
    for (int u = 0; u < count.value; ++u) raw[u] = load_shifted<Q>(from + (int64_t)(i0 + u * kDistillThreads) * 16, bits);
#pragma unroll
    for (int u = 0; u < count.value; ++u) {
      uint4 r;
      if constexpr (sizeof(T) == 4) {
        const Two a = co.at<S>(Raw<T>::pair(raw[u], 0)), b = co.at<S>(Raw<T>::pair(raw[u], 1));
        r = make_uint4(__float_as_uint(a.lo()), __float_as_uint(a.hi()), __float_as_uint(b.lo()), __float_as_uint(b.hi()));
      } else {
        r = make_uint4(Raw<T>::put(co.at<S>(Raw<T>::pair(raw[u], 0))), Raw<T>::put(co.at<S>(Raw<T>::pair(raw[u], 1))),
                       Raw<T>::put(co.at<S>(Raw<T>::pair(raw[u], 2))), Raw<T>::put(co.at<S>(Raw<T>::pair(raw[u], 3))));
      }
      to[i0 + u * kDistillThreads] = r;
    }
  };
  int i = s.from + threadIdx.x;
  for (; i + (kDistillUnroll - 1) * kDistillThreads < s.to; i += kDistillUnroll * kDistillThreads)
    groups(i, std::integral_constant<int, kDistillUnroll>{});
  for (; i < s.to; i += kDistillThreads) groups(i, std::integral_constant<int, 1>{});
}

// z and out lie at the same distance from a 16-byte boundary: nothing is shifted.
template <typename T>
__device__ __forceinline__ bool alike(const T* z, const T* out) {
  return ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
}

template <typename T, Second S>
__device__ __forceinline__ void write_slice(const Slice<T>& s, const T* z, T* out, const Coefficients& co) {
  if (alike(z, out)) {
    write_groups<T, S, -1>(s, z, out, co);
  } else {
    switch ((reinterpret_cast<uintptr_t>(z + s.head) & 15) >> 2) {
      case 0: write_groups<T, S, 0>(s, z, out, co); break;
      case 1: write_groups<T, S, 1>(s, z, out, co); break;
      case 2: write_groups<T, S, 2>(s, z, out, co); break;
      default: write_groups<T, S, 3>(s, z, out, co); break;
    }
  }
  if ((int)threadIdx.x < s.edge) {
    const int j = s.edge_at(threadIdx.x);
    out[j] = Elem<T>::from_f32(co.at<S>(Elem<T>::to_f32(z[j])));
  }
}

// The elements that the teacher or the label names, once each however often they are named.
template <typename T, Second S>
__device__ __forceinline__ void write_entries(const DistillArgs& a, const Entries& e, const Slice<T>& s, T* out, const Coefficients& co,
                                              int slice) {
  for (int i = threadIdx.x; i <= a.k; i += kDistillThreads) {
    const int j = e.at[i];
    if (j < 0 || !s.owns(j, slice == 0, slice + 1 == 1 << a.slices_log)) continue;
    bool again = false;
    float p = e.p[i];
    for (int q = 0; q <= a.k; ++q) {
      if (q == i || e.at[q] != j) continue;
      again |= q < i;
      p += e.p[q];
    }
    if (again) continue;
    float g = co.at<S>(e.z[i]) - co.teach * p;
    if (e.at[a.k] == j) g -= co.hit;
    out[j] = Elem<T>::from_f32(g);
  }
}

template <typename T>
__device__ __forceinline__ void zero_slice(const Slice<T>& s, T* out) {
  uint4* to = reinterpret_cast<uint4*>(out + s.head);
  for (int i = s.from + threadIdx.x; i < s.to; i += kDistillThreads) to[i] = make_uint4(0, 0, 0, 0);
  if ((int)threadIdx.x < s.edge) out[s.edge_at(threadIdx.x)] = Elem<T>::from_f32(0.f);
}

// Loss, and with GRAD the gradient, of a row by a cluster of `slices` blocks: one pass with a running maximum and its
// sums, joined over threads, warps and blocks; the gradient reads the row again, which the L2 still holds.
template <typename T, Second S, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads, kDistillBlocks) distill_kernel(DistillArgs a) {
  constexpr int per = Slice<T>::kPer;
  extern __shared__ char smem[];
  __shared__ Running warps[kDistillWarps];
  __shared__ Running whole;
  __shared__ float some_s;
  const Entries e(smem, a.k);
  grid_dependency_trigger();
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slices = 1 << a.slices_log;
  const int64_t row = blockIdx.x >> a.slices_log;
  const int slice = blockIdx.x & (slices - 1);
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  T* out = GRAD ? static_cast<T*>(a.out) + row * a.ld_out : nullptr;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && (label == a.ignore || (uint64_t)label >= (uint64_t)a.v)) {  // the same for every block of the cluster
    if (slice == 0 && tid == 0) {
      a.loss[row] = 0.f;
      if (a.stats) a.stats[row] = make_float4(0.f, 1.f, 1.f, -1.f);
    }
    if (GRAD) zero_slice(Slice<T>(out, (int)a.v, slice, a.slices_log, false), out);
    return;
  }
  Fetch<T> fetch;
  fetch.begin(a, row, label);

  Running run{-INFINITY, 0.f, 0.f};
  const Slice<T> s(z, (int)a.v, slice, a.slices_log, false);
  {
    const uint4* middle = reinterpret_cast<const uint4*>(z + s.head);
    Two soft(0.f, 0.f), hard(0.f, 0.f);
    auto groups = [&](int i0, auto count) {
      uint4 raw[count.value];
#pragma unroll
      for (int u = 0; u < count.value; ++u) raw[u] = middle[i0 + u * kDistillThreads];
      uint32_t most = Raw<T>::max2(raw[0]);
#pragma unroll
      for (int u = 1; u < count.value; ++u) most = Raw<T>::max2(most, Raw<T>::max2(raw[u]));
      const float top = fmaxf(run.top, Raw<T>::max1(most)), base = base_of(top);
      if (top != run.top) {
        const float d = run.top - top;  // -infinity at first: the sums are 0 and stay it, or NaN
        const float fs = run.top == -INFINITY ? 1.f : ex2(d * a.c), fh = run.top == -INFINITY ? 1.f : ex2(d * kLog2e);
        soft = soft * Two(fs, fs);
        if (S != kNone) hard = hard * Two(fh, fh);
        run.top = top;
      }
      const Two nb(-base, -base), c2(a.c, a.c);
#pragma unroll
      for (int u = 0; u < count.value; ++u) {
#pragma unroll
        for (int j = 0; j < per / 2; ++j) {
          const Two x = Raw<T>::pair(raw[u], j) + nb, p = ex2(x * c2);
          soft = soft + p;
          if (S == kOwn) hard = hard + ex2(x * Two(kLog2e, kLog2e));
          if (S == kSquare) hard = fma2(p, p, hard);
          if (S == kFourth) hard = fma2(p * p, p * p, hard);
        }
      }
    };
    int i = s.from + tid;
    for (; i + (kDistillUnroll - 1) * kDistillThreads < s.to; i += kDistillUnroll * kDistillThreads)
      groups(i, std::integral_constant<int, kDistillUnroll>{});
    for (; i < s.to; i += kDistillThreads) groups(i, std::integral_constant<int, 1>{});
    run.soft = soft.lo() + soft.hi();
    run.hard = hard.lo() + hard.hi();
  }
  if (tid < s.edge) {
    const float edge = Elem<T>::to_f32(z[s.edge_at(tid)]);
    rebase<S>(run, fmaxf(run.top, edge), a.c);
    const float base = base_of(run.top);
    run.soft += power(edge, base, a.c);
    if (S != kNone) run.hard += power(edge, base, kLog2e);
  }
  fetch.end(a, e, row, z, label);
  // the block's maximum first, then sums relative to it
  float top = run.top;
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) warps[warp].top = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kDistillWarps; ++w) top = fmaxf(top, warps[w].top);
  rebase<S>(run, top, a.c);
  run.soft = warp_sum(run.soft);
  if (S != kNone) run.hard = warp_sum(run.hard);
  if (lane == 0) {
    warps[warp].soft = run.soft;
    warps[warp].hard = run.hard;
  }
  __syncthreads();
  run = Running{top, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kDistillWarps; ++w) {
    run.soft += warps[w].soft;
    run.hard += warps[w].hard;
  }
  if (a.slices_log) {
    if (tid == 0) whole = run;
    cluster_sync();
    for (int r = 0; r < slices; ++r) top = fmaxf(top, __uint_as_float(cluster_load(&whole.top, r)));
    run = Running{top, 0.f, 0.f};
    for (int r = 0; r < slices; ++r) {
      Running other{__uint_as_float(cluster_load(&whole.top, r)), __uint_as_float(cluster_load(&whole.soft, r)),
                    __uint_as_float(cluster_load(&whole.hard, r))};
      rebase<S>(other, top, a.c);
      run.soft += other.soft;
      run.hard += other.hard;
    }
    cluster_sync();  // read by all before one of them overwrites its logits or ends
  }
  const float base = base_of(run.top);
  float4 stats = make_float4(run.top, run.soft, S != kNone ? run.hard : run.soft, 0.f);
  if (warp == 0) {
    float kl = 0.f;
    stats.w = weigh(e, a.k, a.c, base, log2f(run.soft), &kl) - 1.f;
    if (lane == 0) some_s = stats.w;
    if (lane == 0 && slice == 0) {
      float loss = a.soft_loss > 0.f ? a.soft_loss * kl : 0.f;  // a term without weight counts nothing, infinite or not
      if (labels && a.hard > 0.f) loss += a.hard * kLn2 * (log2f(stats.z) - (e.z[a.k] - base) * kLog2e);
      a.loss[row] = loss;
      if (a.stats) a.stats[row] = stats;
    }
  }
  if (!GRAD) return;
  __syncthreads();
  stats.w = some_s;
  const Coefficients co = coefficients<S>(a, row, stats, labels);
  const Slice<T> so(out, (int)a.v, slice, a.slices_log, !alike(z, out));
  write_slice<T, S>(so, z, out, co);
  __syncthreads();
  write_entries<T, S>(a, e, so, out, co, slice);
}

// The gradient from the statistics that the forward pass has left.
template <typename T, Second S>
__global__ void __launch_bounds__(kDistillThreads, kDistillBlocks) distill_dpred_kernel(DistillArgs a) {
  extern __shared__ char smem[];
  const Entries e(smem, a.k);
  grid_dependency_trigger();
  grid_dependency_wait();
  const int64_t row = blockIdx.x >> a.slices_log;
  const int slice = blockIdx.x & ((1 << a.slices_log) - 1);
  const T* z = static_cast<const T*>(a.pred) + row * a.ld;
  T* out = static_cast<T*>(a.out) + row * a.ld_out;
  const bool labels = a.labels.p != nullptr;
  const int64_t label = labels ? a.labels[row] : -1;
  if (labels && (label == a.ignore || (uint64_t)label >= (uint64_t)a.v)) {
    zero_slice(Slice<T>(out, (int)a.v, slice, a.slices_log, false), out);
    return;
  }
  const float4 stats = a.stats[row];
  Fetch<T> fetch;
  fetch.begin(a, row, label);
  const bool in_place = a.out == a.pred;
  if (in_place) {  // this block's entries before any of it is overwritten (another block's are not used here)
    fetch.end(a, e, row, z, label);
    __syncthreads();
  }
  const Slice<T> s(out, (int)a.v, slice, a.slices_log, !alike(z, out));
  const Coefficients co = coefficients<S>(a, row, stats, labels);
  write_slice<T, S>(s, z, out, co);
  if (!in_place) fetch.end(a, e, row, z, label);
  __syncthreads();
  if (threadIdx.x < 32) weigh(e, a.k, a.c, 0.f, 0.f, nullptr);
  __syncthreads();
  write_entries<T, S>(a, e, s, out, co, slice);
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
  return a;
}

static Second second_of(const rafb200_distill* d) {
  if (!d->labels || d->alpha == 1.0 || d->temperature == 1.0) return kNone;  // one term, or both at one temperature
  return d->temperature == 2.0 ? kSquare : d->temperature == 4.0 ? kFourth : kOwn;
}

// Blocks of a row, as a power of two: few rows are cut until every SM has work, while a thread keeps a group.
static int row_slices_log(const rafb200_distill* d) {
  int log = 0;
  const int64_t groups = d->v * dtype_size(d->pred_dtype) / 16;
  while (log < 3 && (d->n << (log + 1)) <= 148 * 2 && groups >> (log + 1) >= kDistillThreads) ++log;
  return log;
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
  a.slices_log = row_slices_log(d);
  return with_case(d, [&](auto t, auto second) {
    RAFB200_CUDA(launch_cluster(distill_kernel<decltype(t), decltype(second)::value, false>, 1u << a.slices_log, (unsigned)(d->n << a.slices_log),
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
  a.slices_log = row_slices_log(d);
  return with_case(d, [&](auto t, auto second) {
    RAFB200_CUDA(launch_dependent(distill_dpred_kernel<decltype(t), decltype(second)::value>, dim3((unsigned)(d->n << a.slices_log)),
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
  a.slices_log = row_slices_log(d);
  return with_case(d, [&](auto t, auto second) {
    RAFB200_CUDA(launch_cluster(distill_kernel<decltype(t), decltype(second)::value, true>, 1u << a.slices_log, (unsigned)(d->n << a.slices_log),
                                kDistillThreads, Entries::bytes(d->k), static_cast<cudaStream_t>(stream), a));
    return (int)RAFB200_OK;
  });
}

}  // extern "C"
