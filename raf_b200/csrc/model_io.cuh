// What the operators at the ends of a model (embedding.cu, distill.cu) share: index loads, groups of VEC
// elements at any alignment, launches of thread-block clusters.
#pragma once
#include <atomic>
#include <cstring>
#include <type_traits>

#include "common.h"
#include "vec_io.cuh"

namespace rafb200 {

// Token ids, class ids: int32 or int64 as the caller has them.
struct Ids {
  const void* p;
  int wide;  // 1: int64
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
  }
};
inline bool index_dtype_valid(int t) { return t == RAFB200_I32 || t == RAFB200_I64; }

// The bytes of an access of `bytes` bytes, at most 16 of them.
template <int BYTES>
struct Word;
template <>
struct Word<2> { using type = unsigned short; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

// A 32-bit word of two 16-bit elements, widened and rounded.
template <typename T>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // bf16 -> fp32 is a 16-bit shift
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// VEC consecutive elements widened to fp32, in accesses of up to 16 bytes, which the address must allow.
template <typename T, int VEC>
struct Group {
  static constexpr int kBytes = VEC * sizeof(T) < 16 ? VEC * sizeof(T) : 16, kWords = VEC * sizeof(T) / kBytes;
  static constexpr int kPer = VEC / kWords;
  using W = typename Word<kBytes>::type;
  float x[VEC];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int q = 0; q < kWords; ++q) unpack(reinterpret_cast<const W*>(p)[q], x + q * kPer);
  }
  // from the L2, where other blocks of the grid have written it
  __device__ __forceinline__ void load_coherent(const T* p) {
#pragma unroll
    for (int q = 0; q < kWords; ++q) unpack(__ldcg(reinterpret_cast<const W*>(p) + q), x + q * kPer);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int q = 0; q < kWords; ++q) reinterpret_cast<W*>(p)[q] = pack(x + q * kPer);
  }
  static __device__ __forceinline__ void unpack(const W& w, float* f) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (kBytes == 4) {
        f[0] = __uint_as_float(w);
      } else {
        f[0] = __uint_as_float(w.x);
        f[1] = __uint_as_float(w.y);
        if constexpr (kBytes == 16) {
          f[2] = __uint_as_float(w.z);
          f[3] = __uint_as_float(w.w);
        }
      }
    } else if constexpr (kBytes == 2) {
      f[0] = widen<T>(w).x;
    } else {
      uint32_t v[kBytes / 4];
      if constexpr (kBytes == 4) {
        v[0] = w;
      } else {
        v[0] = w.x;
        v[1] = w.y;
        if constexpr (kBytes == 16) {
          v[2] = w.z;
          v[3] = w.w;
        }
      }
#pragma unroll
      for (int i = 0; i < kBytes / 4; ++i) {
        const float2 g = widen<T>(v[i]);
        f[2 * i] = g.x;
        f[2 * i + 1] = g.y;
      }
    }
  }
  static __device__ __forceinline__ W pack(const float* f) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (kBytes == 4) return __float_as_uint(f[0]);
      else if constexpr (kBytes == 8) return make_uint2(__float_as_uint(f[0]), __float_as_uint(f[1]));
      else return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    } else {
      if constexpr (kBytes == 2) return (unsigned short)narrow<T>(f[0], 0.f);
      else if constexpr (kBytes == 4) return narrow<T>(f[0], f[1]);
      else if constexpr (kBytes == 8) return make_uint2(narrow<T>(f[0], f[1]), narrow<T>(f[2], f[3]));
      else return make_uint4(narrow<T>(f[0], f[1]), narrow<T>(f[2], f[3]), narrow<T>(f[4], f[5]), narrow<T>(f[6], f[7]));
    }
  }
};

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

// ---- rows at any address ----------------------------------------------------------
// A block's part of a row: elements [begin, end), of which `groups` groups of 16 bytes from element `at` on are aligned
// in memory.  The row's first and last elements, which no aligned group holds, are the first and the last block's.
template <typename T>
struct Slice {
  static constexpr int kPer = 16 / sizeof(T);
  int begin, end, at, groups;

  __device__ __forceinline__ Slice() {}
  __device__ __forceinline__ Slice(const T* p, int v, int slice, int slices_log) {
    const int head = min((int)((-(intptr_t)p & 15) / sizeof(T)), v), all = (v - head) / kPer;
    const int each = (all + (1 << slices_log) - 1) >> slices_log, from = min(slice * each, all);
    groups = min(each, all - from);
    at = head + from * kPer;
    begin = slice ? at : 0;
    end = slice + 1 == 1 << slices_log ? v : at + groups * kPer;
  }
  // The same elements, in groups that are aligned at `p` and whose bytes this slice's groups hold.
  __device__ __forceinline__ Slice aligned_at(const T* p) const {
    Slice s;
    s.begin = begin;
    s.end = end;
    s.at = at + (int)((-(intptr_t)(p + at) & 15) / sizeof(T));
    s.groups = max(at + groups * kPer - s.at, 0) / kPer;
    if (s.groups == 0) s.at = at;
    return s;
  }
  // Elements outside the groups: thread i < edges() takes edge_at(i).
  __device__ __forceinline__ int edges() const { return end - begin - groups * kPer; }
  __device__ __forceinline__ int edge_at(int i) const { return begin + i < at ? begin + i : begin + i + groups * kPer; }
  __device__ __forceinline__ bool owns(int j) const { return j >= begin && j < end; }
};

// 16 bytes from an address that is 4 Q + r bytes (r = bits / 8, 0 or 2) behind a 16-byte boundary; Q < 0: at one.
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

// z and out lie at the same distance from a 16-byte boundary: nothing is shifted.
template <typename T>
__device__ __forceinline__ bool alike(const T* z, const T* out) {
  return ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
}

// ---- thread-block clusters ------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
// Stores a word at the same shared-memory address in block `rank` of the cluster.
__device__ __forceinline__ void cluster_store(void* p, uint32_t rank, uint32_t v) {
  uint32_t at = (uint32_t)__cvta_generic_to_shared(p);
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// The word at the same shared-memory address in block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_load(const void* p, uint32_t rank) {
  uint32_t at = (uint32_t)__cvta_generic_to_shared(p), v;
  asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(at) : "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// launch_dependent() for a grid of clusters of `cluster` blocks.
template <typename... Params, typename... Args>
inline cudaError_t launch_cluster(void (*kernel)(Params...), unsigned cluster, unsigned grid, unsigned block, size_t smem,
                                  cudaStream_t s, Args... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

// Lets the kernel take `bytes` of dynamic shared memory on the current device; `most` is what any launch of it takes, and that is
// asked of the driver, once: of two threads neither can lower the limit that the other needs.  48 KB are given unasked, for these
// and for the kernel's own variables, which are below 1 KB.
template <auto kKernel>
inline int allow_smem(size_t bytes, size_t most) {
  static std::atomic<bool> granted[64];
  int device = 0;
  RAFB200_CUDA(cudaGetDevice(&device));
  if (bytes <= 47 * 1024 || (device < 64 && granted[device].load(std::memory_order_acquire))) return RAFB200_OK;
  RAFB200_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
  if (device < 64) granted[device].store(true, std::memory_order_release);
  return RAFB200_OK;
}

// Lets the kernel run in clusters of 16 blocks.
template <auto kKernel>
inline int allow_large_cluster() {
  static std::atomic<bool> granted[64];
  int device = 0;
  RAFB200_CUDA(cudaGetDevice(&device));
  if (device < 64 && granted[device].load(std::memory_order_relaxed)) return RAFB200_OK;
  RAFB200_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (device < 64) granted[device].store(true, std::memory_order_relaxed);
  return RAFB200_OK;
}

// Calls f with a value of the element type of a dtype code (checked before).
template <typename F>
int with_type(int dtype, const F& f) {
  switch (dtype) {
    case RAFB200_F32: return f(float{});
    case RAFB200_F16: return f(__half{});
    default: return f(__nv_bfloat16{});
  }
}

}  // namespace rafb200
