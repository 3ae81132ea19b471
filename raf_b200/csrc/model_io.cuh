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

// VEC consecutive elements widened to fp32: 8 (16-byte accesses, which the address must allow), 2 (4 bytes, for
// 16-bit types) or 1.
template <typename T, int VEC>
struct Group {
  float x[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) {
      x[0] = Elem<T>::to_f32(*p);
    } else if constexpr (VEC == 2) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t r = *reinterpret_cast<const uint32_t*>(p);
        T h[2];
        memcpy(h, &r, 4);
        x[0] = Elem<T>::to_f32(h[0]);
        x[1] = Elem<T>::to_f32(h[1]);
      } else {
        const float2 r = *reinterpret_cast<const float2*>(p);
        x[0] = r.x;
        x[1] = r.y;
      }
    } else {
      constexpr int per = 16 / sizeof(T);
#pragma unroll
      for (int q = 0; q < VEC / per; ++q) {
        const uint4 r = reinterpret_cast<const uint4*>(p)[q];
        unpack<T>(r, x + q * per);
      }
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC == 1) {
      *p = Elem<T>::from_f32(x[0]);
    } else if constexpr (VEC == 2) {
      if constexpr (sizeof(T) == 2) {
        const T h[2] = {Elem<T>::from_f32(x[0]), Elem<T>::from_f32(x[1])};
        uint32_t r;
        memcpy(&r, h, 4);
        *reinterpret_cast<uint32_t*>(p) = r;
      } else {
        *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
      }
    } else {
      constexpr int per = 16 / sizeof(T);
#pragma unroll
      for (int q = 0; q < VEC / per; ++q) reinterpret_cast<uint4*>(p)[q] = pack<T>(x + q * per);
    }
  }
  template <typename U>
  static __device__ __forceinline__ void unpack(const uint4& r, float* f) {
    if constexpr (sizeof(U) == 4) {
      f[0] = __uint_as_float(r.x);
      f[1] = __uint_as_float(r.y);
      f[2] = __uint_as_float(r.z);
      f[3] = __uint_as_float(r.w);
    } else {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<U, __nv_bfloat16>::value) {  // bf16 -> fp32 is a 16-bit shift
          f[2 * i] = __uint_as_float(w[i] << 16);
          f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
          __half2 h;
          memcpy(&h, &w[i], 4);
          const float2 g = __half22float2(h);
          f[2 * i] = g.x;
          f[2 * i + 1] = g.y;
        }
      }
    }
  }
  template <typename U>
  static __device__ __forceinline__ uint4 pack(const float* f) {
    if constexpr (sizeof(U) == 4) {
      return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<U, __nv_bfloat16>::value) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&w[i], &h, 4);
        } else {
          const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&w[i], &h, 4);
        }
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
};

// ---- thread-block clusters ------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
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

// Lets the kernel take `bytes` of dynamic shared memory on the current device, asked of the driver when they grow.
template <auto kKernel>
inline int allow_smem(size_t bytes) {
  static std::atomic<size_t> granted[64];
  int device = 0;
  RAFB200_CUDA(cudaGetDevice(&device));
  if (bytes <= 48 * 1024 || (device < 64 && granted[device].load(std::memory_order_relaxed) >= bytes)) return RAFB200_OK;
  RAFB200_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  if (device < 64) granted[device].store(bytes, std::memory_order_relaxed);
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
