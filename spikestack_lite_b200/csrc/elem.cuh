// Element types of the training and streaming operators: fp32, bf16 and fp16
// tensors whose arithmetic is fp32, rounded once (to nearest even) when an
// output is stored.
#pragma once

#include <cuda_fp16.h>

#include <mutex>
#include <type_traits>

#include "spk_common.cuh"

namespace spk {

__device__ __forceinline__ float elem_to_f32(float v) { return v; }
__device__ __forceinline__ float elem_to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float elem_to_f32(__half v) { return __half2float(v); }

template <typename E>
__device__ __forceinline__ E elem_from_f32(float v);
template <>
__device__ __forceinline__ float elem_from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 elem_from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half elem_from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// V consecutive elements moved as one access (V * sizeof(E) <= 16 bytes, the
// address a multiple of that).
template <typename E, int V>
struct alignas(sizeof(E) * V) Pack {
  E e[V];
};

template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_pack(const E* p) {
  return *reinterpret_cast<const Pack<E, V>*>(p);
}
template <typename E, int V>
__device__ __forceinline__ void store_pack(E* p, const Pack<E, V>& v) {
  *reinterpret_cast<Pack<E, V>*>(p) = v;
}

// V fp32 values rounded to E; 16-bit ones in pairs, one conversion each.
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> pack_f32(const float (&v)[V]) {
  Pack<E, V> p;
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) {
    if constexpr (sizeof(E) == 4) {
      p.e[i] = v[i];
      p.e[i + 1] = v[i + 1];
    } else {
      uint32_t w;
      if constexpr (std::is_same_v<E, __half>)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v[i + 1]), "f"(v[i]));
      else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v[i + 1]), "f"(v[i]));
      reinterpret_cast<uint32_t*>(&p)[i / 2] = w;
    }
  }
  if (V % 2) p.e[V - 1] = elem_from_f32<E>(v[V - 1]);
  return p;
}

// The hardware's exponential of two and reciprocal (relative errors of 2^-22
// and 2^-23; a subnormal argument or result becomes 0).
__device__ __forceinline__ float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Programmatic dependent launch: the next kernel of the stream may start when
// every block has said so; what the previous one wrote is there after the wait.
__device__ __forceinline__ void grid_dependents_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The two halves of a cluster's barrier, and a value in another block's shared
// memory (the address of this block's copy of it).
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 cluster_load(const float2* mine, uint32_t rank) {
  uint32_t there;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(there) : "memory");
  return v;
}

inline size_t elem_bytes(int dtype) { return dtype == SPK_F32 ? 4 : (dtype == SPK_BF16 || dtype == SPK_F16) ? 2 : 0; }

inline bool aligned_to(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Calls f with a value of the element type (dispatch on dtype); false for an
// unknown dtype.
template <typename F>
inline bool with_elem(int dtype, F&& f) {
  switch (dtype) {
    case SPK_F32:
      f(float{});
      return true;
    case SPK_BF16:
      f(__nv_bfloat16{});
      return true;
    case SPK_F16:
      f(__half{});
      return true;
    default:
      return false;
  }
}

// A value worked out once per device (the current one) and kept.
template <typename T>
class PerDevice {
 public:
  template <typename F>
  cudaError_t get(T* out, F&& make) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= kDevices) return make(out);
    std::lock_guard<std::mutex> lk(mu_);
    if (!known_[dev]) {
      e = make(&value_[dev]);
      if (e != cudaSuccess) return e;
      known_[dev] = true;
    }
    *out = value_[dev];
    return cudaSuccess;
  }

 private:
  static constexpr int kDevices = 64;
  std::mutex mu_;
  bool known_[kDevices] = {};
  T value_[kDevices];
};

}  // namespace spk
