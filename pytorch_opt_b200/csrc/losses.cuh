// Device helpers shared by the loss kernels: typed loads and stores, block
// reductions in a fixed order, and a teacher's distribution over one row's
// entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace po {

constexpr int kMaxTop = 1024;  // entries a teacher's row may have

template <int DT>
struct ElemOf;
template <>
struct ElemOf<PO_F32> {
  using T = float;
};
template <>
struct ElemOf<PO_BF16> {
  using T = __nv_bfloat16;
};
template <>
struct ElemOf<PO_F16> {
  using T = __half;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f32(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f32(float v, __half& o) { o = __float2half_rn(v); }

// Two fp32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 bytes of a type as floats and back, two 16-bit values an instruction.
template <int DT>
__device__ __forceinline__ void unpack16(const uint4& v, float (&x)[DT == PO_F32 ? 4 : 8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == PO_F32) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == PO_BF16) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack16(const float (&x)[DT == PO_F32 ? 4 : 8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == PO_F32) {
      w[i] = __float_as_uint(x[i]);
    } else if constexpr (DT == PO_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, long long i) {
  if (dtype == PO_F32) return static_cast<const float*>(p)[i];
  if (dtype == PO_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Over the whole block (any multiple of 32 threads up to 1024); every thread
// gets the result. `buf`: 32 values of shared memory, free again on return.
__device__ __forceinline__ float block_max(float v, float* buf) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = warp_max(static_cast<int>(threadIdx.x & 31) < nw ? buf[threadIdx.x & 31] : -INFINITY);
  __syncthreads();
  return v;
}
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* buf) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  const int nw = blockDim.x >> 5;
  v = warp_sum(static_cast<int>(threadIdx.x & 31) < nw ? buf[threadIdx.x & 31] : T(0));
  __syncthreads();
  return v;
}

// Launches of one call follow one another closely: each may start (blocks
// scheduled, barriers and tensor memory set up) while the one before it drains.
// So every thread of every kernel of a call passes grid_wait(), which returns
// when all earlier work is done and visible, before it touches anything that a
// launch of the call writes (what it does before that needs the caller's inputs
// alone, or nothing), and lets its successor start with grid_launch_next(). What an earlier launch of the call wrote is read with ordinary
// loads: the read-only path wants data that no kernel writes while this one is
// resident.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launch behind the previous kernel of the same call (`first`: behind whatever
// is on the stream, in the ordinary way).
template <class... Params, class... Args>
int launch_next(bool first, void (*kern)(Params...), dim3 grid, int block, size_t smem, cudaStream_t s, const char* what,
                Args... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = first ? 0 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...), what);
}

// Temperatures a teacher's form takes: a^2 (the loss's factor) and log2(e) / a
// (the exponents') are ordinary fp32 numbers.
inline bool temperature_ok(float a) { return a >= 0x1p-60f && a <= 0x1p60f; }

// What a row is to the loss.
enum RowStatus : int { ROW_IGNORED = 0, ROW_COUNTED = 1, ROW_BAD = 2 };

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace po
