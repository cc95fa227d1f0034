// What the kernels of mfcc_amd/csrc/sequence_kernels.h and their launches in sequence_ops.hip use of the HIP runtime, for the
// host build in sequence_sim.cpp: one host fiber per device thread, one workgroup after the other.
#pragma once

#include <math.h>
#include <stdint.h>

#include <functional>
#include <limits>
#include <type_traits>

#define __global__
#define __device__
#define __launch_bounds__(...)
#define __shared__ thread_local   // all fibers of a workgroup run on one host thread
#define __align__(n) alignas(n)

struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
struct uint4 { uint32_t x, y, z, w; };
inline float2 make_float2(float x, float y) { return {x, y}; }
inline float4 make_float4(float x, float y, float z, float w) { return {x, y, z, w}; }
inline uint4 make_uint4(uint32_t x, uint32_t y, uint32_t z, uint32_t w) { return {x, y, z, w}; }

struct dim3 {
  unsigned x, y, z;
  dim3(unsigned x = 1, unsigned y = 1, unsigned z = 1) : x(x), y(y), z(z) {}
};
extern dim3 threadIdx, blockIdx, blockDim;
void __syncthreads();

template <typename A, typename B>
inline auto min(A a, B b) { return b < a ? b : (std::common_type_t<A, B>)a; }
template <typename A, typename B>
inline auto max(A a, B b) { return a < b ? b : (std::common_type_t<A, B>)a; }
inline float __expf(float v) { return expf(v); }
// the hardware's reciprocal and reciprocal root take subnormal arguments for 0
inline float sim_flushed(float v) { return fabsf(v) < std::numeric_limits<float>::min() ? copysignf(0.0f, v) : v; }
#define __builtin_amdgcn_rcpf(v) (1.0f / sim_flushed(v))
#define __builtin_amdgcn_rsqf(v) ((float)(1.0 / sqrt((double)sim_flushed(v))))
inline float sim_frexp_mant(float v) { int e; return isfinite(v) ? frexpf(v, &e) : v; }
inline int sim_frexp_exp(float v) { int e = 0; return isfinite(v) ? frexpf(v, &e), e : 0; }
#define __builtin_amdgcn_frexp_mantf(v) sim_frexp_mant(v)
#define __builtin_amdgcn_frexp_expf(v) sim_frexp_exp(v)
#define __builtin_amdgcn_ldexpf(v, e) ldexpf(v, e)
#define __builtin_amdgcn_readfirstlane(v) (v)

typedef void* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
inline hipError_t hipGetLastError() { return hipSuccess; }
inline const char* hipGetErrorString(hipError_t) { return ""; }

void sim_launch(dim3 grid, dim3 block, size_t shared, const std::function<void()>& thread);
template <typename K, typename... A>
void hipLaunchKernelGGL(K kernel, dim3 grid, dim3 block, size_t shared, hipStream_t, A... args) {
  sim_launch(grid, block, shared, [&] { kernel(args...); });
}
