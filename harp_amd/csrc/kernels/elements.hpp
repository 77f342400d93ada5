// Element types of the hand-written operator kernels: 16 bytes of f32, bf16 or f16 to f32 values
// and back (rounded to nearest even), at any alignment of the element itself.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <tuple>

#include "../operators.hpp"

namespace eh {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));      // rows of an odd number of 16-bit elements start anywhere
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Elem;

template <> struct Elem<kF32> {
  static constexpr uint32_t kMinusInfinity = 0xff800000u;       // a word of them
  static constexpr int N = 4;                              // elements in 16 bytes
  typedef float T;
  __device__ static void unpack(u32x4 v, float* z) {
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = __uint_as_float(v[i]);
  }
  __device__ static u32x4 pack(const float* z) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(z[i]);
    return v;
  }
  __device__ static float get(T x) { return x; }
  __device__ static T put(float x) { return x; }
};

template <> struct Elem<kBF16> {
  static constexpr uint32_t kMinusInfinity = 0xff80ff80u;       // a word of them
  static constexpr int N = 8;
  typedef uint16_t T;
  __device__ static void unpack(u32x4 v, float* z) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[2 * i] = __uint_as_float(v[i] << 16);
      z[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
  __device__ static u32x4 pack(const float* z) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 p = {z[2 * i], z[2 * i + 1]};
      v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
    }
    return v;
  }
  __device__ static float get(T x) { return __uint_as_float(static_cast<uint32_t>(x) << 16); }
  __device__ static T put(float x) { return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x)); }
};

template <> struct Elem<kF16> {
  static constexpr uint32_t kMinusInfinity = 0xfc00fc00u;       // a word of them
  static constexpr int N = 8;
  typedef uint16_t T;
  __device__ static void unpack(u32x4 v, float* z) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f16x2 p = __builtin_bit_cast(f16x2, static_cast<uint32_t>(v[i]));
      z[2 * i] = static_cast<float>(p[0]);
      z[2 * i + 1] = static_cast<float>(p[1]);
    }
  }
  __device__ static u32x4 pack(const float* z) {
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f32x2 p = {z[2 * i], z[2 * i + 1]};
      v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(p, f16x2));
    }
    return v;
  }
  __device__ static float get(T x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
  __device__ static T put(float x) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x)); }
};

__device__ inline u32x4 load16(const void* p) { return *static_cast<const u32x4_any*>(p); }
__device__ inline void store16(void* p, u32x4 v) { *static_cast<u32x4_any*>(p) = v; }
// (past the caches: for results that a launch larger than they are does not read again)
__device__ inline void stream16(void* p, u32x4 v) { __builtin_nontemporal_store(v, static_cast<u32x4_any*>(p)); }

// An element of a run-time type: for the few values a row has besides its logits.
__device__ inline float load_as(const void* p, int64_t i, int dtype) {
  if (dtype == kF32) return static_cast<const float*>(p)[i];
  const uint16_t x = static_cast<const uint16_t*>(p)[i];
  return dtype == kBF16 ? Elem<kBF16>::get(x) : Elem<kF16>::get(x);
}
__device__ inline int64_t load_id(const TokenIds& t, int64_t i) {
  return t.wide ? static_cast<const int64_t*>(t.ids)[i] : static_cast<int64_t>(static_cast<const int32_t*>(t.ids)[i]);
}

// The larger of three numbers, NaN left out.  fmaxf would first quiet each operand it knows nothing
// about with an instruction of its own.  Operands must not be results of exp2_hw or log2_hw: the
// compiler cannot place the wait that those need in front of this instruction.
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }   // 1 ulp; results below 2^-126 are 0
__device__ inline float log2_hw(float x) { return __builtin_amdgcn_logf(x); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// A value moved between the lanes of a wave: quad permutes, mirrored halves and rows of 16, rows
// broadcast to the next ones.  Unwritten lanes keep `keep`.
template <int CTRL, int ROWS = 0xf> __device__ inline float dpp(float keep, float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(keep), __float_as_uint(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS = 0xf> __device__ inline uint32_t dpp(uint32_t keep, uint32_t x) {
  return __builtin_amdgcn_update_dpp(keep, x, CTRL, ROWS, 0xf, false);
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kBcast15 = 0x142, kBcast31 = 0x143;

// The sum (maximum) over the wave, in every lane; the order of the additions is fixed.
__device__ inline float wave_sum(float x) {
  x += dpp<kSwap1>(0.f, x);
  x += dpp<kSwap2>(0.f, x);
  x += dpp<kHalfMirror>(0.f, x);
  x += dpp<kMirror>(0.f, x);
  x += dpp<kBcast15, 0xa>(0.f, x);
  x += dpp<kBcast31, 0xc>(0.f, x);
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ inline float wave_max(float x) {
  x = fmaxf(x, dpp<kSwap1>(x, x));
  x = fmaxf(x, dpp<kSwap2>(x, x));
  x = fmaxf(x, dpp<kHalfMirror>(x, x));
  x = fmaxf(x, dpp<kMirror>(x, x));
  x = fmaxf(x, dpp<kBcast15, 0xa>(x, x));
  x = fmaxf(x, dpp<kBcast31, 0xc>(x, x));
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}

// Queues a kernel and returns what the launch itself returns: the thread's last error may be an earlier call's, of
// anybody's.  An error that is returned here is not left there.
template <class... P, class... A>
hipError_t queue(void (*kernel)(P...), unsigned grid, int threads, size_t lds, hipStream_t stream, const A&... args) {
  static_assert(sizeof...(P) == sizeof...(A));
  std::tuple<P...> values(static_cast<P>(args)...);
  const hipError_t e = std::apply(
      [&](auto&... v) {
        void* list[] = {static_cast<void*>(&v)...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(grid), dim3(static_cast<unsigned>(threads)), list, lds, stream);
      },
      values);
  if (e != hipSuccess) (void)hipGetLastError();
  return e;
}

// The same over a workgroup of THREADS; `lds` holds a value per wave and is free again afterwards.
template <int THREADS> __device__ inline float block_sum(float x, float* lds) {
  x = wave_sum(x);
  if constexpr (THREADS == 64) return x;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) s += lds[i];
  __syncthreads();
  return s;
}
// Two sums at once; `lds` holds two values per wave.
template <int THREADS> __device__ inline void block_sum(float& x, float& y, float* lds) {
  x = wave_sum(x);
  y = wave_sum(y);
  if constexpr (THREADS == 64) {
    __syncthreads();                      // what lanes have left in LDS is there for the others here too
    return;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x, lds[THREADS / 64 + (threadIdx.x >> 6)] = y;
  __syncthreads();
  x = lds[0], y = lds[THREADS / 64];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) x += lds[i], y += lds[THREADS / 64 + i];
  __syncthreads();
}
template <int THREADS> __device__ inline float block_max(float x, float* lds) {
  x = wave_max(x);
  if constexpr (THREADS == 64) return x;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int i = 1; i < THREADS / 64; ++i) s = fmaxf(s, lds[i]);
  __syncthreads();
  return s;
}

}  // namespace
}  // namespace eh
