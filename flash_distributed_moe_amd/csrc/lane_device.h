// Sums and maxima across lanes, for kernels that give a row to 16 lanes or to whole waves.
#pragma once
#include <hip/hip_runtime.h>

namespace fmoe {

// A value of the lane CTRL says, inside rows of 16 lanes (data parallel primitives: no LDS, no wait).
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(int, v)));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140, kRotate8 = 0x128;
constexpr int kNextLane = 0x101;  // the lane on, 0 behind the 16th

// Over the row of 16 lanes, in all of them, in one order: every lane gets the same bits.
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kMirror8>(v);
  return v + dpp<kMirror16>(v);
}
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp<kXor1>(v));
  v = fmaxf(v, dpp<kXor2>(v));
  v = fmaxf(v, dpp<kMirror8>(v));
  return fmaxf(v, dpp<kMirror16>(v));
}
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned umin(unsigned a, unsigned b) { return a < b ? a : b; }
__device__ __forceinline__ unsigned row16_max(unsigned v) {
  v = umax(v, static_cast<unsigned>(dpp<kXor1>(static_cast<int>(v))));
  v = umax(v, static_cast<unsigned>(dpp<kXor2>(static_cast<int>(v))));
  v = umax(v, static_cast<unsigned>(dpp<kMirror8>(static_cast<int>(v))));
  return umax(v, static_cast<unsigned>(dpp<kMirror16>(static_cast<int>(v))));
}
__device__ __forceinline__ unsigned row16_min(unsigned v) {
  v = umin(v, static_cast<unsigned>(dpp<kXor1>(static_cast<int>(v))));
  v = umin(v, static_cast<unsigned>(dpp<kXor2>(static_cast<int>(v))));
  v = umin(v, static_cast<unsigned>(dpp<kMirror8>(static_cast<int>(v))));
  return umin(v, static_cast<unsigned>(dpp<kMirror16>(static_cast<int>(v))));
}
// Over the wave, in a scalar register.
__device__ __forceinline__ float wave_sum(float v) {
  const int r = __builtin_bit_cast(int, row16_sum(v));
  const auto at = [&](int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(r, lane)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

__device__ __forceinline__ int wave_sum(int v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kMirror8>(v);
  v += dpp<kMirror16>(v);
  const auto at = [&](int lane) { return __builtin_amdgcn_readlane(v, lane); };
  return (at(0) + at(16)) + (at(32) + at(48));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  const unsigned lo = static_cast<unsigned>(dpp<CTRL>(static_cast<int>(b))), hi = static_cast<unsigned>(dpp<CTRL>(static_cast<int>(b >> 32)));
  return __builtin_bit_cast(double, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp<kXor1>(v);
  v += dpp<kXor2>(v);
  v += dpp<kMirror8>(v);
  v += dpp<kMirror16>(v);
  const long long b = __builtin_bit_cast(long long, v);
  const auto at = [&](int lane) {
    const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(b), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), lane);
    return __builtin_bit_cast(double, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
  };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// This wave's LDS writes have arrived before its later reads of other lanes' data.
__device__ __forceinline__ void wave_lds_ready() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace fmoe
