// MXFP4 quantisation of rows and the way back.
//
// A block is 32 consecutive values of a row. With m the largest magnitude of a block its scale is
// 2^s, s = floor(log2 m) - 2 (at least -127): 2 is the exponent of the largest value of the grid, 6, so
// m / 2^s lies in [4, 8) and what is over 6 becomes 6. The values are v / 2^s rounded to the nearest of
// the grid, ties to the even code. A block with an infinity or a NaN gets the scale byte 255, which
// stands for NaN: all of its values are NaN.
#include "ffn_device.h"

namespace fmoe {

// four lanes a block, eight values a lane
template <bool F32>
__global__ __launch_bounds__(256) void mxfp4_quantize_kernel(const void* x, long long ldx, long long rows, int row_blocks,
                                                             unsigned* codes, unsigned char* scales) {
  const long long at = blockIdx.x * 256LL + threadIdx.x, block = at >> 2;
  const int part = threadIdx.x & 3;
  const bool in = block < rows * row_blocks;
  const long long row = in ? block / row_blocks : 0;
  const long long from = row * ldx + (in ? block - row * row_blocks : 0) * 32 + part * 8;
  float v[8];
  if constexpr (F32) {
    const f32x4 lo = *reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + from);
    const f32x4 hi = *reinterpret_cast<const f32x4*>(static_cast<const float*>(x) + from + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const unsigned short*>(x) + from);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
  // magnitudes order as their bits do, infinities and NaN above all others
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  most = max(most, __shfl_xor(most, 1, 64));
  most = max(most, __shfl_xor(most, 2, 64));
  const unsigned exponent = most >> 23;  // of numbers below 2^-126 zero: their scale is the smallest anyway
  const unsigned byte = exponent == 255 ? 255 : exponent < 2 ? 0 : exponent - 2;
  // the conversion divides by the scale, rounds to nearest even and stops at 6; a byte of 0 is 2^-127
  const float scale = __uint_as_float(byte == 0 ? 0x00400000u : (byte == 255 ? 254u : byte) << 23);
  unsigned word = 0;
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[0], v[1], scale, 0);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[2], v[3], scale, 1);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[4], v[5], scale, 2);
  word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, v[6], v[7], scale, 3);
  if (in) {
    codes[at] = word;
    if (part == 0) scales[block] = static_cast<unsigned char>(byte);
  }
}

template <bool F32>
__global__ __launch_bounds__(256) void mxfp4_dequantize_kernel(const unsigned* codes, const unsigned char* scales, long long rows,
                                                               int row_blocks, void* out, long long ldo) {
  const long long at = blockIdx.x * 256LL + threadIdx.x, block = at >> 2;
  if (block >= rows * row_blocks) return;
  const long long row = block / row_blocks;
  const long long to = row * ldo + (block - row * row_blocks) * 32 + (threadIdx.x & 3) * 8;
  const unsigned word = codes[at];
  const float scale = __uint_as_float(static_cast<unsigned>(scales[block]) << 23);
  u32x4 w;
  w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0));
  w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1));
  w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2));
  w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3));
  if constexpr (F32) {  // every value is a bfloat16
    float* o = static_cast<float*>(out) + to;
    *reinterpret_cast<u32x4*>(o) = u32x4{w[0] << 16, w[0] & 0xFFFF0000u, w[1] << 16, w[1] & 0xFFFF0000u};
    *reinterpret_cast<u32x4*>(o + 4) = u32x4{w[2] << 16, w[2] & 0xFFFF0000u, w[3] << 16, w[3] & 0xFFFF0000u};
  } else {
    *reinterpret_cast<u32x4*>(static_cast<unsigned short*>(out) + to) = w;
  }
}

static bool grid_for(long long rows, int k, unsigned& blocks) {
  const long long n = (rows * (k / 32) * 4 + 255) / 256;
  blocks = static_cast<unsigned>(n);
  return n * 256 <= 0xFFFFFFFFll;  // threads of a launch
}

hipError_t launch_mxfp4_quantize(int dtype, const void* x, long long ldx, int rows, int k, void* codes, void* scales,
                                 hipStream_t stream) {
  unsigned blocks;
  if (!grid_for(rows, k, blocks)) return hipErrorInvalidValue;
  if (blocks == 0) return hipSuccess;
  auto kernel = dtype == 0 ? mxfp4_quantize_kernel<true> : mxfp4_quantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, x, ldx, static_cast<long long>(rows), k / 32,
                     static_cast<unsigned*>(codes), static_cast<unsigned char*>(scales));
  return hipGetLastError();
}

hipError_t launch_mxfp4_dequantize(int dtype, const void* codes, const void* scales, int rows, int k, void* out,
                                   long long ldo, hipStream_t stream) {
  unsigned blocks;
  if (!grid_for(rows, k, blocks)) return hipErrorInvalidValue;
  if (blocks == 0) return hipSuccess;
  auto kernel = dtype == 0 ? mxfp4_dequantize_kernel<true> : mxfp4_dequantize_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, static_cast<const unsigned*>(codes),
                     static_cast<const unsigned char*>(scales), static_cast<long long>(rows), k / 32, out, ldo);
  return hipGetLastError();
}

}  // namespace fmoe
