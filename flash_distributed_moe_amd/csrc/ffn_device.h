// Device helpers of the dense feed-forward kernels: operand tiles in LDS, the fragments the matrix
// instructions take from them, and the activation with its slope.
//
// A tile is the same for every type: ROWS rows of 128 bytes a step of the k loop (64 bfloat16, 32
// float32 or 256 MXFP4 values) where a row of memory holds consecutive k, and as many bytes as k rows
// of ROWS values where a row of memory is one k. It is loaded 16 bytes a lane straight to LDS, which
// puts the lanes of a wave side by side; so where a 16-byte piece goes is decided by which piece a
// lane asks for. Places outside the matrix are asked for beyond the end of the buffer descriptor and
// arrive as zeros: no tile needs a tail of its own.
#pragma once
#include <hip/hip_runtime.h>

#include "ffn_params.h"

namespace fmoe {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

#define FFN_LDS __attribute__((address_space(3)))

enum ElemKind { KIND_BF16 = 0, KIND_F32 = 1, KIND_MXFP4 = 2 };
__host__ __device__ constexpr int step_k(int kind) { return kind == KIND_BF16 ? 64 : kind == KIND_F32 ? 32 : 256; }
__host__ __device__ constexpr int piece_k(int kind) { return step_k(kind) / 8; }  // values in 16 bytes

constexpr unsigned kOutside = 0x80000000u;  // past the end of every descriptor

// The F blocks of 16 rows a wave takes are dealt eight rows at a time: row r of block f is row
// 8F * (r / 8) + 8f + r % 8 of the wave's 16F. So a lane and the one 16 on have, of one block, eight
// neighbouring results between them, and of the next block the eight that follow.
template <int F>
__device__ __forceinline__ int dealt_row(int f, int r) {
  return 8 * F * (r >> 3) + 8 * f + (r & 7);
}

// Rows of the gated kernels' weight tile: a wave's blocks are half gate and half up rows of the same columns.
template <int F>
__device__ __forceinline__ int gated_row(int f, int r) {
  return 8 * (F / 2) * (r >> 3) + 8 * (f % (F / 2)) + (r & 7);
}

// Where a row is one k, a matrix instruction's operand is read transposed (ds_read_b64_tr_b16): 16 lanes read four
// rows of two 16-byte pieces F pieces apart, and the next 16 lanes the rows eight further on at the same
// time. The pieces of row k are swapped about by bits 0, 1 and 3 of k so that these sixteen lie in
// different banks. (With rows dealt four at a time half of the reads' time were conflicts.)
template <int F>
__device__ __forceinline__ int k_row_swap(int k) {
  const int q = k & 3, g = (k >> 3) & 1;
  return F == 4 ? q | g << 3 : (q & 1) | (q & 2) << 1 | g << 3;
}
// float32: 4 bytes a lane of every k row, sixteen lanes two runs of 32 bytes, and four rows eight apart at once
template <int F>
__device__ __forceinline__ int f32_k_row_swap(int k) {
  const int g = (k >> 3) & 3;
  return F >= 4 ? g << 1 : (g & 1) << 1 | (g & 2) << 2;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00020000);
}
__device__ __forceinline__ void load_to_lds16(__amdgpu_buffer_rsrc_t r, char* lds, unsigned offset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (FFN_LDS void*)lds, 16, static_cast<int>(offset), 0, 0, 0);
}

// ------------------------------------------------------------------ activation
// Both activations are g * sigmoid(w): w = g for SiLU, and for GELU in its tanh form
// (1 + tanh z) / 2 = sigmoid(2z), which has no cancellation for negative z. EXACT (float32 results)
// takes the library's exponential and division; results that are rounded to bfloat16 take the
// hardware's, whose errors (2^-22) are far below that rounding.
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float w) {
  if constexpr (EXACT) return 1.0f / (1.0f + expf(-w));
  return __builtin_amdgcn_rcpf(1.0f + __expf(-w));
}
template <bool EXACT>
__device__ __forceinline__ float act_of(int act, float g) {
  const float w = act == ACT_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g * sigmoid<EXACT>(w);
}
// act(g) and act'(g) = sigmoid(w) + g sigmoid(w) (1 - sigmoid(w)) dw/dg. The sigmoid is 0 or 1 long before g^2 is 10^12,
// and with more dw/dg would be infinite from 2 * 10^19 on, which the zero beside it does not make a number again.
template <bool EXACT>
__device__ __forceinline__ void act_and_slope(int act, float g, float& a, float& slope) {
  const float g2 = fminf(g * g, 1e12f);
  const float w = act == ACT_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g2 * g);
  const float dw = act == ACT_SILU ? 1.0f : 1.5957691216057308f * (1.0f + 0.134145f * g2);
  const float s = sigmoid<EXACT>(w);
  a = g * s;
  slope = s + a * (1.0f - s) * dw;
}

__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
  const bf16x2 v = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};  // nearest, ties to even
  return __builtin_bit_cast(unsigned, v);
}

}  // namespace fmoe
