// What the dense gated feed-forward block's and MXFP4's host code and kernels share.
#pragma once
#include <hip/hip_runtime.h>

namespace fmoe {

// One matrix product C[m, n] = sum_k A(m, k) B(n, k) of a launch. An operand lies with its k
// inside a row (A[m * lda + k]) or with a row a k (A[k * lda + m]); which, its type and what
// becomes of the sums are template parameters of the kernel.
struct GemmArgs {
  const void* a;
  const void* b;
  const unsigned char* a_scales;  // MXFP4 operands: a byte for 32 k, rows of K / 32
  const unsigned char* b_scales;
  void* c;          // sums; h [M, N] of the gated kernels; the gradients of both projections [M, 2N] of the slope kernels
  float* gu;        // gated: the projections [M, 2N] are written there, or NULL; slope: read
  long long lda, ldb, ldc;  // elements between rows
  int M, N, K;
  int act;
  int grid_m, grid_n;
};

// A way to tile a product: rows and columns of C a workgroup takes, and what a step of its k loop costs a CU
// while it has one such workgroup, and for each while it has several (microseconds, measured).
struct TileCost {
  int rows, columns;
  double alone, shared;
};
// Which of `count` ways is done first on 256 CUs.
inline int pick_tile(const TileCost* ways, int count, int M, int N) {
  int best = 0;
  double least = 0;
  for (int i = 0; i < count; ++i) {
    const long long tiles = ((M + ways[i].rows - 1LL) / ways[i].rows) * ((N + ways[i].columns - 1LL) / ways[i].columns);
    const long long each = (tiles + 255) / 256;  // tiles of the fullest CU
    const double cost = each == 1 ? ways[i].alone : each * ways[i].shared;
    if (i == 0 || cost < least) best = i, least = cost;
  }
  return best;
}

enum { ACT_SILU = 0, ACT_GELU_TANH = 1 };
enum { EPI_STORE = 0, EPI_GATED = 1, EPI_SLOPE = 2 };

// A matrix product in bfloat16 or float32 (k_outer_*: the operand's rows are k); epi as above.
hipError_t launch_ffn_gemm(int dtype, bool k_outer_a, bool k_outer_b, int epi, GemmArgs p, hipStream_t stream);
// MXFP4 weights b times bfloat16 rows (x_mxfp4 false) or MXFP4 rows; EPI_STORE or EPI_GATED (bfloat16 rows only).
hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, GemmArgs p, hipStream_t stream);
hipError_t launch_ffn_gemm_f32(bool k_outer_a, bool k_outer_b, int epi, const GemmArgs& p, hipStream_t stream);
// The same for few rows, where these take the call (A and B with their k inside the rows).
bool ffn_skinny_takes(int dtype, const GemmArgs& p);
bool mxfp4_skinny_takes(bool x_mxfp4, const GemmArgs& p);
hipError_t launch_ffn_skinny(int dtype, bool gated, const GemmArgs& p, hipStream_t stream);
hipError_t launch_mxfp4_skinny(bool x_mxfp4, bool gated, const GemmArgs& p, hipStream_t stream);
hipError_t launch_mxfp4_quantize(int dtype, const void* x, long long ldx, int rows, int k, void* codes, void* scales,
                                 hipStream_t stream);
hipError_t launch_mxfp4_dequantize(int dtype, const void* codes, const void* scales, int rows, int k, void* out,
                                   long long ldo, hipStream_t stream);

}  // namespace fmoe
