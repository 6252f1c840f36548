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

// A way to tile a product: rows and columns of C a workgroup takes, and what it costs a CU in microseconds, measured:
// once, and for a step of the k loop while the CU has one such workgroup, two, and for each while it has more.
struct TileCost {
  int rows, columns;
  double once, one, two, more;
};
inline double tile_count(const TileCost& way, const GemmArgs& p) {
  return static_cast<double>((p.M + way.rows - 1LL) / way.rows) * ((p.N + way.columns - 1LL) / way.columns);
}
// Which of `count` ways is done first on 256 CUs; step: k of a step.
inline int pick_tile(const TileCost* ways, int count, int step, const GemmArgs& p) {
  int best = 0;
  double least = 0;
  for (int i = 0; i < count; ++i) {
    const TileCost& way = ways[i];
    const long long each = static_cast<long long>((tile_count(way, p) + 255) / 256);  // tiles of the fullest CU
    const double cost = way.once + (p.K + step - 1) / step * (each <= 1 ? way.one : each == 2 ? way.two : each * way.more);
    if (i == 0 || cost < least) best = i, least = cost;
  }
  return best;
}

enum { ACT_SILU = 0, ACT_GELU_TANH = 1 };
enum { EPI_STORE = 0, EPI_GATED = 1, EPI_SLOPE = 2 };

// The three products of a backward pass that depend on no other of them; one that is not wanted has no rows
// (M = 0). begin: the first workgroup of each.
struct FfnGrads {
  GemmArgs dx, dw13, dw2;
  int begin[3];
};

// Workgroup ranges for tiles of rows x columns, each begun on a multiple of 8 (see tile_of); their number.
inline long long lay_out_grads(FfnGrads& p, int rows, int columns) {
  GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  long long at = 0;
  for (int i = 0; i < 3; ++i) {
    of[i]->grid_m = (of[i]->M + rows - 1) / rows;
    of[i]->grid_n = (of[i]->N + columns - 1) / columns;
    p.begin[i] = static_cast<int>(at < 0x7FFFFFFF ? at : 0x7FFFFFFF);
    at = (at + static_cast<long long>(of[i]->grid_m) * of[i]->grid_n + 7) / 8 * 8;
  }
  return at;
}

// Which of `count` ways is done with all three first on 256 CUs, which take tiles as they come: the work
// spread over all of them and, as the ends never meet, half of the shortest tile; or the longest tile alone.
inline int pick_grads_tile(const TileCost* ways, int count, int step, const FfnGrads& p) {
  const GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  int best = 0;
  double least = 0;
  for (int i = 0; i < count; ++i) {
    double work = 0, longest = 0, shortest = 0;
    for (const GemmArgs* g : of) {
      const double tiles = tile_count(ways[i], *g);
      if (tiles == 0) continue;
      const double steps = (g->K + step - 1) / step;
      work += tiles * steps * ways[i].more / 256;
      longest = longest > steps * ways[i].one ? longest : steps * ways[i].one;
      shortest = shortest == 0 || steps * ways[i].more < shortest ? steps * ways[i].more : shortest;
    }
    const double cost = work + shortest / 2 > longest ? work + shortest / 2 : longest;
    if (i == 0 || cost < least) best = i, least = cost;
  }
  return best;
}

// A matrix product in bfloat16 or float32 (k_outer_*: the operand's rows are k); epi as above.
hipError_t launch_ffn_gemm(int dtype, bool k_outer_a, bool k_outer_b, int epi, GemmArgs p, hipStream_t stream);
// MXFP4 weights b times bfloat16 rows (x_mxfp4 false) or MXFP4 rows; EPI_STORE or EPI_GATED (bfloat16 rows only).
hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, GemmArgs p, hipStream_t stream);
hipError_t launch_ffn_grads(int dtype, const FfnGrads& p, hipStream_t stream);
hipError_t launch_ffn_grads_f32(FfnGrads p, hipStream_t stream);
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
