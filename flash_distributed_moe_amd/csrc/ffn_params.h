// What the dense gated feed-forward block's and MXFP4's host code and kernels share.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>

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
  // A product whose k is dealt to `splits` workgroups a tile, `per` steps each: their sums go to partial,
  // [splits, M, partial_ld(columns of B's rows)] float32, and a kernel of its own finishes. One split: unused.
  float* partial;
  int splits, per;
};
__host__ __device__ inline long long partial_ld(int columns) { return (columns + 7LL) / 8 * 8; }

// A way to tile a product: rows and columns of C a workgroup takes, and what it costs a CU in microseconds, measured:
// once, and for a step of the k loop while the CU has one such workgroup, two, and for each while it has more.
// together (of the gradients' ways): how many of them a CU holds.
struct TileCost {
  int rows, columns;
  double once, one, two, more;
  int together;
};
inline double tile_count(const TileCost& way, const GemmArgs& p) {
  return static_cast<double>((p.M + way.rows - 1LL) / way.rows) * ((p.N + way.columns - 1LL) / way.columns);
}
// Which way is done first on 256 CUs, and with how many workgroups sharing a tile's k.
struct TilePlan {
  int way, splits, per;
};
// What it takes to write and read `splits` partial sums of M x columns and to launch the kernel that does the latter:
// an estimate, a short kernel's time and the rate of a copy
inline double finish_cost(int splits, double sums) { return splits > 1 ? 4.0 + splits * sums * 8 / 4.5e6 : 0.0; }
inline double tile_cost(const TileCost& way, double tiles, int steps) {
  const long long each = static_cast<long long>((tiles + 255) / 256);  // tiles of the fullest CU
  return way.once + steps * (each <= 1 ? way.one : each == 2 ? way.two : each * way.more);
}
// step: k of a step; columns: rows of B; room: bytes of memory for partial sums. Measured, a whole call
// without and with splits, us: T=87, H=144, I=6520 bf16 39 and 18 (the second product has 6 tiles of 64 x 64);
// MXFP4 weights, T=67, H=384, I=7680 40 and 22; a product with MXFP4 weights, M=703, N=591, K=7520 36 and 24; a training
// step, T=2480, H=416, I=8520 bf16 547 and 406. Against the best of all ways and splits this loses 0.3 to 0.9 % (40 random
// calls of each type).
inline size_t partial_bytes(const TilePlan& plan, int M, int columns) {
  return plan.splits > 1 ? static_cast<size_t>(plan.splits) * M * partial_ld(columns) * 4 : 0;
}
inline TilePlan plan_tiles(const TileCost* ways, int count, int step, const GemmArgs& p, int columns, size_t room) {
  const int steps = (p.K + step - 1) / step;
  TilePlan best = {0, 1, steps};
  double least = -1;
  for (int i = 0; i < count; ++i) {
    const double tiles = tile_count(ways[i], p);
    for (int splits = 1; splits == 1 || (room > 0 && tiles * splits <= 1024 && splits <= 64 && splits * 4 <= steps);
         splits += splits < 4 ? 1 : splits / 2) {
      const int per = (steps + splits - 1) / splits, used = steps == 0 ? 1 : (steps + per - 1) / per;
      const TilePlan plan = {i, used, per};
      if (partial_bytes(plan, p.M, columns) > room) continue;
      const double cost = tile_cost(ways[i], tiles * used, per) + finish_cost(used, static_cast<double>(p.M) * columns);
      if (least < 0 || cost < least) best = plan, least = cost;
    }
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

// Which of `count` ways is done with all three first on 256 CUs, which take tiles as they come: a product's last tile
// begins when the whole rounds before it are over, of tiles as long as they are on average so far, and ends one
// of its own lengths later. x's gradient and the weights' are split into numbers of their own. room: bytes for
// partial sums; a plan with some is taken if it promises 5 % (the estimate is no better: with float32 kernels 7 % faster than today's
// a step T=1001, H=2048, I=768 took 207 us so and 228 where 4 % were enough; with today's it is 232 both ways). Against the best of all ways and
// splits of 110 random shapes a type this loses 2 to 3 % (bfloat16 on 160 more 2.1), the spread work plus half of the shortest tile, or the
// longest tile, 5 %.
struct GradsPlan {
  int way;
  TilePlan of[3];
};
inline GradsPlan plan_grads(const TileCost* ways, int count, int step, const FfnGrads& p, size_t room) {
  const GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  constexpr int OPTIONS = 6;  // 1, 2, 4, 8, 16, 32 splits; of the weights' gradients the first three
  GradsPlan best{};
  double least = -1;
  for (int i = 0; i < count; ++i) {
    const TileCost& way = ways[i];
    double tiles[3];
    TilePlan parts[3][OPTIONS];
    int options[3];
    for (int k = 0; k < 3; ++k) {
      const GemmArgs& g = *of[k];
      const int steps = (g.K + step - 1) / step;
      tiles[k] = g.M > 0 ? tile_count(way, g) : 0;
      options[k] = 0;
      for (int o = 0; o < (k == 0 ? OPTIONS : 3); ++o) {
        const int wanted = 1 << o, per = (steps + wanted - 1) / wanted;
        if (o > 0 && (wanted * 3 > steps || tiles[k] == 0 || room == 0)) break;
        parts[k][o] = {i, steps == 0 ? 1 : (steps + per - 1) / per, per};
        options[k] = o + 1;
      }
    }
    const int w_options = options[1] > options[2] ? options[1] : options[2];
    for (int ox = 0; ox < options[0]; ++ox) {
      for (int ow = 0; ow < w_options; ++ow) {
        const TilePlan* plan[3] = {&parts[0][ox], &parts[1][ow < options[1] ? ow : options[1] - 1],
                                   &parts[2][ow < options[2] ? ow : options[2] - 1]};
        double all = 0, bytes = 0;
        for (int k = 0; k < 3; ++k) {
          all += tiles[k] * plan[k]->splits;
          if (tiles[k] > 0 && plan[k]->splits > 1) bytes += static_cast<double>(partial_bytes(*plan[k], of[k]->M, of[k]->N));
        }
        if (bytes > static_cast<double>(room)) continue;
        const int each = all > 256.0 * (way.together - 1) ? way.together : all > 256 ? static_cast<int>((all + 255) / 256) : 1;
        const double one = each == 1 ? way.one : each == 2 ? way.two : each * way.more;
        const double slots = 256.0 * each;
        double done = 0, work = 0, end = 0;
        for (int k = 0; k < 3; ++k) {
          if (tiles[k] == 0) continue;
          const double n = tiles[k] * plan[k]->splits, length = plan[k]->per * one;
          done += n, work += n * length;
          const double last = static_cast<double>(static_cast<long long>((done - 1) / slots)) * (work / done) + length;
          end = end > last ? end : last;
        }
        const double cost = bytes > 0 ? 1.05 * (end + 3.0 + 2 * bytes / 4.5e6) : end;
        if (least < 0 || cost < least) best = {i, {*plan[0], *plan[1], *plan[2]}}, least = cost;
      }
    }
  }
  return best;
}

// Workgroup ranges and partial sums of a plan; the number of workgroups (each range begun on a multiple of 8, see
// tile_of). partial: plan_bytes of memory, or NULL without splits.
inline long long lay_out_grads(const GradsPlan& plan, const TileCost& way, FfnGrads& p, float* partial) {
  GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  long long at = 0;
  for (int i = 0; i < 3; ++i) {
    GemmArgs& g = *of[i];
    g.grid_m = (g.M + way.rows - 1) / way.rows;
    g.grid_n = (g.N + way.columns - 1) / way.columns;
    g.splits = plan.of[i].splits, g.per = plan.of[i].per, g.partial = partial;
    if (g.M > 0) partial += partial_bytes(plan.of[i], g.M, g.N) / 4;
    p.begin[i] = static_cast<int>(at < 0x7FFFFFFF ? at : 0x7FFFFFFF);
    at = (at + static_cast<long long>(g.grid_m) * g.grid_n * g.splits + 7) / 8 * 8;
  }
  return at;
}
inline size_t plan_bytes(const GradsPlan& plan, const FfnGrads& p) {
  const GemmArgs* of[] = {&p.dx, &p.dw13, &p.dw2};
  size_t bytes = 0;
  for (int i = 0; i < 3; ++i) bytes += of[i]->M > 0 ? partial_bytes(plan.of[i], of[i]->M, of[i]->N) : 0;
  return bytes;
}

// A matrix product in bfloat16 or float32 (k_outer_b: a row of B is one k); epi as above. *_bytes: memory for
// p.partial that a call with these sizes can use (0: none); room: how much of it there is (with p.partial NULL
// none): a call whose plan wants more takes one that wants less.
hipError_t launch_ffn_gemm(int dtype, bool k_outer_b, int epi, GemmArgs p, size_t room, hipStream_t stream);
size_t ffn_gemm_bytes(int dtype, bool k_outer_b, int epi, const GemmArgs& p);
hipError_t launch_ffn_gemm_f32(bool k_outer_b, int epi, const GemmArgs& p, size_t room, hipStream_t stream);
size_t ffn_gemm_f32_bytes(int epi, const GemmArgs& p);
// (partial: `room` bytes or NULL)
hipError_t launch_ffn_grads(int dtype, const FfnGrads& p, float* partial, size_t room, hipStream_t stream);
size_t ffn_grads_bytes(int dtype, const FfnGrads& p);
hipError_t launch_ffn_grads_f32(FfnGrads p, float* partial, size_t room, hipStream_t stream);
size_t ffn_grads_f32_bytes(const FfnGrads& p);
// What a split product's partial sums become; of the three gradients those that were split.
hipError_t launch_ffn_finish(int dtype, int epi, const GemmArgs& p, hipStream_t stream);
hipError_t launch_ffn_finish_grads(int dtype, const FfnGrads& p, hipStream_t stream);
// MXFP4 weights b times bfloat16 rows (x_mxfp4 false) or MXFP4 rows; EPI_STORE or EPI_GATED (bfloat16 rows only).
hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, const GemmArgs& p, size_t room, hipStream_t stream);
size_t mxfp4_gemm_bytes(bool x_mxfp4, int epi, const GemmArgs& p);
// The same for few rows, where these take the call (A and B with their k inside the rows).
bool ffn_skinny_takes(const GemmArgs& p);
bool mxfp4_skinny_takes(bool x_mxfp4, const GemmArgs& p);
hipError_t launch_ffn_skinny(int dtype, bool gated, const GemmArgs& p, hipStream_t stream);
hipError_t launch_mxfp4_skinny(bool x_mxfp4, bool gated, const GemmArgs& p, hipStream_t stream);
hipError_t launch_mxfp4_quantize(int dtype, const void* x, long long ldx, int rows, int k, void* codes, void* scales,
                                 hipStream_t stream);
hipError_t launch_mxfp4_dequantize(int dtype, const void* codes, const void* scales, int rows, int k, void* out,
                                   long long ldo, hipStream_t stream);

}  // namespace fmoe
