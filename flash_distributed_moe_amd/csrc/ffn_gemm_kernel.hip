// The matrix products of the dense gated feed-forward block in bfloat16.
#include "ffn_gemm_device.h"

namespace fmoe {

// Tile `id` of a product, by a workgroup with S::LDS_BYTES of LDS
template <class S>
__device__ __forceinline__ void gemm_tile(const GemmArgs& p, char* lds, int id) {
  int split, first, steps, tile_m, tile_n;
  share_of(p, (p.K + S::STEP - 1) / S::STEP, id, split, first, steps);
  tile_of(p, id, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS), tid = threadIdx.x % S::THREADS;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / S::WN, wn = wave % S::WN;
  char* mine = lds + group * 2 * S::STAGE_BYTES;

  TileLoader<S::KIND, S::OUTER_A, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<S::KIND, S::OUTER_B, S::BN, S::THREADS, S::FN, S::EPI == EPI_GATED> load_b;
  load_a.init(p.a, p.lda, m0, p.M, tid);
  load_b.init(p.b, p.ldb, n0, p.N, tid);

  Accumulators<S> acc;
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // a group's turns: stages group, group + GROUPS, ...
  const int turns = (steps + S::GROUPS - 1) / S::GROUPS;
  auto load = [&](int turn) {
    const int s = turn * S::GROUPS + group;
    if (S::GROUPS > 1 && s >= steps) return;
    char* to = mine + (turn & 1) * S::STAGE_BYTES;
    load_a.load(to, first + s, p.K - (first + s) * S::STEP);
    load_b.load(to + S::BM * 128, first + s, p.K - (first + s) * S::STEP);
  };
  if (turns > 0) load(0);
  for (int turn = 0; turn < turns; ++turn) {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's pieces of the stage have landed ...
    __syncthreads();                // ... and everybody's; all are done with the other buffer
    if (turn + 1 < turns) load(turn + 1);
    if (S::GROUPS > 1 && turn * S::GROUPS + group >= steps) continue;
    const char* now = mine + (turn & 1) * S::STAGE_BYTES;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Fragments<KIND_BF16, S::OUTER_B, S::BN, S::FN> b;
      Fragments<KIND_BF16, S::OUTER_A, S::BM, S::FM> a;
      if constexpr (!S::OUTER_A) a.read(now, wm * S::FM * 16, half);
      b.read(now + S::BM * 128, wn * S::FN * 16, half);
      if constexpr (S::OUTER_A) a.read(now, wm * S::FM * 16, half);
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn)
          acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b.v[fn]),
                                                                  __builtin_bit_cast(bf16x8, a.v[fm]), acc.v[fm][fn], 0, 0, 0);
    }
  }
  add_groups<S>(lds, group, acc);
  if (group != 0) return;
  if (p.splits > 1) write_partial<S>(p, split, m0, n0, acc);
  else write_results<S>(p, m0, n0, acc);
}

template <class S>
__global__ __launch_bounds__(S::THREADS * S::GROUPS) void ffn_gemm_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(128))) char lds[S::LDS_BYTES];
  gemm_tile<S>(p, lds, blockIdx.x);
}

// The gradients of x (a product with its weights' rows as k) and of both weights (sums over the tokens) in one
// launch: none waits for another, and the CUs that the last tiles of one leave empty take the next one's.
// The longest sums first.
template <int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM * WN * 64) void ffn_grads_kernel(FfnGrads p) {
  typedef GemmShape<KIND_BF16, false, true, EPI_STORE, WM, WN, FM, FN> X;
  typedef GemmShape<KIND_BF16, true, true, EPI_STORE, WM, WN, FM, FN> W;
  __shared__ __attribute__((aligned(128))) char lds[X::LDS_BYTES];
  const int id = blockIdx.x;
  if (id < p.begin[1]) {
    if (id < p.dx.grid_m * p.dx.grid_n * p.dx.splits) gemm_tile<X>(p.dx, lds, id);
  } else {
    const bool second = id >= p.begin[2];
    const GemmArgs& dw = second ? p.dw2 : p.dw13;
    const int at = id - p.begin[second ? 2 : 1];
    if (at < dw.grid_m * dw.grid_n * dw.splits) gemm_tile<W>(dw, lds, at);
  }
}

template <class S>
static hipError_t launch(GemmArgs p, const TilePlan& plan, hipStream_t stream) {
  p.grid_m = (p.M + S::BM - 1) / S::BM;
  p.grid_n = (p.N + S::CN - 1) / S::CN;
  p.splits = plan.splits, p.per = plan.per;
  const long long blocks = static_cast<long long>(p.grid_m) * p.grid_n * p.splits;
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL(ffn_gemm_kernel<S>, dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS * S::GROUPS), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.splits == 1 ? e : launch_ffn_finish(1, S::EPI, p, stream);
}

// Measured, 256 x 256 (sixteen waves) / 128 x 128 (eight) / 64 x 64 (four) rows of A and B, us: M=8192, N=4096, K=12288
// 575 / 754 / 1570; M=4096, N=2048, K=6144 124 / 88 / 140; M=333, N=1344, K=736 19.5 / 8.8 / 5.6. (256 x 128 and 128 x 256
// lie between their neighbours everywhere. 256 x 256 with eight waves takes 627: four waves a SIMD fill each
// other's waits for LDS and for the barrier; a third stage, which would not fit, or operands read ahead into
// registers gain nothing beside that. The library's product of that size takes 529.)
// Where CUs have one small tile or two, groups of waves share its k, 1 / 2 / 4 groups: M=64, N=2048, K=6144 28.2 / 20.9 / 17.9;
// M=1024 50.1 / 38.2 / 53.1; M=333, N=1344, K=736 6.0 / 5.5 / 5.8; 128 x 128 in 1 / 2: M=1024, N=2048, K=6144 65.1 / 52.2.
static const TileCost kWays[] = {{256, 256, 0, 1.45, 2.9, 1.45}, {128, 128, 0, 0.55, 0.96, 0.48}, {128, 128, 0.8, 0.45, 1.0, 0.55},
                                 {64, 64, 0, 0.33, 0.5, 0.21},   {64, 64, 0.8, 0.25, 0.37, 0.245}, {64, 64, 1.8, 0.2, 0.53, 0.27}};
static const TileCost kGatedWays[] = {{256, 128, 0, 1.45, 2.9, 1.45}, {128, 64, 0, 0.55, 0.96, 0.48}, {128, 64, 0.8, 0.45, 1.0, 0.55},
                                      {64, 32, 0, 0.33, 0.5, 0.21},   {64, 32, 0.8, 0.25, 0.37, 0.245}, {64, 32, 1.8, 0.2, 0.53, 0.27}};

static TilePlan plan(int epi, const GemmArgs& p, size_t room) {
  return plan_tiles(epi == EPI_GATED ? kGatedWays : kWays, 6, 64, p, epi == EPI_GATED ? 2 * p.N : p.N, room);
}

template <bool OB, int EPI>
static hipError_t pick(const GemmArgs& p, size_t room, hipStream_t stream) {
  const TilePlan chosen = plan(EPI, p, p.partial != nullptr ? room : 0);
  switch (chosen.way) {
    case 0: return launch<GemmShape<KIND_BF16, false, OB, EPI, 4, 4, 4, 4>>(p, chosen, stream);
    case 1: return launch<GemmShape<KIND_BF16, false, OB, EPI, 4, 2, 2, 4>>(p, chosen, stream);
    case 2: return launch<GemmShape<KIND_BF16, false, OB, EPI, 4, 2, 2, 4, 2>>(p, chosen, stream);
    case 3: return launch<GemmShape<KIND_BF16, false, OB, EPI, 2, 2, 2, 2>>(p, chosen, stream);
    case 4: return launch<GemmShape<KIND_BF16, false, OB, EPI, 2, 2, 2, 2, 2>>(p, chosen, stream);
    default: return launch<GemmShape<KIND_BF16, false, OB, EPI, 2, 2, 2, 2, 4>>(p, chosen, stream);
  }
}

static const TileCost kGradsWays[] = {{256, 256, 0, 1.55, 3.1, 1.55, 1}, {128, 128, 0, 0.6, 0.98, 0.49, 2}, {64, 64, 0, 0.33, 0.5, 0.22, 4}};

static hipError_t launch_ffn_grads_bf16(FfnGrads p, float* partial, size_t room, hipStream_t stream) {
  const GradsPlan chosen = plan_grads(kGradsWays, 3, 64, p, partial != nullptr ? room : 0);
  const long long blocks = lay_out_grads(chosen, kGradsWays[chosen.way], p, partial);
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (chosen.way == 0) hipLaunchKernelGGL((ffn_grads_kernel<4, 4, 4, 4>), grid, dim3(1024), 0, stream, p);
  else if (chosen.way == 1) hipLaunchKernelGGL((ffn_grads_kernel<4, 2, 2, 4>), grid, dim3(512), 0, stream, p);
  else hipLaunchKernelGGL((ffn_grads_kernel<2, 2, 2, 2>), grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : launch_ffn_finish_grads(1, p, stream);
}

hipError_t launch_ffn_gemm(int dtype, bool k_outer_b, int epi, GemmArgs p, size_t room, hipStream_t stream) {
  if (k_outer_b != (epi == EPI_SLOPE)) return hipErrorInvalidValue;
  if (!k_outer_b && ffn_skinny_takes(p)) return launch_ffn_skinny(dtype, epi == EPI_GATED, p, stream);
  if (dtype != 1) return launch_ffn_gemm_f32(k_outer_b, epi, p, room, stream);
  if (epi == EPI_SLOPE) return pick<true, EPI_SLOPE>(p, room, stream);
  return epi == EPI_GATED ? pick<false, EPI_GATED>(p, room, stream) : pick<false, EPI_STORE>(p, room, stream);
}

size_t ffn_gemm_bytes(int dtype, bool k_outer_b, int epi, const GemmArgs& p) {
  if (!k_outer_b && ffn_skinny_takes(p)) return 0;
  return dtype != 1 ? ffn_gemm_f32_bytes(epi, p) : partial_bytes(plan(epi, p, ~size_t{0}), p.M, epi == EPI_GATED ? 2 * p.N : p.N);
}

hipError_t launch_ffn_grads(int dtype, const FfnGrads& p, float* partial, size_t room, hipStream_t stream) {
  return dtype == 1 ? launch_ffn_grads_bf16(p, partial, room, stream) : launch_ffn_grads_f32(p, partial, room, stream);
}

size_t ffn_grads_bytes(int dtype, const FfnGrads& p) {
  return dtype != 1 ? ffn_grads_f32_bytes(p) : plan_bytes(plan_grads(kGradsWays, 3, 64, p, ~size_t{0}), p);
}

}  // namespace fmoe
