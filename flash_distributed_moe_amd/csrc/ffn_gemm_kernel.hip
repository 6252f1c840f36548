// The matrix products of the dense gated feed-forward block, bfloat16 and float32.
#include "ffn_gemm_device.h"

namespace fmoe {

template <class S>
__global__ __launch_bounds__(S::THREADS) void ffn_gemm_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(128))) char lds[2 * S::STAGE_BYTES];
  int tile_m, tile_n;
  tile_of(p, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;

  TileLoader<S::KIND, S::OUTER_A, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<S::KIND, S::OUTER_B, S::BN, S::THREADS, S::FN, S::EPI == EPI_GATED> load_b;
  load_a.init(p.a, p.lda, m0, p.M);
  load_b.init(p.b, p.ldb, n0, p.N);

  Accumulators<S> acc;
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int steps = (p.K + S::STEP - 1) / S::STEP;
  if (steps > 0) {
    load_a.load(lds, 0, p.K);
    load_b.load(lds + S::BM * 128, 0, p.K);
  }
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's pieces of stage s have landed ...
    __syncthreads();                // ... and everybody's; all are done with the other buffer
    char* next = lds + ((s + 1) & 1) * S::STAGE_BYTES;
    if (s + 1 < steps) {
      load_a.load(next, s + 1, p.K - (s + 1) * S::STEP);
      load_b.load(next + S::BM * 128, s + 1, p.K - (s + 1) * S::STEP);
    }
    const char* now = lds + (s & 1) * S::STAGE_BYTES;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Fragments<S::KIND, S::OUTER_B, S::BN, S::FN> b;
      Fragments<S::KIND, S::OUTER_A, S::BM, S::FM> a;
      b.read(now + S::BM * 128, wn * S::FN * 16, half);
      a.read(now, wm * S::FM * 16, half);
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn) {
          if constexpr (S::KIND == KIND_BF16) {
            acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b.v[fn]),
                                                                    __builtin_bit_cast(bf16x8, a.v[fm]), acc.v[fm][fn], 0, 0, 0);
          } else {
            const f32x4 bf = __builtin_bit_cast(f32x4, b.v[fn]), af = __builtin_bit_cast(f32x4, a.v[fm]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x4f32(bf[j], af[j], acc.v[fm][fn], 0, 0, 0);
          }
        }
    }
  }
  write_results<S>(p, m0, n0, acc);
}

template <class S>
static hipError_t launch(GemmArgs p, hipStream_t stream) {
  p.grid_m = (p.M + S::BM - 1) / S::BM;
  p.grid_n = (p.N + S::CN - 1) / S::CN;
  const long long blocks = static_cast<long long>(p.grid_m) * p.grid_n;
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL(ffn_gemm_kernel<S>, dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS), 0, stream, p);
  return hipGetLastError();
}

template <int KIND, bool OA, bool OB, int EPI>
static hipError_t pick(GemmArgs p, hipStream_t stream) {
  return launch<GemmShape<KIND, OA, OB, EPI, 2, 2, 4, 4>>(p, stream);
}

template <int KIND>
static hipError_t dispatch(bool oa, bool ob, int epi, const GemmArgs& p, hipStream_t stream) {
  if (epi == EPI_GATED) return oa || ob ? hipErrorInvalidValue : pick<KIND, false, false, EPI_GATED>(p, stream);
  if (epi == EPI_SLOPE) return oa || !ob ? hipErrorInvalidValue : pick<KIND, false, true, EPI_SLOPE>(p, stream);
  if (oa) return !ob ? hipErrorInvalidValue : pick<KIND, true, true, EPI_STORE>(p, stream);
  return ob ? pick<KIND, false, true, EPI_STORE>(p, stream) : pick<KIND, false, false, EPI_STORE>(p, stream);
}

hipError_t launch_ffn_gemm(int dtype, bool k_outer_a, bool k_outer_b, int epi, GemmArgs p, hipStream_t stream) {
  if (!k_outer_a && !k_outer_b && ffn_skinny_takes(dtype, p)) return launch_ffn_skinny(dtype, epi == EPI_GATED, p, stream);
  return dtype == 1 ? dispatch<KIND_BF16>(k_outer_a, k_outer_b, epi, p, stream)
                    : dispatch<KIND_F32>(k_outer_a, k_outer_b, epi, p, stream);
}

}  // namespace fmoe
