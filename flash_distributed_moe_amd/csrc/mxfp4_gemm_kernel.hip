// Matrix products with MXFP4 weights: 32 consecutive values of a row share a scale 2^(byte - 127), a
// value is 4 bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even one in its low half.
#include "ffn_gemm_device.h"

namespace fmoe {

// The scale byte of a lane's 32 k (block `kb` of `blocks`) of one of its rows. Behind the last block
// the values are zeros, and so must the scale be a number.
__device__ __forceinline__ unsigned scale_byte(const unsigned char* row, int kb, int blocks) {
  return kb < blocks ? row[kb] : 127u;
}

// MXFP4 rows times MXFP4 weights on the scaled matrix instructions: 16 x 16 x 128, a lane's operand is
// one block of 32 values (16 bytes) and that block's scale.
template <class S>
__global__ __launch_bounds__(S::THREADS) void mxfp4_both_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(128))) char lds[2 * S::STAGE_BYTES];
  int tile_m, tile_n;
  tile_of(p, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;

  TileLoader<S::KIND, false, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<S::KIND, false, S::BN, S::THREADS, S::FN, false> load_b;
  load_a.init(p.a, p.lda, m0, p.M);
  load_b.init(p.b, p.ldb, n0, p.N);
  const int blocks = p.K / 32;
  const unsigned char* scale_a[S::FM];
  const unsigned char* scale_b[S::FN];
#pragma unroll
  for (int f = 0; f < S::FM; ++f) {
    const int m = m0 + wm * S::FM * 16 + dealt_row<S::FM>(f, r);
    scale_a[f] = p.a_scales + static_cast<long long>(m < p.M ? m : 0) * blocks;
  }
#pragma unroll
  for (int f = 0; f < S::FN; ++f) {
    const int n = n0 + wn * S::FN * 16 + dealt_row<S::FN>(f, r);
    scale_b[f] = p.b_scales + static_cast<long long>(n < p.N ? n : 0) * blocks;
  }

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
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    char* next = lds + ((s + 1) & 1) * S::STAGE_BYTES;
    if (s + 1 < steps) {
      load_a.load(next, s + 1, p.K - (s + 1) * S::STEP);
      load_b.load(next + S::BM * 128, s + 1, p.K - (s + 1) * S::STEP);
    }
    const char* now = lds + (s & 1) * S::STAGE_BYTES;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Fragments<S::KIND, false, S::BN, S::FN> b;
      Fragments<S::KIND, false, S::BM, S::FM> a;
      b.read(now + S::BM * 128, wn * S::FN * 16, half);
      a.read(now, wm * S::FM * 16, half);
      unsigned sa[S::FM], sb[S::FN];
#pragma unroll
      for (int f = 0; f < S::FM; ++f) sa[f] = scale_byte(scale_a[f], s * 8 + half * 4 + g, blocks);
#pragma unroll
      for (int f = 0; f < S::FN; ++f) sb[f] = scale_byte(scale_b[f], s * 8 + half * 4 + g, blocks);
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn) {
          const i32x8 bv = {b.v[fn][0], b.v[fn][1], b.v[fn][2], b.v[fn][3], 0, 0, 0, 0};
          const i32x8 av = {a.v[fm][0], a.v[fm][1], a.v[fm][2], a.v[fm][3], 0, 0, 0, 0};
          acc.v[fm][fn] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bv, av, acc.v[fm][fn], 4, 4, 0, sb[fn], 0, sa[fm]);
        }
    }
  }
  write_results<S>(p, m0, n0, acc);
}

// bfloat16 rows times MXFP4 weights: the weights stay in 4 bits up to the wave that multiplies them and
// become bfloat16 there, which holds every one of their values. A step is 64 k, of which lane l takes
// the (l / 16)-th quarter: 16 weights (8 bytes) under one scale, and 16-byte pieces 2 (l / 16) and
// 2 (l / 16) + 1 of its rows of A.
template <int ROWS, int THREADS, int F, bool GATED>
struct CodeLoader {
  static constexpr int PIECES = ROWS * 2 / THREADS;
  static_assert(PIECES * THREADS == ROWS * 2, "whole pieces a thread");
  unsigned offset[PIECES];
  const char* base;
  long long up_bytes;

  __device__ __forceinline__ void init(const void* p, long long ld, int row0, int rows) {
    base = static_cast<const char*>(p) + row0 * ld / 2;
    up_bytes = GATED ? rows * ld / 2 : 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + threadIdx.x, block = at >> 5, r = at & 15, half = (at >> 4) & 1, f = block % F;
      const int src = GATED ? block / F * (8 * F) + gated_row<F>(f, r) : block / F * (16 * F) + dealt_row<F>(f, r);
      offset[i] = row0 + src < rows ? static_cast<unsigned>(src * ld / 2) + half * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void load(char* lds, int s, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int half = (threadIdx.x >> 4) & 1;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      // a wave loads two blocks of 16 rows, which the gated kernels' F >= 4 keep on one side
      const int f = ((i * THREADS + wave * 64) >> 5) % F;
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + s * 32 + (GATED && f >= F / 2 ? up_bytes : 0), 0x7FFFFFFFu);
      load_to_lds16(rs, lds + wave * 1024 + i * THREADS * 16, half * 32 < left ? offset[i] : kOutside);
    }
  }
};

template <class S>
__global__ __launch_bounds__(S::THREADS) void mxfp4_weights_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(128))) char lds[2 * (S::BM * 128 + S::BN * 32)];
  constexpr bool GATED = S::EPI == EPI_GATED;
  constexpr int STAGE = S::BM * 128 + S::BN * 32;
  static_assert(S::FN % 4 == 0, "pairs of blocks on one side");
  int tile_m, tile_n;
  tile_of(p, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;

  TileLoader<KIND_BF16, false, S::BM, S::THREADS, S::FM, false> load_a;
  CodeLoader<S::BN, S::THREADS, S::FN, GATED> load_b;
  load_a.init(p.a, p.lda, m0, p.M);
  load_b.init(p.b, p.ldb, n0, p.N);
  const int blocks = p.K / 32;
  const unsigned char* scale_b[S::FN];
#pragma unroll
  for (int f = 0; f < S::FN; ++f) {
    const int n = GATED ? n0 + wn * S::FN * 8 + gated_row<S::FN>(f, r) : n0 + wn * S::FN * 16 + dealt_row<S::FN>(f, r);
    const int row = n < p.N ? n + (GATED && f >= S::FN / 2 ? p.N : 0) : 0;
    scale_b[f] = p.b_scales + static_cast<long long>(row) * blocks;
  }

  Accumulators<S> acc;
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int steps = (p.K + 63) / 64;
  if (steps > 0) {
    load_a.load(lds, 0, p.K);
    load_b.load(lds + S::BM * 128, 0, p.K);
  }
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    char* next = lds + ((s + 1) & 1) * STAGE;
    if (s + 1 < steps) {
      load_a.load(next, s + 1, p.K - (s + 1) * 64);
      load_b.load(next + S::BM * 128, s + 1, p.K - (s + 1) * 64);
    }
    const char* now = lds + (s & 1) * STAGE;
    u32x2 codes[S::FN];
    float scale[S::FN];
#pragma unroll
    for (int f = 0; f < S::FN; ++f) {
      codes[f] = *(const FFN_LDS u32x2*)(now + S::BM * 128 + (wn * S::FN + f) * 512 + (g >> 1) * 256 + r * 16 + (g & 1) * 8);
      scale[f] = __uint_as_float(scale_byte(scale_b[f], s * 2 + (g >> 1), blocks) << 23);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      bf16x8 b[S::FN];
#pragma unroll
      for (int f = 0; f < S::FN; ++f) {
        const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[f][half], scale[f], 0);
        const bf16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[f][half], scale[f], 1);
        const bf16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[f][half], scale[f], 2);
        const bf16x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes[f][half], scale[f], 3);
        b[f] = bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
      }
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm) {
        const bf16x8 a = *(const FFN_LDS bf16x8*)(now + ((wm * S::FM + fm) * 16 + r) * 128 + (((2 * g + half) ^ (r & 7)) << 4));
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn)
          acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[fn], a, acc.v[fm][fn], 0, 0, 0);
      }
    }
  }
  write_results<S>(p, m0, n0, acc);
}

template <class S, typename Kernel>
static hipError_t launch(Kernel kernel, GemmArgs p, hipStream_t stream) {
  p.grid_m = (p.M + S::BM - 1) / S::BM;
  p.grid_n = (p.N + S::CN - 1) / S::CN;
  const long long tiles = static_cast<long long>(p.grid_m) * p.grid_n;
  if (tiles == 0) return hipSuccess;
  if (tiles > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles)), dim3(S::THREADS), 0, stream, p);
  return hipGetLastError();
}

hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, GemmArgs p, hipStream_t stream) {
  if (x_mxfp4 && epi != EPI_STORE) return hipErrorInvalidValue;
  if (mxfp4_skinny_takes(x_mxfp4, p)) return launch_mxfp4_skinny(x_mxfp4, epi == EPI_GATED, p, stream);
  if (x_mxfp4) {
    typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 2, 2, 4, 4> S;
    return launch<S>(mxfp4_both_kernel<S>, p, stream);
  }
  if (epi == EPI_GATED) {
    typedef GemmShape<KIND_BF16, false, false, EPI_GATED, 2, 2, 4, 4> S;
    return launch<S>(mxfp4_weights_kernel<S>, p, stream);
  }
  typedef GemmShape<KIND_BF16, false, false, EPI_STORE, 2, 2, 4, 4> S;
  return launch<S>(mxfp4_weights_kernel<S>, p, stream);
}

}  // namespace fmoe
