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
  tile_of(p, blockIdx.x, tile_m, tile_n);
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
  static constexpr int PIECES = (ROWS * 2 + THREADS - 1) / THREADS;
  static constexpr int BYTES = PIECES * THREADS * 16;  // in LDS; behind the rows, zeros
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
      offset[i] = block * 16 < ROWS && row0 + src < rows ? static_cast<unsigned>(src * ld / 2) + half * 16 : kOutside;
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

__device__ __forceinline__ bf16x8 eight_values(unsigned codes, float scale) {
  const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

template <class S>
__global__ __launch_bounds__(S::THREADS) void mxfp4_weights_kernel(GemmArgs p) {
  constexpr bool GATED = S::EPI == EPI_GATED;
  constexpr int STAGE = S::BM * 128 + CodeLoader<S::BN, S::THREADS, S::FN, GATED>::BYTES;
  __shared__ __attribute__((aligned(128))) char lds[2 * STAGE];
  static_assert(S::FN % 4 == 0, "pairs of blocks on one side");
  int tile_m, tile_n;
  tile_of(p, blockIdx.x, tile_m, tile_n);
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
      for (int f = 0; f < S::FN; ++f) b[f] = eight_values(codes[f][half], scale[f]);
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

// ------------------------------------------------------------------ scales on 4-byte boundaries
// The kernels below take their scales through LDS, 8 bytes of a row (256 k) a stage: 2 KiB for 256 rows, a load of
// 4 bytes a lane. That wants rows of scales on 4 bytes: K a multiple of 128. (The ones above read single bytes
// from memory whenever they need one, and wait for them: 258 us against 105 at M=2048, N=8192, K=4096.)
template <int ROWS, int THREADS, int F, bool GATED>
struct ScaleLoader {
  static constexpr int PIECES = (ROWS * 2 + THREADS - 1) / THREADS;
  static constexpr int BYTES = PIECES * THREADS * 4;  // in LDS; behind the rows, zeros
  unsigned offset[PIECES];
  const unsigned char* base;
  int blocks;

  __device__ __forceinline__ void init(const unsigned char* p, int row0, int rows, int blocks_) {
    blocks = blocks_;
    base = p + static_cast<long long>(row0) * blocks;
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + tid, row = at >> 1, f = row % (16 * F) >> 4, r = row & 15;
      const int src = GATED ? row / (16 * F) * (8 * F) + gated_row<F>(f, r) : row / (16 * F) * (16 * F) + dealt_row<F>(f, r);
      offset[i] = row < ROWS && row0 + src < rows ? static_cast<unsigned>(src * blocks) + (at & 1) * 4 : kOutside;
    }
    up = GATED ? static_cast<long long>(rows) * blocks : 0;
  }
  long long up;

  // the 8 blocks from `first` (a multiple of 8) on
  __device__ __forceinline__ void load(char* lds, int first) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = first + (threadIdx.x & 1) * 4 < blocks;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int f = ((i * THREADS + wave * 64) >> 1) % (16 * F) >> 4;  // a wave loads two blocks of 16 rows, on one side
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base + first + (GATED && f >= F / 2 ? up : 0), 0x7FFFFFFFu);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (FFN_LDS void*)(lds + (wave * 64 + i * THREADS) * 4), 4,
                                               static_cast<int>(in ? offset[i] : kOutside), 0, 0, 0);
    }
  }
};

__device__ __forceinline__ unsigned lds_byte(const char* p) { return *(const FFN_LDS unsigned char*)p; }

template <class S>
__global__ __launch_bounds__(S::THREADS) void mxfp4_both_tiled_kernel(GemmArgs p) {
  typedef ScaleLoader<S::BM, S::THREADS, S::FM, false> ScaleA;
  typedef ScaleLoader<S::BN, S::THREADS, S::FN, false> ScaleB;
  constexpr int TILES = S::STAGE_BYTES, STAGE = TILES + ScaleA::BYTES + ScaleB::BYTES;
  __shared__ __attribute__((aligned(128))) char lds[2 * STAGE];
  int tile_m, tile_n;
  tile_of(p, blockIdx.x, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;

  TileLoader<S::KIND, false, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<S::KIND, false, S::BN, S::THREADS, S::FN, false> load_b;
  ScaleA scale_a;
  ScaleB scale_b;
  load_a.init(p.a, p.lda, m0, p.M);
  load_b.init(p.b, p.ldb, n0, p.N);
  scale_a.init(p.a_scales, m0, p.M, p.K / 32);
  scale_b.init(p.b_scales, n0, p.N, p.K / 32);

  Accumulators<S> acc;
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int steps = (p.K + S::STEP - 1) / S::STEP;
  auto load = [&](int s) {
    char* to = lds + (s & 1) * STAGE;
    load_a.load(to, s, p.K - s * S::STEP);
    load_b.load(to + S::BM * 128, s, p.K - s * S::STEP);
    scale_a.load(to + TILES, s * 8);
    scale_b.load(to + TILES + ScaleA::BYTES, s * 8);
  };
  if (steps > 0) load(0);
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
    const char* now = lds + (s & 1) * STAGE;
    const char* sa_at = now + TILES + (wm * S::FM * 16 + r) * 8 + g;
    const char* sb_at = now + TILES + ScaleA::BYTES + (wn * S::FN * 16 + r) * 8 + g;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Fragments<S::KIND, false, S::BN, S::FN> b;
      Fragments<S::KIND, false, S::BM, S::FM> a;
      unsigned sa[S::FM], sb[S::FN];
      b.read(now + S::BM * 128, wn * S::FN * 16, half);
      a.read(now, wm * S::FM * 16, half);
#pragma unroll
      for (int f = 0; f < S::FN; ++f) sb[f] = lds_byte(sb_at + f * 128 + half * 4);
#pragma unroll
      for (int f = 0; f < S::FM; ++f) sa[f] = lds_byte(sa_at + f * 128 + half * 4);
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

// The k loop of bfloat16 rows times MXFP4 weights. A stage is multiplied in four parts, two halves of its k for two
// halves of the wave's rows of A, each part while the next one's operands come from LDS. Before the last part
// all of the stage is in registers, and its buffer is loaded with the stage after next. (With eight waves,
// which convert each weight twice; sixteen, in the plain loop of the other kernels, convert it four times:
// M=2048, N=8192, K=4096 113 us and 125.) LOADS: load instructions of a wave for a stage.
template <int LOADS, class A, class B, class Load, class ReadA, class ReadB, class Multiply>
__device__ __forceinline__ void stage_loop(int steps, Load load, ReadA read_a, ReadB read_b, Multiply multiply) {
  if (steps == 0) return;
  A a0, a1;
  B b0, b1;
  load(0);
  if (steps > 1) load(1);
  // stage 0 has landed when no more than the other's loads are on their way
  if (steps > 1) asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __builtin_amdgcn_s_barrier();
  read_b(b0, 0, 0);
  read_a(a0, 0, 0, 0);
  for (int s = 0; s < steps; ++s) {
    read_a(a1, s, 0, 1);
    multiply(a0, b0, 0);
    read_b(b1, s, 1);
    read_a(a0, s, 1, 0);
    multiply(a1, b0, 1);
    read_a(a1, s, 1, 1);
    multiply(a0, b1, 0);
    // stage s + 1 has landed, stage s is read
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_barrier();
    if (s + 2 < steps) load(s + 2);
    if (s + 1 < steps) {
      read_b(b0, s + 1, 0);
      read_a(a0, s + 1, 0, 0);
    }
    multiply(a1, b1, 1);
  }
}

template <class S>
__global__ __launch_bounds__(S::THREADS) void mxfp4_weights_tiled_kernel(GemmArgs p) {
  constexpr bool GATED = S::EPI == EPI_GATED;
  typedef CodeLoader<S::BN, S::THREADS, S::FN, GATED> Codes;
  typedef ScaleLoader<S::BN, S::THREADS, S::FN, GATED> ScaleB;
  constexpr int TILES = S::BM * 128 + Codes::BYTES, STAGE = TILES + ScaleB::BYTES;
  static_assert(S::FN % 4 == 0, "pairs of blocks on one side");
  __shared__ __attribute__((aligned(128))) char lds[2 * STAGE];
  int tile_m, tile_n;
  tile_of(p, blockIdx.x, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;

  TileLoader<KIND_BF16, false, S::BM, S::THREADS, S::FM, false> load_a;
  Codes load_b;
  ScaleB scale_b;
  load_a.init(p.a, p.lda, m0, p.M);
  load_b.init(p.b, p.ldb, n0, p.N);
  scale_b.init(p.b_scales, n0, p.N, p.K / 32);

  Accumulators<S> acc;
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  constexpr int HM = S::FM / 2, LOADS = S::BM * 8 / S::THREADS + Codes::PIECES + ScaleB::PIECES;
  struct A {
    bf16x8 v[HM];
  };
  struct B {
    unsigned codes[S::FN];
    float scale[S::FN];
  };
  stage_loop<LOADS, A, B>(
      (p.K + 63) / 64,
      [&](int s) {
        char* to = lds + (s & 1) * STAGE;
        load_a.load(to, s, p.K - s * 64);
        load_b.load(to + S::BM * 128, s, p.K - s * 64);
        scale_b.load(to + TILES, s * 2 & ~7);
      },
      [&](A& a, int s, int half, int group) {
#pragma unroll
        for (int f = 0; f < HM; ++f)
          a.v[f] = *(const FFN_LDS bf16x8*)(lds + (s & 1) * STAGE + ((wm * S::FM + group * HM + f) * 16 + r) * 128 +
                                            (((2 * g + half) ^ (r & 7)) << 4));
      },
      [&](B& b, int s, int half) {
        const char* from = lds + (s & 1) * STAGE;
#pragma unroll
        for (int f = 0; f < S::FN; ++f) {
          const int block = wn * S::FN + f;
          b.codes[f] = *(const FFN_LDS unsigned*)(from + S::BM * 128 + block * 512 + (g >> 1) * 256 + r * 16 + (g & 1) * 8 + half * 4);
          b.scale[f] = __uint_as_float(lds_byte(from + TILES + (block * 16 + r) * 8 + (s * 2 & 7) + (g >> 1)) << 23);
        }
      },
      [&](const A& a, const B& b, int group) {
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn) {
          const bf16x8 w = eight_values(b.codes[fn], b.scale[fn]);
#pragma unroll
          for (int fm = 0; fm < HM; ++fm) {
            f32x4& c = acc.v[group * HM + fm][fn];
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, a.v[fm], c, 0, 0, 0);
          }
        }
      });
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

// Whether both kinds of scales can be read 4 bytes at a time
static bool scales_on_fours(const GemmArgs& p) {
  const auto fours = [](const void* a) { return (reinterpret_cast<unsigned long long>(a) & 3) == 0; };
  return p.K % 128 == 0 && fours(p.b_scales) && fours(p.a_scales);
}

// Measured at M=2048, N=8192, K=4096, 256 x 256 (eight waves) / 128 x 128 (four): 113 / 134 us; M=256 94 / 46.
template <int EPI>
static hipError_t launch_weights(const GemmArgs& p, hipStream_t stream) {
  constexpr int PER = EPI == EPI_GATED ? 2 : 1;
  typedef GemmShape<KIND_BF16, false, false, EPI, 2, 2, 4, 4> Small;
  typedef GemmShape<KIND_BF16, false, false, EPI, 2, 4, 8, 4> Large;
  if (!scales_on_fours(p)) return launch<Small>(mxfp4_weights_kernel<Small>, p, stream);
  static const TileCost ways[] = {{256, 256 / PER, 1.75, 1.75}, {128, 128 / PER, 0.68, 0.52}};
  if (pick_tile(ways, 2, p.M, p.N) == 0) return launch<Large>(mxfp4_weights_tiled_kernel<Large>, p, stream);
  return launch<Small>(mxfp4_weights_tiled_kernel<Small>, p, stream);
}

// Measured at M=4096, N=8192, K=4096, 256 x 256 (sixteen waves) / 128 x 128 (four): 80.5 / 93.1 us; M=512 31.5 / 18.0.
static hipError_t launch_both(const GemmArgs& p, hipStream_t stream) {
  typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 2, 2, 4, 4> Small;
  typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 4, 4, 4, 4> Large;
  if (!scales_on_fours(p)) return launch<Small>(mxfp4_both_kernel<Small>, p, stream);
  static const TileCost ways[] = {{256, 256, 2.4, 2.4}, {128, 128, 1.0, 0.73}};
  if (pick_tile(ways, 2, p.M, p.N) == 0) return launch<Large>(mxfp4_both_tiled_kernel<Large>, p, stream);
  return launch<Small>(mxfp4_both_tiled_kernel<Small>, p, stream);
}

hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, GemmArgs p, hipStream_t stream) {
  if (x_mxfp4 && epi != EPI_STORE) return hipErrorInvalidValue;
  if (mxfp4_skinny_takes(x_mxfp4, p)) return launch_mxfp4_skinny(x_mxfp4, epi == EPI_GATED, p, stream);
  if (x_mxfp4) return launch_both(p, stream);
  return epi == EPI_GATED ? launch_weights<EPI_GATED>(p, stream) : launch_weights<EPI_STORE>(p, stream);
}

}  // namespace fmoe
