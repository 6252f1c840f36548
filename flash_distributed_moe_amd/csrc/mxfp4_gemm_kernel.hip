// Matrix products of many rows with MXFP4 weights: 32 consecutive values of a row share a scale 2^(byte - 127), a
// value is 4 bits (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), two to a byte, the even one in its low half.
//
// MXFP4 rows go through the scaled matrix instructions, 16 x 16 x 128: a lane's operand is one block of 32 values
// (16 bytes) and that block's scale, and a step of 256 k has the bfloat16 kernels' 128 bytes a row.
// With bfloat16 rows the weights stay in 4 bits up to the wave that multiplies them and become bfloat16
// there, which holds every one of their values. A step is 64 k, of which lane l takes the (l / 16)-th
// quarter: 16 weights (8 bytes) under one scale, and 16-byte pieces 2 (l / 16) and 2 (l / 16) + 1 of its rows of A.
//
// Scales go through LDS, byte by byte through registers, a stage ahead. (Read from memory by the lane that needs one,
// when it needs it, they had taken more time than everything else: M=2048, N=8192, K=4096 250 us instead of 112.) Of
// two operands in 4 bits there are as many scales as make that felt, and where rows of scales begin on 4 bytes (K a
// multiple of 128) they are loaded 4 at a time straight to LDS: M=4096, N=8192, K=4096 99 us by bytes, 86 by fours.
#include "ffn_gemm_device.h"

namespace fmoe {

__device__ __forceinline__ unsigned lds_byte(const char* p) { return *(const FFN_LDS unsigned char*)p; }

__device__ __forceinline__ bf16x8 eight_values(unsigned codes, float scale) {
  const bf16x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const bf16x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const bf16x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const bf16x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return bf16x8{v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
}

// The weights' codes of bfloat16 rows' products: of each block of 16 rows a step's first 16 bytes, then the other 16.
template <int ROWS, int THREADS, int F, bool GATED>
struct CodeLoader {
  static constexpr int PIECES = (ROWS * 2 + THREADS - 1) / THREADS;
  static constexpr int BYTES = PIECES * THREADS * 16;  // in LDS; behind the rows, zeros
  unsigned offset[PIECES];
  const char* base;
  long long up_bytes;
  int tid;

  __device__ __forceinline__ void init(const void* p, long long ld, int row0, int rows, int tid_) {
    tid = tid_;
    base = static_cast<const char*>(p) + row0 * ld / 2;
    up_bytes = GATED ? rows * ld / 2 : 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + tid, block = at >> 5, r = at & 15, half = (at >> 4) & 1, f = block % F;
      const int src = GATED ? block / F * (8 * F) + gated_row<F>(f, r) : block / F * (16 * F) + dealt_row<F>(f, r);
      offset[i] = block * 16 < ROWS && row0 + src < rows ? static_cast<unsigned>(src * ld / 2) + half * 16 : kOutside;
    }
  }
  __device__ __forceinline__ void load(char* lds, int s, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int half = (tid >> 4) & 1;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      // a wave loads two blocks of 16 rows, which the gated kernels' F >= 4 keep on one side
      const int f = ((i * THREADS + wave * 64) >> 5) % F;
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(base + s * 32 + (GATED && f >= F / 2 ? up_bytes : 0), 0x7FFFFFFFu);
      load_to_lds16(rs, lds + wave * 1024 + i * THREADS * 16, half * 32 < left ? offset[i] : kOutside);
    }
  }
};

// Which row of the matrix (gated: which column of C) lies at `row` of a tile, from its first one
template <int F, bool GATED>
__device__ __forceinline__ int row_of_tile(int row) {
  const int f = row % (16 * F) >> 4, r = row & 15;
  return GATED ? row / (16 * F) * (8 * F) + gated_row<F>(f, r) : row / (16 * F) * (16 * F) + dealt_row<F>(f, r);
}

// A tile's scales, PER blocks of a row a step; block kb lies at byte kb % 8 of its row's 8. Behind the last block of a row
// the values are zeros, and so must the scale be a number: zero is one.
template <int ROWS, int THREADS, int F, bool GATED, int PER, bool FOURS>
struct ScaleLoader;

template <int ROWS, int THREADS, int F, bool GATED, int PER>
struct ScaleLoader<ROWS, THREADS, F, GATED, PER, true> {
  static constexpr int PIECES = (ROWS * 2 + THREADS - 1) / THREADS;
  static constexpr int BYTES = PIECES * THREADS * 4;  // in LDS; behind the rows, zeros
  unsigned offset[PIECES];
  const unsigned char* base;
  long long up;
  int blocks, tid;

  __device__ __forceinline__ void init(const unsigned char* p, int row0, int rows, int blocks_, int tid_) {
    blocks = blocks_, tid = tid_;
    base = p + static_cast<long long>(row0) * blocks;
    up = GATED ? static_cast<long long>(rows) * blocks : 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + tid, row = at >> 1, src = row_of_tile<F, GATED>(row);
      offset[i] = row < ROWS && row0 + src < rows ? static_cast<unsigned>(src * blocks) + (at & 1) * 4 : kOutside;
    }
  }
  // a step's blocks and, where they are fewer, the rest of the row's 8
  __device__ __forceinline__ void load(char* lds, int s) {
    const int first = s * PER & ~7, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool in = first + (tid & 1) * 4 < blocks;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int f = ((i * THREADS + wave * 64) >> 1) % (16 * F) >> 4;  // a wave loads two blocks of 16 rows, on one side
      const __amdgpu_buffer_rsrc_t r = make_rsrc(base + first + (GATED && f >= F / 2 ? up : 0), 0x7FFFFFFFu);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (FFN_LDS void*)(lds + (wave * 64 + i * THREADS) * 4), 4,
                                               static_cast<int>(in ? offset[i] : kOutside), 0, 0, 0);
    }
  }
  __device__ __forceinline__ void landed(char*, int) const {}
};

template <int ROWS, int THREADS, int F, bool GATED, int PER>
struct ScaleLoader<ROWS, THREADS, F, GATED, PER, false> {
  static constexpr int PIECES = (ROWS * PER + THREADS - 1) / THREADS, BYTES = ROWS * 8;
  unsigned value[PIECES];
  const unsigned char* base;
  long long up;
  int blocks, tid, left;  // left: rows from this tile's first one on

  __device__ __forceinline__ void init(const unsigned char* p, int row0, int rows, int blocks_, int tid_) {
    blocks = blocks_, tid = tid_, left = rows - row0;
    base = p + static_cast<long long>(row0) * blocks;
    up = GATED ? static_cast<long long>(rows) * blocks : 0;
  }
  __device__ __forceinline__ void load(char*, int s) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + tid, row = at / PER, kb = s * PER + at % PER, src = row_of_tile<F, GATED>(row);
      const bool in = row < ROWS && src < left && kb < blocks;
      const long long from = static_cast<long long>(src) * blocks + kb + (GATED && row % (16 * F) / 16 >= F / 2 ? up : 0);
      value[i] = in ? base[from] : 0u;
    }
  }
  // what load asked for, to LDS: behind the wait for it, before the barrier
  __device__ __forceinline__ void landed(char* lds, int s) const {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int at = i * THREADS + tid, row = at / PER, kb = s * PER + at % PER;
      if (row < ROWS) *(FFN_LDS unsigned char*)(lds + row * 8 + (kb & 7)) = static_cast<unsigned char>(value[i]);
    }
  }
};

template <class S>
__device__ __forceinline__ void clear(Accumulators<S>& acc) {
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

template <class S, bool FOURS>
__global__ __launch_bounds__(S::THREADS * S::GROUPS) void mxfp4_both_kernel(GemmArgs p) {
  typedef ScaleLoader<S::BM, S::THREADS, S::FM, false, 8, FOURS> ScaleA;
  typedef ScaleLoader<S::BN, S::THREADS, S::FN, false, 8, FOURS> ScaleB;
  constexpr int TILES = S::STAGE_BYTES, STAGE = TILES + ScaleA::BYTES + ScaleB::BYTES;
  __shared__ __attribute__((aligned(128))) char lds[2 * S::GROUPS * STAGE];
  int id = blockIdx.x, split, first, steps, tile_m, tile_n;
  share_of(p, (p.K + S::STEP - 1) / S::STEP, id, split, first, steps);
  tile_of(p, id, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS), tid = threadIdx.x % S::THREADS;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / S::WN, wn = wave % S::WN;
  char* mine = lds + group * 2 * STAGE;

  TileLoader<S::KIND, false, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<S::KIND, false, S::BN, S::THREADS, S::FN, false> load_b;
  ScaleA scale_a;
  ScaleB scale_b;
  load_a.init(p.a, p.lda, m0, p.M, tid);
  load_b.init(p.b, p.ldb, n0, p.N, tid);
  scale_a.init(p.a_scales, m0, p.M, p.K / 32, tid);
  scale_b.init(p.b_scales, n0, p.N, p.K / 32, tid);
  Accumulators<S> acc;
  clear(acc);

  const int turns = (steps + S::GROUPS - 1) / S::GROUPS;
  auto load = [&](int turn) {
    const int s = turn * S::GROUPS + group;
    if (S::GROUPS > 1 && s >= steps) return;
    char* to = mine + (turn & 1) * STAGE;
    load_a.load(to, first + s, p.K - (first + s) * S::STEP);
    load_b.load(to + S::BM * 128, first + s, p.K - (first + s) * S::STEP);
    scale_a.load(to + TILES, first + s);
    scale_b.load(to + TILES + ScaleA::BYTES, first + s);
  };
  load(0);
  for (int turn = 0; turn < turns; ++turn) {
    const int s = turn * S::GROUPS + group;
    char* now = mine + (turn & 1) * STAGE;
    __builtin_amdgcn_s_waitcnt(0);  // this wave's pieces of the stage have landed ...
    if (S::GROUPS == 1 || s < steps) {
      scale_a.landed(now + TILES, first + s);
      scale_b.landed(now + TILES + ScaleA::BYTES, first + s);
    }
    __syncthreads();  // ... and everybody's; all are done with the other buffer
    if (turn + 1 < turns) load(turn + 1);
    if (S::GROUPS > 1 && s >= steps) continue;
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
  add_groups<S>(lds, group, acc);
  if (group != 0) return;
  if (p.splits > 1) write_partial<S>(p, split, m0, n0, acc);
  else write_results<S, S::EPI == EPI_STORE>(p, m0, n0, acc);
}

template <class S>
__global__ __launch_bounds__(S::THREADS * S::GROUPS) void mxfp4_weights_kernel(GemmArgs p) {
  constexpr bool GATED = S::EPI == EPI_GATED;
  typedef CodeLoader<S::BN, S::THREADS, S::FN, GATED> Codes;
  typedef ScaleLoader<S::BN, S::THREADS, S::FN, GATED, 2, false> ScaleB;
  constexpr int TILES = S::BM * 128 + Codes::BYTES, STAGE = TILES + ScaleB::BYTES;
  constexpr int SUMS = (S::GROUPS - 1) * S::BM * S::BN * 4, ALL = 2 * S::GROUPS * STAGE;
  static_assert(S::FN % 4 == 0, "pairs of blocks on one side");
  __shared__ __attribute__((aligned(128))) char lds[SUMS > ALL ? SUMS : ALL];
  int id = blockIdx.x, split, first, steps, tile_m, tile_n;
  share_of(p, (p.K + 64 - 1) / 64, id, split, first, steps);
  tile_of(p, id, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS), tid = threadIdx.x % S::THREADS;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / S::WN, wn = wave % S::WN;
  char* mine = lds + group * 2 * STAGE;

  TileLoader<KIND_BF16, false, S::BM, S::THREADS, S::FM, false> load_a;
  Codes load_b;
  ScaleB scale_b;
  load_a.init(p.a, p.lda, m0, p.M, tid);
  load_b.init(p.b, p.ldb, n0, p.N, tid);
  scale_b.init(p.b_scales, n0, p.N, p.K / 32, tid);
  Accumulators<S> acc;
  clear(acc);

  const int turns = (steps + S::GROUPS - 1) / S::GROUPS;
  auto load = [&](int turn) {
    const int s = turn * S::GROUPS + group;
    if (S::GROUPS > 1 && s >= steps) return;
    char* to = mine + (turn & 1) * STAGE;
    load_a.load(to, first + s, p.K - (first + s) * 64);
    load_b.load(to + S::BM * 128, first + s, p.K - (first + s) * 64);
    scale_b.load(to + TILES, first + s);
  };
  // rows of A and weights of a stage's half from LDS
  auto a_at = [&](const char* now, int fm, int half) {
    return *(const FFN_LDS bf16x8*)(now + ((wm * S::FM + fm) * 16 + r) * 128 + (((2 * g + half) ^ (r & 7)) << 4));
  };
  auto codes_at = [&](const char* now, int fn) { return now + S::BM * 128 + (wn * S::FN + fn) * 512 + (g >> 1) * 256 + r * 16 + (g & 1) * 8; };
  auto scale_at = [&](const char* now, int fn, int s) {
    return __uint_as_float(lds_byte(now + TILES + ((wn * S::FN + fn) * 16 + r) * 8 + (s * 2 & 7) + (g >> 1)) << 23);
  };
  load(0);
  for (int turn = 0; turn < turns; ++turn) {
    const int s = turn * S::GROUPS + group;
    char* now = mine + (turn & 1) * STAGE;
    __builtin_amdgcn_s_waitcnt(0);
    if (S::GROUPS == 1 || s < steps) scale_b.landed(now + TILES, first + s);
    __syncthreads();
    if (turn + 1 < turns) load(turn + 1);
    if (S::GROUPS > 1 && s >= steps) continue;
    u32x2 codes[S::FN];
    float scale[S::FN];
#pragma unroll
    for (int f = 0; f < S::FN; ++f) {
      codes[f] = *(const FFN_LDS u32x2*)codes_at(now, f);
      scale[f] = scale_at(now, f, first + s);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      bf16x8 b[S::FN];
#pragma unroll
      for (int f = 0; f < S::FN; ++f) b[f] = eight_values(codes[f][half], scale[f]);
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm) {
        const bf16x8 a = a_at(now, fm, half);
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn)
          acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[fn], a, acc.v[fm][fn], 0, 0, 0);
      }
    }
  }
  add_groups<S, sizeof(lds)>(lds, group, acc);
  if (group != 0) return;
  if (p.splits > 1) write_partial<S>(p, split, m0, n0, acc);
  else write_results<S, S::EPI == EPI_STORE>(p, m0, n0, acc);
}

template <class S, typename Kernel>
static hipError_t launch(Kernel kernel, GemmArgs p, const TilePlan& plan, hipStream_t stream) {
  p.grid_m = (p.M + S::BM - 1) / S::BM;
  p.grid_n = (p.N + S::CN - 1) / S::CN;
  p.splits = plan.splits, p.per = plan.per;
  const long long blocks = static_cast<long long>(p.grid_m) * p.grid_n * p.splits;
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS * S::GROUPS), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.splits == 1 ? e : launch_ffn_finish(1, S::EPI, p, stream);
}

// Measured at N=8192, K=4096, 256 x 256 (sixteen waves) / 128 x 128 (four) / 64 x 128 in four groups / 64 x 64 in four
// groups of two waves, us: M=2048 112 / 140 / 226 / 304; M=1024 99 / 67 / 114 / 153; M=256 96 / 48 / 29 / 38; M=64
// 88 / 44 / 24 / 17.
static const TileCost kWeightsWays[] = {{256, 256, 0, 1.7, 3.4, 1.7}, {128, 128, 0, 0.68, 1.02, 0.53}, {64, 128, 1, 0.4, 0.9, 0.45},
                                        {64, 64, 1, 0.22, 0.55, 0.28}};
static const TileCost kGatedWeightsWays[] = {{256, 128, 0, 1.7, 3.4, 1.7}, {128, 64, 0, 0.68, 1.02, 0.53}, {64, 64, 1, 0.4, 0.9, 0.45},
                                             {64, 32, 1, 0.22, 0.55, 0.28}};
// Measured at N=8192, K=4096, 256 x 256 (sixteen waves) / 128 x 128 (four) / the same in two groups / 64 x 64 in two
// groups, us: M=4096 86 / 99 / 122 / 163; M=512 32 / 19 / 17 / 22; M=128 28 / 16 / 14 / 8.6.
static const TileCost kBothWays[] = {{256, 256, 0, 2.5, 5.2, 2.6}, {128, 128, 0, 1.0, 1.7, 0.77}, {128, 128, 0.5, 0.87, 1.9, 0.95},
                                     {64, 64, 0.5, 0.35, 0.65, 0.31}};

static TilePlan plan(bool both, int epi, const GemmArgs& p, size_t room) {
  if (both) return plan_tiles(kBothWays, 4, 256, p, p.N, room);
  return epi == EPI_GATED ? plan_tiles(kGatedWeightsWays, 4, 64, p, 2 * p.N, room) : plan_tiles(kWeightsWays, 4, 64, p, p.N, room);
}

template <int EPI>
static hipError_t launch_weights(const GemmArgs& p, size_t room, hipStream_t stream) {
  const TilePlan chosen = plan(false, EPI, p, p.partial != nullptr ? room : 0);
  switch (chosen.way) {
    case 0: {
      typedef GemmShape<KIND_BF16, false, false, EPI, 4, 4, 4, 4> S;
      return launch<S>(mxfp4_weights_kernel<S>, p, chosen, stream);
    }
    case 1: {
      typedef GemmShape<KIND_BF16, false, false, EPI, 2, 2, 4, 4> S;
      return launch<S>(mxfp4_weights_kernel<S>, p, chosen, stream);
    }
    case 2: {
      typedef GemmShape<KIND_BF16, false, false, EPI, 2, 2, 2, 4, 4> S;
      return launch<S>(mxfp4_weights_kernel<S>, p, chosen, stream);
    }
    default: {
      typedef GemmShape<KIND_BF16, false, false, EPI, 2, 1, 2, 4, 4> S;
      return launch<S>(mxfp4_weights_kernel<S>, p, chosen, stream);
    }
  }
}

template <bool FOURS>
static hipError_t launch_both(const GemmArgs& p, size_t room, hipStream_t stream) {
  const TilePlan chosen = plan(true, EPI_STORE, p, p.partial != nullptr ? room : 0);
  switch (chosen.way) {
    case 0: {
      typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 4, 4, 4, 4> S;
      return launch<S>(mxfp4_both_kernel<S, FOURS>, p, chosen, stream);
    }
    case 1: {
      typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 2, 2, 4, 4> S;
      return launch<S>(mxfp4_both_kernel<S, FOURS>, p, chosen, stream);
    }
    case 2: {
      typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 2, 2, 4, 4, 2> S;
      return launch<S>(mxfp4_both_kernel<S, FOURS>, p, chosen, stream);
    }
    default: {
      typedef GemmShape<KIND_MXFP4, false, false, EPI_STORE, 2, 2, 2, 2, 2> S;
      return launch<S>(mxfp4_both_kernel<S, FOURS>, p, chosen, stream);
    }
  }
}

// Whether both kinds of scales can be read 4 bytes at a time
static bool scales_on_fours(const GemmArgs& p) {
  const auto fours = [](const void* a) { return (reinterpret_cast<unsigned long long>(a) & 3) == 0; };
  return p.K % 128 == 0 && fours(p.b_scales) && fours(p.a_scales);
}

hipError_t launch_mxfp4_gemm(bool x_mxfp4, int epi, const GemmArgs& p, size_t room, hipStream_t stream) {
  if (x_mxfp4 && epi != EPI_STORE) return hipErrorInvalidValue;
  if (mxfp4_skinny_takes(x_mxfp4, p)) return launch_mxfp4_skinny(x_mxfp4, epi == EPI_GATED, p, stream);
  if (x_mxfp4) return scales_on_fours(p) ? launch_both<true>(p, room, stream) : launch_both<false>(p, room, stream);
  return epi == EPI_GATED ? launch_weights<EPI_GATED>(p, room, stream) : launch_weights<EPI_STORE>(p, room, stream);
}

size_t mxfp4_gemm_bytes(bool x_mxfp4, int epi, const GemmArgs& p) {
  if (mxfp4_skinny_takes(x_mxfp4, p)) return 0;
  return partial_bytes(plan(x_mxfp4, epi, p, ~size_t{0}), p.M, epi == EPI_GATED ? 2 * p.N : p.N);
}

}  // namespace fmoe
