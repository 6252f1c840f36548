// The dense block's matrix products in float32, on the bfloat16 matrix instructions.
//
// A float32 is split into three bfloat16 parts, each the rest rounded to nearest: x = hi + mid + lo exactly (8 bits
// and a sign each). Of the nine products of parts the six largest are summed in float32; the three left out are
// below 2^-24 of a product, of either sign, about what a rounded multiplication may be off by (with parts cut off instead
// it is 2^-21, always towards zero, and 3 % faster). Six instructions at 16 times the rate of the float32 ones: 2.7 times as
// fast.
// The parts live in registers only; a tile in LDS is float32, and a wave splits what it reads.
//
// Parts below bfloat16's smallest number, 2^-133, are lost (the instruction keeps what is below 2^-126): an operand is its
// parts to 2^-134. With operands below kLarge a sum of K products is off by less than K 2^-133 kLarge from that, which is below
// 2^-24 of a sum of small_sum(K) and more. So a sum is taken again, on the float32 matrix instructions, if it is smaller than
// that and not zero, if its row or column holds a larger operand, or if it is no finite number (an infinity has no parts): a
// workgroup with such a sum goes over its k once more, other sums stay as they are. Larger operands are noticed by the sums of
// the squares of all rows' high parts, one more instruction a block: 4 to 5 % of a call (T=1001, H=2048, I=768, step 222 ->
// 232 us, with parts cut off and none of this 217, all in one run; the largest magnitude by vector instructions costs more).
// That second pass takes 2 to 3 times a tile's time: a step of this size 0.47 ms with a NaN among its tokens. (A sum that
// comes out as zero is left: ordinary ones do now and then. Of operands below 2^-134 alone, times others below kLarge, it may
// be off by K 2^-101.)
#include "ffn_gemm_device.h"

namespace fmoe {

// Eight values a lane: the (l / 16)-th quarter of a stage's 32 k, of rows l % 16
template <bool OUTER, int ROWS, int F>
__device__ __forceinline__ void read_f32(float (&v)[8], const char* tile, int wave_row, int f) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  if constexpr (!OUTER) {
    const char* row = tile + (wave_row + f * 16 + r) * 128;
    const f32x4 lo = *(const FFN_LDS f32x4*)(row + (((2 * g) ^ (r & 7)) << 4));
    const f32x4 hi = *(const FFN_LDS f32x4*)(row + (((2 * g + 1) ^ (r & 7)) << 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
  } else {
    const int col = wave_row + dealt_row<F>(f, r);
    const char* at = tile + g * 8 * ROWS * 4 + (((col >> 2) ^ f32_k_row_swap<F>(g * 8)) << 4) + (col & 3) * 4;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *(const FFN_LDS float*)(at + i * ROWS * 4);
  }
}

struct Parts {
  i32x4 hi, mid, lo;  // eight bfloat16 each
};
// The two values of a word of bfloat16. (Written as a shift and a mask the compiler converts each value once more: two
// instructions of eleven a pair; T=1001, H=2048, I=768, forward 90 us instead of 82.)
__device__ __forceinline__ float low_of(unsigned word) { return __uint_as_float(__builtin_amdgcn_perm(word, word, 0x01000C0Cu)); }
__device__ __forceinline__ float high_of(unsigned word) { return __uint_as_float(__builtin_amdgcn_perm(word, word, 0x03020C0Cu)); }
__device__ __forceinline__ Parts split(const float (&v)[8]) {
  Parts p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i], b = v[2 * i + 1];
    const unsigned hi = pack_bf16(a, b);
    const float ar = a - low_of(hi), br = b - high_of(hi);
    const unsigned mid = pack_bf16(ar, br);
    p.hi[i] = static_cast<int>(hi);
    p.mid[i] = static_cast<int>(mid);
    p.lo[i] = static_cast<int>(pack_bf16(ar - low_of(mid), br - high_of(mid)));
  }
  return p;
}

constexpr float kLarge = 4294967296.0f;  // 2^32
__device__ __forceinline__ float small_sum(int K) { return static_cast<float>(K) * 6.6174449004242214e-24f; }  // K 2^-77

// A workgroup's sums over its share of the k, in its GROUPS groups. PLAIN: with the float32 instructions, and the largest
// magnitudes that this lane read of each block's rows; else with the products of parts, and `squares`: of the rows' high
// parts, summed (some of its elements are, and none is larger).
template <class S, bool PLAIN, class LoaderA, class LoaderB>
__device__ __forceinline__ void sum_tile_f32(const GemmArgs& p, const LoaderA& load_a, const LoaderB& load_b, char* mine, int group, int first,
                                             int steps, Accumulators<S>& acc, f32x4& squares, float (&most_a)[S::FM], float (&most_b)[S::FN]) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x % S::THREADS >> 6), wm = wave / S::WN, wn = wave % S::WN;
  squares = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int fm = 0; fm < S::FM; ++fm) {
    most_a[fm] = 0.0f;
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, most_b[fn] = 0.0f;
  }
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
    if constexpr (PLAIN) {
      float b[S::FN][8];
#pragma unroll
      for (int fn = 0; fn < S::FN; ++fn) {
        read_f32<S::OUTER_B, S::BN, S::FN>(b[fn], now + S::BM * 128, wn * S::FN * 16, fn);
#pragma unroll
        for (int i = 0; i < 8; ++i) most_b[fn] = fmaxf(most_b[fn], fabsf(b[fn][i]));
      }
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm) {
        float a[8];
        read_f32<S::OUTER_A, S::BM, S::FM>(a, now, wm * S::FM * 16, fm);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          most_a[fm] = fmaxf(most_a[fm], fabsf(a[i]));
#pragma unroll
          for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[fn][i], a[i], acc.v[fm][fn], 0, 0, 0);
        }
      }
    } else {
      Parts b[S::FN];
      auto square = [&](const i32x4& hi) {
        squares = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, hi), __builtin_bit_cast(bf16x8, hi), squares, 0, 0, 0);
      };
#pragma unroll
      for (int fn = 0; fn < S::FN; ++fn) {
        float v[8];
        read_f32<S::OUTER_B, S::BN, S::FN>(v, now + S::BM * 128, wn * S::FN * 16, fn);
        b[fn] = split(v);
        square(b[fn].hi);
      }
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm) {
        float v[8];
        read_f32<S::OUTER_A, S::BM, S::FM>(v, now, wm * S::FM * 16, fm);
        const Parts a = split(v);
        square(a.hi);
        // the small products first
        auto add = [&](const i32x4 Parts::*pb, const i32x4 Parts::*pa) {
#pragma unroll
          for (int fn = 0; fn < S::FN; ++fn)
            acc.v[fm][fn] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b[fn].*pb),
                                                                    __builtin_bit_cast(bf16x8, a.*pa), acc.v[fm][fn], 0, 0, 0);
        };
        add(&Parts::lo, &Parts::hi);
        add(&Parts::mid, &Parts::mid);
        add(&Parts::hi, &Parts::lo);
        add(&Parts::mid, &Parts::hi);
        add(&Parts::hi, &Parts::mid);
        add(&Parts::hi, &Parts::hi);
      }
    }
  }
}

// A sum's place in the order infinity, NaN, zero, small to large
__device__ __forceinline__ unsigned sum_order(float v) { return (__float_as_uint(v) << 1) + 0x01000000u; }
__device__ __forceinline__ bool doubtful(float v, float small) { return sum_order(v) < sum_order(small) && v != 0.0f; }

// Tile `id` of a product, by a workgroup with S::LDS_BYTES of LDS
template <class S>
__device__ __forceinline__ void gemm_tile_f32(const GemmArgs& p, char* lds, int id) {
  int share, first, steps, tile_m, tile_n;
  share_of(p, (p.K + S::STEP - 1) / S::STEP, id, share, first, steps);
  tile_of(p, id, tile_m, tile_n);
  const int m0 = tile_m * S::BM, n0 = tile_n * S::CN;
  const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / S::THREADS), tid = threadIdx.x % S::THREADS;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / S::WN, wn = wave % S::WN;
  char* mine = lds + group * 2 * S::STAGE_BYTES;

  TileLoader<KIND_F32, S::OUTER_A, S::BM, S::THREADS, S::FM, false> load_a;
  TileLoader<KIND_F32, S::OUTER_B, S::BN, S::THREADS, S::FN, S::EPI == EPI_GATED> load_b;
  load_a.init(p.a, p.lda, m0, p.M, tid);
  load_b.init(p.b, p.ldb, n0, p.N, tid);

  Accumulators<S> acc;
  f32x4 squares;
  float most_a[S::FM], most_b[S::FN];
  sum_tile_f32<S, false>(p, load_a, load_b, mine, group, first, steps, acc, squares, most_a, most_b);
  add_groups<S>(lds, group, acc);

  const float small = small_sum(p.K);
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) odd |= !(fabsf(squares[i]) < kLarge * kLarge);
  if (group == 0) {  // (the others' sums are in this one's)
    unsigned least = 0xFFFFFFFFu;
#pragma unroll
    for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < S::FN; ++fn)
#pragma unroll
        for (int i = 0; i < 4; ++i) least = min(least, sum_order(acc.v[fm][fn][i]));
    if (__any(least < sum_order(small))) {
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn)
#pragma unroll
          for (int i = 0; i < 4; ++i) odd |= doubtful(acc.v[fm][fn][i], small);
    }
  }
  // (words in the stages' memory: beside LDS of another name the compiler waits, in the loop over k, for the next stage's
  // loads before it reads this one's, 5 to 15 % of a call)
  unsigned* words = reinterpret_cast<unsigned*>(lds);
  const bool any = __any(odd);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) words[threadIdx.x >> 6] = any;
  __syncthreads();
  unsigned again = 0;
#pragma unroll
  for (int w = 0; w < S::WAVES * S::GROUPS; ++w) again |= words[w];
  if (__builtin_amdgcn_readfirstlane(again) != 0) {
    __syncthreads();
    Accumulators<S> plain;
    sum_tile_f32<S, true>(p, load_a, load_b, mine, group, first, steps, plain, squares, most_a, most_b);
    // the rows' largest values, of all groups
    const int lane = threadIdx.x & 63, r = lane & 15;
    unsigned* most = words + wm * S::FM * 16;
    unsigned* most_of_b = words + S::BM + wn * S::FN * 16;
    __syncthreads();
    for (int i = threadIdx.x; i < S::BM + S::BN; i += S::THREADS * S::GROUPS) words[i] = 0;
    __syncthreads();
#pragma unroll
    for (int fm = 0; fm < S::FM; ++fm) atomicMax(&most[fm * 16 + r], __float_as_uint(most_a[fm]));
#pragma unroll
    for (int fn = 0; fn < S::FN; ++fn) atomicMax(&most_of_b[fn * 16 + r], __float_as_uint(most_b[fn]));
    __syncthreads();
#pragma unroll
    for (int fm = 0; fm < S::FM; ++fm) {
      const float row = __uint_as_float(most[fm * 16 + r]);
#pragma unroll
      for (int fn = 0; fn < S::FN; ++fn)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float column = __uint_as_float(most_of_b[fn * 16 + (lane >> 4) * 4 + i]);
          if (fmaxf(row, column) >= kLarge) acc.v[fm][fn][i] = __builtin_nanf("");
        }
    }
    add_groups<S, S::LDS_BYTES, true>(lds, group, plain);
#pragma unroll
    for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
      for (int fn = 0; fn < S::FN; ++fn)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (doubtful(acc.v[fm][fn][i], small)) acc.v[fm][fn][i] = plain.v[fm][fn][i];
  }
  if (group != 0) return;
  if (p.splits > 1) write_partial<S>(p, share, m0, n0, acc);
  else write_results<S>(p, m0, n0, acc);
}

template <class S>
__global__ __launch_bounds__(S::THREADS * S::GROUPS, 2) void ffn_gemm_f32_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(128))) char lds[S::LDS_BYTES];
  gemm_tile_f32<S>(p, lds, blockIdx.x);
}

// As ffn_grads_kernel
template <int WM, int WN, int FM, int FN>
__global__ __launch_bounds__(WM * WN * 64, 2) void ffn_grads_f32_kernel(FfnGrads p) {
  typedef GemmShape<KIND_F32, false, true, EPI_STORE, WM, WN, FM, FN> X;
  typedef GemmShape<KIND_F32, true, true, EPI_STORE, WM, WN, FM, FN> W;
  __shared__ __attribute__((aligned(128))) char lds[X::LDS_BYTES];
  const int id = blockIdx.x;
  if (id < p.begin[1]) {
    if (id < p.dx.grid_m * p.dx.grid_n * p.dx.splits) gemm_tile_f32<X>(p.dx, lds, id);
  } else {
    const bool second = id >= p.begin[2];
    const GemmArgs& dw = second ? p.dw2 : p.dw13;
    const int at = id - p.begin[second ? 2 : 1];
    if (at < dw.grid_m * dw.grid_n * dw.splits) gemm_tile_f32<W>(dw, lds, at);
  }
}

template <class S>
static hipError_t launch_f32(GemmArgs p, const TilePlan& plan, hipStream_t stream) {
  p.grid_m = (p.M + S::BM - 1) / S::BM;
  p.grid_n = (p.N + S::CN - 1) / S::CN;
  p.splits = plan.splits, p.per = plan.per;
  const long long blocks = static_cast<long long>(p.grid_m) * p.grid_n * p.splits;
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  hipLaunchKernelGGL(ffn_gemm_f32_kernel<S>, dim3(static_cast<unsigned>(blocks)), dim3(S::THREADS * S::GROUPS), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.splits == 1 ? e : launch_ffn_finish(0, S::EPI, p, stream);
}

// Large tiles split each value for more products, small ones fill more CUs, and groups of waves that share a tile's k fill
// their waits. Measured on M=1001, N=768 gated, K=2048, 128 x 128 / 128 x 64 / 64 x 64 rows of A and B, us:
// 113 / 75 / 75 in one group, 91 / 62 / 67 in two, 64 x 64 in four 72; M=1001, N=768, K=2048 with B's rows as k
// 122 / 79 / 55, 101 / 64 / 42, 37; M=N=K=4096 683 / 819 / 969 in one.
// The costs below are those of parts that were cut off, before large operands were looked for, 5 to 20 % less; by the present ones
// 60 random calls take 0.3 % more, and their steps 0.5 %.
static const TileCost kF32Ways[] = {{128, 128, 0, 1.7, 2.5, 1.25}, {128, 128, 1, 1.32, 2.7, 1.35}, {128, 64, 0, 1.1, 1.6, 0.72},
                                    {64, 64, 0, 0.78, 0.98, 0.42}, {64, 64, 0.8, 0.54, 0.85, 0.45}, {64, 64, 1.8, 0.48, 0.95, 0.48}};
static const TileCost kF32GatedWays[] = {{128, 64, 0, 1.7, 2.5, 1.25}, {128, 64, 1, 1.32, 2.7, 1.35}, {128, 32, 0, 1.1, 1.6, 0.72},
                                         {64, 32, 0, 0.78, 0.98, 0.42}, {64, 32, 0.8, 0.54, 0.85, 0.45}, {64, 32, 1.8, 0.48, 0.95, 0.48}};

static TilePlan plan_f32(int epi, const GemmArgs& p, size_t room) {
  return plan_tiles(epi == EPI_GATED ? kF32GatedWays : kF32Ways, 6, 32, p, epi == EPI_GATED ? 2 * p.N : p.N, room);
}

template <bool OB, int EPI>
static hipError_t pick_f32(const GemmArgs& p, size_t room, hipStream_t stream) {
  const TilePlan chosen = plan_f32(EPI, p, p.partial != nullptr ? room : 0);
  switch (chosen.way) {
    case 0: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 4, 4>>(p, chosen, stream);
    case 1: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 4, 4, 2>>(p, chosen, stream);
    case 2: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 4, 2>>(p, chosen, stream);
    case 3: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 2, 2>>(p, chosen, stream);
    case 4: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 2, 2, 2>>(p, chosen, stream);
    default: return launch_f32<GemmShape<KIND_F32, false, OB, EPI, 2, 2, 2, 2, 4>>(p, chosen, stream);
  }
}

hipError_t launch_ffn_gemm_f32(bool k_outer_b, int epi, const GemmArgs& p, size_t room, hipStream_t stream) {
  if (epi == EPI_SLOPE) return pick_f32<true, EPI_SLOPE>(p, room, stream);
  return epi == EPI_GATED ? pick_f32<false, EPI_GATED>(p, room, stream) : pick_f32<false, EPI_STORE>(p, room, stream);
}

size_t ffn_gemm_f32_bytes(int epi, const GemmArgs& p) {
  return partial_bytes(plan_f32(epi, p, ~size_t{0}), p.M, epi == EPI_GATED ? 2 * p.N : p.N);
}

static const TileCost kF32GradsWays[] = {{128, 128, 0, 1.7, 2.5, 1.25, 2}, {128, 64, 0, 1.1, 1.6, 0.72, 3}, {64, 64, 0, 0.78, 0.98, 0.45, 4}};

hipError_t launch_ffn_grads_f32(FfnGrads p, float* partial, size_t room, hipStream_t stream) {
  const GradsPlan chosen = plan_grads(kF32GradsWays, 3, 32, p, partial != nullptr ? room : 0);
  const long long blocks = lay_out_grads(chosen, kF32GradsWays[chosen.way], p, partial);
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (chosen.way == 0) hipLaunchKernelGGL((ffn_grads_f32_kernel<2, 2, 4, 4>), grid, dim3(256), 0, stream, p);
  else if (chosen.way == 1) hipLaunchKernelGGL((ffn_grads_f32_kernel<2, 2, 4, 2>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((ffn_grads_f32_kernel<2, 2, 2, 2>), grid, dim3(256), 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess ? e : launch_ffn_finish_grads(0, p, stream);
}

size_t ffn_grads_f32_bytes(const FfnGrads& p) { return plan_bytes(plan_grads(kF32GradsWays, 3, 32, p, ~size_t{0}), p); }

}  // namespace fmoe
