// The tiled matrix product of the dense feed-forward kernels, C[m, n] = sum_k A(m, k) B(n, k).
//
// A workgroup of WM x WN waves takes a tile of WM*FM*16 by WN*FN*16 results; a wave FM by FN blocks
// of 16 x 16. The matrix instructions get the rows of B as their first operand, so that a lane ends
// up with 4 FN neighbouring columns of one row of C and stores them 16 bytes at a time.
#pragma once
#include "ffn_device.h"

namespace fmoe {

// GROUPS such sets of waves share a tile's steps of k, each with LDS of its own, and add up their sums in the end.
template <int KIND_, bool OUTER_A_, bool OUTER_B_, int EPI_, int WM_, int WN_, int FM_, int FN_, int GROUPS_ = 1>
struct GemmShape {
  static constexpr int KIND = KIND_;
  static constexpr bool OUTER_A = OUTER_A_, OUTER_B = OUTER_B_;
  static constexpr int EPI = EPI_, WM = WM_, WN = WN_, FM = FM_, FN = FN_, GROUPS = GROUPS_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int BM = WM * FM * 16, BN = WN * FN * 16;     // rows of the two tiles
  static constexpr int CN = EPI == EPI_GATED ? BN / 2 : BN;      // columns of C a workgroup writes
  static constexpr int STEP = step_k(KIND);
  static constexpr int ESIZE = KIND == KIND_F32 ? 4 : 2;         // bytes a value (MXFP4: see bytes_of)
  static constexpr int STAGE_BYTES = (BM + BN) * 128;
  static constexpr int LDS_BYTES = 2 * GROUPS * STAGE_BYTES;
};

template <int KIND>
__device__ __forceinline__ long long bytes_of(long long values) {
  return KIND == KIND_MXFP4 ? values / 2 : KIND == KIND_F32 ? values * 4 : values * 2;
}

// One operand's loads: which bytes of memory this lane asks for in each of its pieces of a stage.
// GATED: the tile's rows are gate rows of `matrix rows / 2` and the up rows of the same columns.
template <int KIND, bool OUTER, int ROWS, int THREADS, int F, bool GATED>
struct TileLoader {
  static constexpr int PIECES = ROWS * 8 / THREADS;
  static constexpr int PK = piece_k(KIND);
  static constexpr int LINE = OUTER ? ROWS / PK : 8;  // pieces of a k, or of a row
  static_assert(PIECES * THREADS == ROWS * 8, "whole pieces a thread");
  static_assert(!GATED || !OUTER, "gated weights have their k inside the rows");
  unsigned offset[PIECES];
  const char* base;
  long long step_bytes, up_bytes;
  int tid;  // of the THREADS that load

  // k of this lane's piece i inside a stage (the first of its values)
  __device__ __forceinline__ int k_of(int i) const {
    const int at = i * THREADS + tid;
    return OUTER ? at / LINE : ((at & 7) ^ ((at >> 3) & 7)) * PK;
  }

  // row0: the tile's first row (gated: its first column of C) of `rows`
  __device__ __forceinline__ void init(const void* p, long long ld, int row0, int rows, int tid_) {
    tid = tid_;
    up_bytes = GATED ? bytes_of<KIND>(rows * ld) : 0;
    if constexpr (!OUTER) {
      base = static_cast<const char*>(p) + bytes_of<KIND>(row0 * ld);
      step_bytes = 128;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int row = (i * THREADS + tid) >> 3, piece = (tid & 7) ^ (row & 7);
        const int in_wave = row % (16 * F), f = in_wave >> 4, r = in_wave & 15;
        const int src = GATED ? row / (16 * F) * (8 * F) + gated_row<F>(f, r) : row / (16 * F) * (16 * F) + dealt_row<F>(f, r);
        offset[i] = row0 + src < rows ? static_cast<unsigned>(bytes_of<KIND>(src * ld)) + piece * 16 : kOutside;
      }
    } else {
      base = static_cast<const char*>(p) + bytes_of<KIND>(row0);
      step_bytes = bytes_of<KIND>(ld * step_k(KIND));
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int at = i * THREADS + tid, k = at / LINE;
        int piece = at % LINE;
        if constexpr (KIND == KIND_BF16) piece ^= k_row_swap<F>(k) & (LINE - 1);
        else piece ^= f32_k_row_swap<F>(k) & (LINE - 1);
        offset[i] = row0 + piece * PK < rows ? static_cast<unsigned>(bytes_of<KIND>(k * ld)) + piece * 16 : kOutside;
      }
    }
  }

  // Stage s into `lds`; left: how many k there are from its first one on
  __device__ __forceinline__ void load(char* lds, int s, int left) const {
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const char* from = base + s * step_bytes;
    char* to = lds + wave * 1024;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int f = ((i * THREADS + wave * 64) >> 3) % (16 * F) / 16;  // gated: the same for all of a wave's lanes
      const __amdgpu_buffer_rsrc_t r = make_rsrc(from + (GATED && f >= F / 2 ? up_bytes : 0), 0x7FFFFFFFu);
      const bool in = left >= step_k(KIND) || k_of(i) < left;
      load_to_lds16(r, to + i * THREADS * 16, in ? offset[i] : kOutside);
    }
  }
};

__device__ __forceinline__ unsigned lds_address(const char* p) {
  return static_cast<unsigned>(reinterpret_cast<unsigned long long>((const FFN_LDS char*)p));
}
// Four rows of k from at[f] on and the four at at[f] + FOUR, transposed. In assembly with their wait: around the builtin of these
// reads the compiler waits for every load to LDS that is on its way, the next stage's, which were to arrive
// during this one. (Training step T=4096, H=2048, I=6144: 989 us with the builtin, 911 so; the three gradients 523 and 465.)
template <int FOUR>
__device__ __forceinline__ void read_transposed(const unsigned (&at)[2], u32x2 (&lo)[2], u32x2 (&hi)[2]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %5\n\t"
      "ds_read_b64_tr_b16 %3, %5 offset:%6\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
      : "v"(at[0]), "v"(at[1]), "n"(FOUR)
      : "memory");
}
template <int FOUR>
__device__ __forceinline__ void read_transposed(const unsigned (&at)[4], u32x2 (&lo)[4], u32x2 (&hi)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %2, %9\n\t"
      "ds_read_b64_tr_b16 %3, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %10\n\t"
      "ds_read_b64_tr_b16 %5, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %11\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]), "=&v"(hi[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(FOUR)
      : "memory");
}

// A wave's F blocks of an operand for one of the stage's two halves (bfloat16 32 k, MXFP4 128).
// Lane l holds row l % 16 of each block and the (l / 16)-th quarter of the k, 16 bytes.
template <int KIND, bool OUTER, int ROWS, int F>
struct Fragments {
  static constexpr int LINE_BYTES = ROWS * 2;  // of a k, where a row is one k
  i32x4 v[F];

  __device__ __forceinline__ void read(const char* tile, int wave_row, int half) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    if constexpr (!OUTER) {
      const char* at = tile + (wave_row + r) * 128 + (((half * 4 + g) ^ (r & 7)) << 4);
#pragma unroll
      for (int f = 0; f < F; ++f) v[f] = *(const FFN_LDS i32x4*)(at + f * 2048);
    } else {
      static_assert(KIND == KIND_BF16, "read transposed");
      const int k = half * 32 + g * 8 + (r >> 2), swap = k_row_swap<F>(g * 8 + (r >> 2)) & (ROWS / 8 - 1);
      const unsigned line = lds_address(tile + k * LINE_BYTES);
      unsigned at[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const int col = wave_row + dealt_row<F>(f, (r & 3) * 4);
        at[f] = line + (((col >> 3) ^ swap) << 4) + (r & 1) * 8;
      }
      u32x2 lo[F], hi[F];
      read_transposed<4 * LINE_BYTES>(at, lo, hi);
#pragma unroll
      for (int f = 0; f < F; ++f)
        v[f] = i32x4{static_cast<int>(lo[f][0]), static_cast<int>(lo[f][1]), static_cast<int>(hi[f][0]), static_cast<int>(hi[f][1])};
    }
  }
};

// Workgroup `id`'s share of the tile's k: steps first .. first + count - 1. Splits of a tile lie a whole round of tiles
// apart, so id becomes the tile's number.
__device__ __forceinline__ void share_of(const GemmArgs& p, int steps, int& id, int& split, int& first, int& count) {
  split = first = 0, count = steps;
  if (p.splits > 1) {
    const int tiles = p.grid_m * p.grid_n;
    split = id / tiles, id -= split * tiles;
    first = split * p.per;
    count = steps - first < p.per ? steps - first : p.per;
  }
}

// The workgroup's tile. Neighbouring workgroup numbers lie on different XCDs, each with an L2 of its
// own, so an XCD gets a run of the order; the order walks GROUP tile rows column by column, so
// that the tiles in flight on an XCD share rows of both operands.
__device__ __forceinline__ void tile_of(const GemmArgs& p, int id, int& tile_m, int& tile_n) {
  constexpr int XCDS = 8, GROUP = 8;
  const int count = p.grid_m * p.grid_n;
  const int xcd = id % XCDS, each = count / XCDS, extra = count % XCDS;
  const int at = xcd * each + (xcd < extra ? xcd : extra) + id / XCDS;
  const int first = at / (GROUP * p.grid_n) * GROUP;
  const int rows = p.grid_m - first < GROUP ? p.grid_m - first : GROUP;
  const int inside = at - first * p.grid_n;
  tile_m = first + inside % rows;
  tile_n = inside / rows;
}

template <class S>
struct Accumulators {
  f32x4 v[S::FM][S::FN];
};

struct __attribute__((packed, aligned(2))) Anywhere16 {
  u32x4 v;
};
__device__ __forceinline__ void store8(unsigned short* to, const f32x4& a, const f32x4& b) {
  reinterpret_cast<Anywhere16*>(to)->v = u32x4{pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(b[0], b[1]), pack_bf16(b[2], b[3])};
}
__device__ __forceinline__ void store4(unsigned short* to, const f32x4& a) {
  *reinterpret_cast<u32x2*>(to) = u32x2{pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3])};
}
// the first `count` of eight
__device__ __forceinline__ void store_some(unsigned short* to, int count, const f32x4& a, const f32x4& b) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < count) to[j] = static_cast<unsigned short>(pack_bf16(j < 4 ? a[j & 3] : b[j & 3], 0.0f) & 0xFFFF);
}

// The groups' sums of a tile, into the first group's, in the groups' order. Of the others nobody is left to write results.
// FRUGAL: a row of blocks at a time, for callers with few registers left.
template <class S, int ROOM = S::LDS_BYTES, bool FRUGAL = false>
__device__ __forceinline__ void add_groups(char* lds, int group, Accumulators<S>& acc) {
  if constexpr (S::GROUPS > 1) {
    f32x4* part = reinterpret_cast<f32x4*>(lds);
    const int tid = threadIdx.x % S::THREADS;
    static_assert((S::GROUPS - 1) * S::BM * S::BN * 4 <= ROOM, "room for the others' sums");
    __syncthreads();
    if (group > 0) {
#pragma unroll
      for (int fm = 0; fm < S::FM; ++fm)
#pragma unroll
        for (int fn = 0; fn < S::FN; ++fn) part[(((group - 1) * S::FM + fm) * S::FN + fn) * S::THREADS + tid] = acc.v[fm][fn];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int other = 1; other < S::GROUPS; ++other)
#pragma unroll
        for (int fm = 0; fm < S::FM; ++fm) {
#pragma unroll
          for (int fn = 0; fn < S::FN; ++fn) acc.v[fm][fn] += part[(((other - 1) * S::FM + fm) * S::FN + fn) * S::THREADS + tid];
          if constexpr (FRUGAL) asm volatile("" : : : "memory");
        }
    }
  }
}

// Two blocks' results of a lane, four neighbours each, against those of the lane 16 on or back: afterwards the
// lane has eight neighbours, of the first block if l / 16 is even and else of the second.
__device__ __forceinline__ void trade(f32x4& a, f32x4& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[i]), __float_as_uint(b[i]), false, false);
    a[i] = __uint_as_float(v[0]);
    b[i] = __uint_as_float(v[1]);
  }
}

// A lane's results v[COUNT] of one row of C: block f's are columns col + 8 f + 0..3 (col: with the lane's own 4 * (g % 2)).
// ANY_WIDTH: bfloat16 rows whose width is no multiple of 8 begin anywhere: the same wide writes, which memory takes at any
// address, but value by value across a row's end.
// Every lane of a wave takes part, `in` says whether its row exists.
template <int KIND, int COUNT, bool ANY_WIDTH = false>
__device__ __forceinline__ void store_row(void* row, int col, int columns, bool in, f32x4 (&v)[COUNT]) {
  if constexpr (KIND == KIND_F32) {
#pragma unroll
    for (int f = 0; f < COUNT; ++f)
      if (in && col + 8 * f < columns) *reinterpret_cast<f32x4*>(static_cast<float*>(row) + col + 8 * f) = v[f];
  } else {
    unsigned short* to = static_cast<unsigned short*>(row) + col;
    if constexpr (COUNT == 1) {
      static_assert(!ANY_WIDTH, "pairs of blocks");
      if (in && col < columns) store4(to, v[0]);
    } else {
      static_assert(COUNT % 2 == 0, "pairs of blocks");
      const int odd = (threadIdx.x >> 4) & 1;
#pragma unroll
      for (int f = 0; f < COUNT; f += 2) {
        trade(v[f], v[f + 1]);
        const int at = 8 * f + odd * 4;  // the second block's eight begin 4 before this lane's own column of it
        if (in && col + at + (ANY_WIDTH ? 8 : 1) <= columns) store8(to + at, v[f], v[f + 1]);
        else if (ANY_WIDTH && in && col + at < columns) store_some(to + at, columns - col - at, v[f], v[f + 1]);
      }
    }
  }
}

// A split's sums as they are: of a gated product gate columns and, behind the N of them, up columns
template <class S>
__device__ __forceinline__ void write_partial(const GemmArgs& p, int split, int m0, int n0, Accumulators<S>& acc) {
  constexpr int FN = S::FN, FM = S::FM;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int wm = wave / S::WN, wn = wave % S::WN;
  const long long ld = partial_ld(S::EPI == EPI_GATED ? 2 * p.N : p.N);
  float* part = p.partial + split * (p.M * ld);
#pragma unroll
  for (int fm = 0; fm < FM; ++fm) {
    const int m = m0 + wm * FM * 16 + dealt_row<FM>(fm, r);
    if (m >= p.M) continue;
#pragma unroll
    for (int fn = 0; fn < FN; ++fn) {
      if constexpr (S::EPI == EPI_GATED) {
        const int col = n0 + wn * FN * 8 + gated_row<FN>(fn, 4 * g);
        if (col < p.N) *reinterpret_cast<f32x4*>(part + m * ld + (fn >= FN / 2 ? p.N : 0) + col) = acc.v[fm][fn];
      } else {
        const int col = n0 + wn * FN * 16 + dealt_row<FN>(fn, 4 * g);
        if (col < p.N) *reinterpret_cast<f32x4*>(part + m * ld + col) = acc.v[fm][fn];
      }
    }
  }
}

// What becomes of the sums. Of a gated product the first half of the blocks are gate columns and the others
// the same up columns.
// The slope kernel at M=4096, N=6144, K=2048 bfloat16 (174 us): 107 without what follows its sums, 131 without
// reading the projections, 151 without writing: 200 MB and 100 MB at memory's rate. Asking for all of a row's
// projections together, a row ahead, made no difference.
template <class S, bool ANY_WIDTH = false>
__device__ __forceinline__ void write_results(const GemmArgs& p, int m0, int n0, Accumulators<S>& acc) {
  constexpr int FN = S::FN, FM = S::FM;
  constexpr bool EXACT = S::KIND == KIND_F32;
  constexpr int OUT = EXACT ? KIND_F32 : KIND_BF16, OSIZE = EXACT ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
  for (int fm = 0; fm < FM; ++fm) {
    const int m = m0 + wm * FM * 16 + dealt_row<FM>(fm, r);
    const bool in = m < p.M;
    if constexpr (S::EPI == EPI_STORE) {
      store_row<OUT, FN, ANY_WIDTH>(static_cast<char*>(p.c) + m * p.ldc * OSIZE, n0 + wn * FN * 16 + dealt_row<FN>(0, 4 * g), p.N, in, acc.v[fm]);
    } else if constexpr (S::EPI == EPI_GATED) {
      const int col = n0 + wn * FN * 8 + gated_row<FN>(0, 4 * g);
      f32x4 h[FN / 2], gate[FN / 2], up[FN / 2];
#pragma unroll
      for (int f = 0; f < FN / 2; ++f) {
        gate[f] = acc.v[fm][f];
        up[f] = acc.v[fm][FN / 2 + f];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[f][i] = act_of<EXACT>(p.act, gate[f][i]) * up[f][i];
      }
      store_row<OUT, FN / 2>(static_cast<char*>(p.c) + m * p.ldc * OSIZE, col, p.N, in, h);
      if (p.gu != nullptr) {
        float* row = p.gu + m * (2LL * p.N);
        store_row<KIND_F32, FN / 2>(row, col, p.N, in, gate);
        store_row<KIND_F32, FN / 2>(row + p.N, col, p.N, in, up);
      }
    } else {
      const int col = n0 + wn * FN * 16 + dealt_row<FN>(0, 4 * g);
      const float* row = p.gu + m * (2LL * p.N);
      f32x4 dg[FN], du[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        dg[f] = du[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!in || col + 8 * f >= p.N) continue;
        const f32x4 gate = *reinterpret_cast<const f32x4*>(row + col + 8 * f);
        const f32x4 up = *reinterpret_cast<const f32x4*>(row + p.N + col + 8 * f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float dh = acc.v[fm][f][i];
          float a, slope;
          act_and_slope<EXACT>(p.act, gate[i], a, slope);
          dg[f][i] = dh * up[i] * slope;
          du[f][i] = dh * a;
        }
      }
      char* out = static_cast<char*>(p.c) + m * p.ldc * OSIZE;
      store_row<OUT, FN>(out, col, p.N, in, dg);
      store_row<OUT, FN>(out + static_cast<long long>(p.N) * OSIZE, col, p.N, in, du);
    }
  }
}

}  // namespace fmoe
