// The router's choice as an operator of its own: from logits [T, E] the k experts of every token and their weights, how
// many tokens each expert got, the loss that balances them and the one that keeps logits small; and the gradient of the logits.
//
//   p = softmax of a token's candidates (logits above their type's lowest value; padding has none)
//   w_j = p of the j-th largest logit (the lowest index of equals), over the sum of the k if they are renormalised
//   balance = E sum_e (counts_e / slots) (sum_t p_te / n),  z = sum_t lse_t^2 / n,  n rows with a candidate, slots winners
//   dlogit = D + p (g - sum p g) + (2 dz / n) lse p,  g_e = dbalance E counts_e / (slots n),
//   D = w_j (dw_j - sum w dw) at the winners, or with plain probabilities dw_j joins g there
//
// Sixteen lanes have a token, four logits of every 64 each, so that a load is whole lines of four tokens and every cross-lane step is a data
// parallel primitive that serves four tokens. The winners are taken in k rounds, of the lanes' greatest. For those a logit and its place are
// one whole number, no two of them equal, so that a comparison says who goes first and a winner is found by its key.
// A float32 logit has nine bits too many for that; where two neighbours among the first k + 1 agree in what is kept, the
// wave takes its four tokens again by whole logits (of normally distributed ones with an offset an expert 1 token in 300 at E=128
// and 256, k=8, 1 wave's pass in 70; at E=256, k=32 1 token in 35, 1 pass in 9).
// The backward pass is bound by reading and writing the logits from some 65536 tokens on (131072 x 256 in float32 51 us, 5.3 TB/s). The
// forward pass is bound by neither memory nor the vector units: there it takes 52 us where the reading takes 25 and the instructions 31,
// since the k + 1 rounds depend on one another and four waves a SIMD are all there is to cover them; more winners cost accordingly
// (whole calls with k=8 and 32 58 and 169 us, in bfloat16 46 and 99).
#include <float.h>

#include "ffn_device.h"
#include "lane_device.h"
#include "layer_params.h"

namespace fmoe {
namespace {

// A row's logits as they are in memory: value i of a lane is column 64 (i / 4) + 4 lane + i % 4.
template <bool BF, int V>
struct Raw {
  unsigned u[BF ? V / 2 : V];
};
__device__ __forceinline__ int column(int lane, int i) { return (i >> 2) * 64 + lane * 4 + (i & 3); }

// WHOLE: E is a multiple of four and rows begin on four values. Columns outside are -inf.
template <bool BF, int V, bool WHOLE>
__device__ __forceinline__ Raw<BF, V> load_row(const void* logits, size_t at, int lane, int E) {
  Raw<BF, V> r;
#pragma unroll
  for (int c = 0; c < V / 4; ++c) {
    const int col = c * 64 + lane * 4;
    if constexpr (BF) {
      const unsigned short* p = reinterpret_cast<const unsigned short*>(logits) + at + col;
      u32x2 q = {0xFF80FF80u, 0xFF80FF80u};
      if constexpr (WHOLE) {
        if (col < E) q = *reinterpret_cast<const u32x2*>(p);
      } else {
        unsigned v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = col + i < E ? p[i] : 0xFF80u;
        q = {v[0] | v[1] << 16, v[2] | v[3] << 16};
      }
      r.u[2 * c] = q.x, r.u[2 * c + 1] = q.y;
    } else {
      const unsigned* p = reinterpret_cast<const unsigned*>(logits) + at + col;
      u32x4 q = {0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u};
      if constexpr (WHOLE) {
        if (col < E) q = *reinterpret_cast<const u32x4*>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (col + i < E) q[i] = p[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) r.u[4 * c + i] = q[i];
    }
  }
  return r;
}
template <bool BF>
__device__ __forceinline__ float value_of(const unsigned* u, int i) {
  if constexpr (BF) return __uint_as_float(i & 1 ? u[i >> 1] & 0xFFFF0000u : u[i >> 1] << 16);
  return __uint_as_float(u[i]);
}
template <bool BF>
__device__ __forceinline__ float value_at(const void* logits, size_t at) {
  if constexpr (BF) return __uint_as_float(unsigned(reinterpret_cast<const unsigned short*>(logits)[at]) << 16);
  return reinterpret_cast<const float*>(logits)[at];
}
// Nothing at or below it is a candidate, and NaN is none.
template <bool BF>
__device__ __forceinline__ float lowest() {
  return BF ? __uint_as_float(0xFF7F0000u) : -FLT_MAX;
}
// Greater logit <=> greater unsigned; the two zeros are equal.
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned u = __float_as_uint(v + 0.0f);
  return u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// e^x of x <= 0 with the hardware's 2^t: off by |x| 2^-24 for the product's rounding, a fifth of that for the constant's, and
// 2^-23; results below 2^-126 are zeros. The library's function takes three times as many instructions, and a token has E of these.
__device__ __forceinline__ float exp_down(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// Value i of a lane if it is a candidate, else -inf.
template <bool BF, int V>
__device__ __forceinline__ void candidates(const Raw<BF, V>& r, bool open, float (&v)[V]) {
  const float above = open ? lowest<BF>() : INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float x = value_of<BF>(r.u, i);
    v[i] = x > above ? x : -INFINITY;
  }
}
template <int V>
__device__ __forceinline__ float lane_max(const float (&v)[V]) {
  float m = v[V - 1];
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) m = fmaxf(fmaxf(m, v[i]), v[i + 1]);
  return m;
}

// The greatest of a lane's keys below `last`, 0 if there is none. Keys have 31 bits, so of their distances from `last` (mod 2^32) those of
// smaller keys are above 2^31 and the others below, and nothing has to be struck out: three instructions for two keys.
template <int V>
__device__ __forceinline__ unsigned next_below(const unsigned (&key)[V], unsigned last) {
  unsigned best = key[V - 1] - last;
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) best = umax(umax(best, key[i] - last), key[i + 1] - last);
  return best >> 31 ? best + last : 0u;
}

// Winner j of a token lies in lane j % 16, the second sixteen in `second`: 1 + its column, 0 for a slot that stays empty.
struct Winners {
  unsigned first, second;
};

// v: candidates(). again(): the row once more, for the tokens that are taken by whole logits; kept in registers it would cost all others.
template <bool BF, int V, typename Again>
__device__ __forceinline__ Winners pick(const float (&v)[V], Again again, int lane, int E, int k) {
  // 31 bits: the logit's 16 (bfloat16) or first 23, and its place backwards, so that equals go to the lowest one; no two are equal
  unsigned key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) key[i] = (BF ? ordered(v[i]) >> 16 << 8 : ordered(v[i]) >> 1 & 0x7FFFFF00u) | (255 - column(lane, i));
  // of the lowest candidate: all others' keys are those of -inf, which are below
  const unsigned least = BF ? ordered(lowest<BF>()) >> 16 << 8 : ordered(lowest<BF>()) >> 1 & 0x7FFFFF00u;
  // A lane's three greatest in order. When the third is taken, though nobody may want a fourth, that one is looked for: at k=8 for 1
  // wave's pass in 3 (E=64) to 6 in 10 (E=256), at E=256, k=16 and 32 for nearly every one.
  unsigned t0 = key[V - 1];
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) t0 = umax(umax(t0, key[i]), key[i + 1]);
  unsigned t1 = next_below<V>(key, t0), t2 = next_below<V>(key, t1);
  const int rounds = BF ? k : min(k + 1, E);
  unsigned last = 0, first = 0, second = 0;
  for (int j = 0; j < rounds; ++j) {
    last = row16_max(t0);
    if (j < k && lane == (j & 15)) {
      if (j < 16) first = last;
      else second = last;
    }
    const bool mine = t0 == last;
    t0 = mine ? t1 : t0, t1 = mine ? t2 : t1, t2 = mine ? 0u : t2;
    if (__any(mine && t0 == 0u)) {
      if (mine && t0 == 0u) t0 = next_below<V>(key, last);
    }
  }
  const auto slot = [&](unsigned won) { return won >= least ? 256 - (won & 255) : 0u; };
  Winners w = {slot(first), slot(second)};
  if constexpr (!BF) {
    // `last` is winner k's if there was a round for it
    const unsigned extra = rounds > k ? last : 0u;
    unsigned after = static_cast<unsigned>(dpp<kNextLane>(static_cast<int>(first)));
    unsigned after2 = static_cast<unsigned>(dpp<kNextLane>(static_cast<int>(second)));
    const unsigned second0 = __shfl(second, 0, 16);
    if (lane == 15) after = second0;
    if (lane == k - 1) after = extra;
    if (lane == k - 17) after2 = extra;
    const bool near = (lane < k && first >= least && (first ^ after) >> 8 == 0) ||
                      (lane + 16 < k && second >= least && (second ^ after2) >> 8 == 0);
    if (__any(near)) {
      float x[V];
      again(x);
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = x[i] > -INFINITY ? ordered(x[i]) : 0u;
      w = {0u, 0u};
      for (int j = 0; j < k; ++j) {
        unsigned best = 0, at = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (key[i] > best) best = key[i], at = column(lane, i) + 1;
        const unsigned most = row16_max(best);
        const unsigned won = row16_min(most != 0 && best == most ? at : 0xFFFFu);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (column(lane, i) + 1 == won) key[i] = 0u;
        if (lane == (j & 15)) {
          if (j < 16) w.first = most != 0 ? won : 0u;
          else w.second = most != 0 ? won : 0u;
        }
      }
    }
  }
  return w;
}

struct Totals {
  double both, squares;  // sum of counts times probabilities, of squared logsumexps
  int slots, rows;
};
// By one whole workgroup; thread e < E has expert e's count and sum of probabilities, any thread some of the squares and of the rows.
__device__ __forceinline__ void finish(const RouteArgs& a, int count, double probs, double squares, int rows, Totals* room) {
  const bool mine = static_cast<int>(threadIdx.x) < a.E;
  if (mine) a.counts[threadIdx.x] = count;
  if (mine && a.kept != nullptr) a.kept[2 + threadIdx.x] = count;
  const Totals wave{wave_sum(mine ? count * probs : 0.0), wave_sum(squares), wave_sum(mine ? count : 0), wave_sum(rows)};
  if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = wave;
  __syncthreads();
  if (threadIdx.x != 0) return;
  Totals t{};
  for (unsigned i = 0; i < blockDim.x / 64; ++i)
    t.both += room[i].both, t.squares += room[i].squares, t.slots += room[i].slots, t.rows += room[i].rows;
  if (a.kept != nullptr) a.kept[0] = t.rows, a.kept[1] = t.slots;
  *a.balance = static_cast<float>(t.slots > 0 ? a.E * t.both / (static_cast<double>(t.slots) * t.rows) : t.both);
  *a.zed = static_cast<float>(t.rows > 0 ? t.squares / t.rows : t.squares);
}

template <bool BF, int V, bool WHOLE>
__global__ __launch_bounds__(1024) void route_kernel(RouteArgs a) {
  __shared__ int hist[kRouteExperts];
  __shared__ float probs[16][kRouteExperts];
  __shared__ Totals room[16];
  const int lane = threadIdx.x & 15, wave = threadIdx.x >> 6;
  const int rows_here = blockDim.x / 16;
  const long long step = static_cast<long long>(gridDim.x) * rows_here;
  for (int e = threadIdx.x; e < kRouteExperts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  float sum[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  float squares = 0.0f;
  int rows = 0;
  long long row = static_cast<long long>(blockIdx.x) * rows_here + (threadIdx.x >> 4);
  // rows behind the last one are read as the last one and count for nothing
  const auto place = [&](long long r) { return static_cast<size_t>(min(r, a.T - 1LL)) * a.ld; };
  // the next row is asked for while this one is worked on, but of sixteen values a lane, where four waves hide each other's loads
  // and the registers are needed (with 33 of them in scratch T=131072, E=256 took 114 us instead of 54)
  constexpr bool kAhead = V < 16;
  Raw<BF, V> next{};
  if (kAhead && a.T > 0) next = load_row<BF, V, WHOLE>(a.logits, place(row), lane, a.E);
  // all of a wave's rows go round together: the cross-lane steps need every lane
  for (long long first = row - (threadIdx.x >> 4 & 3); first < a.T; first += step, row += step) {
    Raw<BF, V> now = next;
    if constexpr (!kAhead) now = load_row<BF, V, WHOLE>(a.logits, place(row), lane, a.E);
    if (kAhead && first + step < a.T) next = load_row<BF, V, WHOLE>(a.logits, place(row + step), lane, a.E);
    const bool open = row < a.T && (a.mask == nullptr || a.mask[row] != 0);
    float v[V], e[V], s = 0.0f;
    candidates(now, open, v);
    float m = row16_max(lane_max(v));
    const bool some = m > -INFINITY;
    m = some ? m : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = exp_down(v[i] - m), s += e[i];
    s = row16_sum(s);
    const float each = some ? 1.0f / s : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = fmaf(e[i], each, sum[i]);
    if (lane == 0 && some) {
      const float lse = m + logf(s);
      squares = fmaf(lse, lse, squares);
      ++rows;
    }
    const auto again = [&](float (&x)[V]) {
      asm volatile("" ::: "memory");
      candidates(load_row<BF, V, WHOLE>(a.logits, place(row), lane, a.E), open, x);
    };
    const Winners w = pick<BF, V>(v, again, lane, a.E, a.k);
    const float w0 = w.first != 0 ? exp_down(value_at<BF>(a.logits, place(row) + w.first - 1) - m) : 0.0f;
    const float w1 = w.second != 0 ? exp_down(value_at<BF>(a.logits, place(row) + w.second - 1) - m) : 0.0f;
    const float of = a.renormalize ? row16_sum(w0 + w1) : s;
    const float share = some ? 1.0f / of : 0.0f;
    if (row < a.T) {
      const size_t at = static_cast<size_t>(row) * a.k + lane;
      if (lane < a.k) {
        a.weights[at] = w0 * share;
        a.experts[at] = static_cast<int>(w.first) - 1;
        if (w.first != 0) atomicAdd(&hist[w.first - 1], 1);
      }
      if (lane + 16 < a.k) {
        a.weights[at + 16] = w1 * share;
        a.experts[at + 16] = static_cast<int>(w.second) - 1;
        if (w.second != 0) atomicAdd(&hist[w.second - 1], 1);
      }
    }
  }
  // the wave's four tokens at a time, then the waves, in one order
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float v = sum[i];
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    if ((threadIdx.x & 63) < 16 && column(lane, i) < kRouteExperts) probs[wave][column(lane, i)] = v;
  }
  __syncthreads();
  const int e = threadIdx.x, waves = blockDim.x / 64;
  float p = 0.0f;
  if (e < a.E)
    for (int i = 0; i < waves; ++i) p += probs[i][e];
  if (gridDim.x == 1) {
    finish(a, e < a.E ? hist[e] : 0, p, squares, rows, room);
    return;
  }
  float* sums = a.partial + static_cast<size_t>(blockIdx.x) * kRouteColumns;
  int* counts = reinterpret_cast<int*>(a.partial + static_cast<size_t>(gridDim.x + blockIdx.x) * kRouteColumns);
  if (e < a.E) sums[e] = p, counts[e] = hist[e];
  const float wave_squares = wave_sum(squares);
  const int wave_rows = wave_sum(rows);
  if ((e & 63) == 0) room[wave].squares = wave_squares, room[wave].rows = wave_rows;
  __syncthreads();
  if (e == 0) {
    double all_squares = 0.0;
    int all_rows = 0;
    for (int i = 0; i < waves; ++i) all_squares += room[i].squares, all_rows += room[i].rows;
    sums[kRouteExperts] = static_cast<float>(all_squares), counts[kRouteExperts] = all_rows;
  }
}

// The workgroups' sums, by one: four threads to a column.
__global__ __launch_bounds__(1024) void route_finish_kernel(RouteArgs a, int blocks) {
  __shared__ double probs[4][kRouteExperts];
  __shared__ int counts[4][kRouteExperts];
  __shared__ Totals room[16];
  const int e = threadIdx.x & 255, part = threadIdx.x >> 8;
  const int* partial_counts = reinterpret_cast<const int*>(a.partial + static_cast<size_t>(blocks) * kRouteColumns);
  double p = 0.0;
  int c = 0;
  if (e < a.E) {
#pragma unroll 16
    for (int b = part; b < blocks; b += 4) {
      p += a.partial[static_cast<size_t>(b) * kRouteColumns + e];
      c += partial_counts[static_cast<size_t>(b) * kRouteColumns + e];
    }
  }
  probs[part][e] = p, counts[part][e] = c;
  double squares = 0.0;
  int rows = 0;
  if (static_cast<int>(threadIdx.x) < blocks) {
    squares = a.partial[static_cast<size_t>(threadIdx.x) * kRouteColumns + kRouteExperts];
    rows = partial_counts[static_cast<size_t>(threadIdx.x) * kRouteColumns + kRouteExperts];
  }
  __syncthreads();
  p = (probs[0][e] + probs[1][e]) + (probs[2][e] + probs[3][e]);
  c = (counts[0][e] + counts[1][e]) + (counts[2][e] + counts[3][e]);
  finish(a, c, p, squares, rows, room);
}

template <bool BF, int V, bool WHOLE>
__global__ __launch_bounds__(256) void route_backward_kernel(RouteArgs a) {
  // what the winners' weights add to a token's gradient, where each lane finds its columns
  __shared__ __align__(16) float add[16][kRouteExperts];
  const int lane = threadIdx.x & 15;
  float* mine = add[threadIdx.x >> 4];
  const int n = a.kept[0], slots = a.kept[1];
  const float toward = a.dbalance != nullptr && slots > 0 ? *a.dbalance * a.E / (static_cast<float>(slots) * n) : 0.0f;
  const float pull = a.dzed != nullptr && n > 0 ? 2.0f * *a.dzed / n : 0.0f;
  float g[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = column(lane, i);
    g[i] = c < a.E ? toward * a.kept[2 + c] : 0.0f;
    mine[c] = 0.0f;
  }
  const long long step = static_cast<long long>(gridDim.x) * 16;
  long long row = static_cast<long long>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const auto place = [&](long long r) { return static_cast<size_t>(min(r, a.T - 1LL)); };
  struct Slot {
    int expert;
    float weight, d;
  };
  const auto slot_at = [&](size_t r, int j) {
    const size_t at = r * a.k + j;
    if (j >= a.k) return Slot{-1, 0.0f, 0.0f};
    return Slot{a.experts[at], a.weights[at], a.dweights != nullptr ? a.dweights[at] : 0.0f};
  };
  Raw<BF, V> next = load_row<BF, V, WHOLE>(a.logits, place(row) * a.ld, lane, a.E);
  Slot coming = slot_at(place(row), lane), coming2 = slot_at(place(row), lane + 16);
  for (long long first = row - (threadIdx.x >> 4 & 3); first < a.T; first += step, row += step) {
    const Raw<BF, V> now = next;
    if (first + step < a.T) next = load_row<BF, V, WHOLE>(a.logits, place(row + step) * a.ld, lane, a.E);
    const bool open = row < a.T && (a.mask == nullptr || a.mask[row] != 0);
    // a slot that nobody won has a constant weight, whatever its gradient is said to be
    const auto won = [&](const Slot& s) { return static_cast<unsigned>(s.expert) < static_cast<unsigned>(a.E) ? s : Slot{-1, 0.0f, 0.0f}; };
    const Slot one = won(coming), two = won(coming2);
    if (first + step < a.T) coming = slot_at(place(row + step), lane), coming2 = slot_at(place(row + step), lane + 16);
    const int e0 = open ? one.expert : -1, e1 = open ? two.expert : -1;
    float v[V], p[V], s = 0.0f;
    candidates(now, open, v);
    float m = row16_max(lane_max(v));
    const bool some = m > -INFINITY;
    m = some ? m : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = exp_down(v[i] - m), s += p[i];
    s = row16_sum(s);
    const float each = some ? 1.0f / s : 0.0f;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] *= each, dot = fmaf(p[i], g[i], dot);
    // the weights' own slope: winners alone under renormalisation, else p's among the others
    const float mean = a.renormalize ? row16_sum(one.weight * one.d + two.weight * two.d) : 0.0f;
    const float a0 = one.weight * (one.d - mean), a1 = two.weight * (two.d - mean);
    if (!a.renormalize) dot += a0 + a1;
    dot = row16_sum(dot);
    if (e0 >= 0) mine[e0] = a0;
    if (e1 >= 0) mine[e1] = a1;
    wave_lds_ready();
    const float zed = some ? pull * (m + logf(s)) - dot : 0.0f;
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = fmaf(p[i], g[i] + zed, mine[column(lane, i)]);
    wave_lds_ready();
    if (e0 >= 0) mine[e0] = 0.0f;
    if (e1 >= 0) mine[e1] = 0.0f;
    if (row < a.T) {
#pragma unroll
      for (int c = 0; c < V / 4; ++c) {
        const int col = c * 64 + lane * 4;
        const float* v = d + 4 * c;
        if constexpr (BF) {
          unsigned short* to = reinterpret_cast<unsigned short*>(a.dlogits) + static_cast<size_t>(row) * a.ldd + col;
          const u32x2 q = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
          if constexpr (WHOLE) {
            if (col < a.E) *reinterpret_cast<u32x2*>(to) = q;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (col + i < a.E) to[i] = static_cast<unsigned short>(q[i >> 1] >> (16 * (i & 1)));
          }
        } else {
          float* to = reinterpret_cast<float*>(a.dlogits) + static_cast<size_t>(row) * a.ldd + col;
          if constexpr (WHOLE) {
            if (col < a.E) *reinterpret_cast<f32x4*>(to) = f32x4{v[0], v[1], v[2], v[3]};
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (col + i < a.E) to[i] = v[i];
          }
        }
      }
    }
  }
}

// Rows that begin on four values, E a multiple of four: loads and stores of four at a time.
bool whole_fours(const void* p, long long ld, int E, int dtype) {
  const int size = dtype == 0 ? 4 : 2;
  return E % 4 == 0 && ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (4 * size) == 0;
}

template <bool BF, int V, bool WHOLE>
void enqueue(const RouteArgs& a, bool backward, hipStream_t stream) {
  if (backward) {
    // eight workgroups of four waves a CU
    const long long blocks = (a.T + 15LL) / 16;
    route_backward_kernel<BF, V, WHOLE><<<dim3(static_cast<unsigned>(blocks < 2048 ? blocks : 2048)), dim3(256), 0, stream>>>(a);
    return;
  }
  const RouteGrid g = route_grid(a.T);
  route_kernel<BF, V, WHOLE><<<dim3(g.blocks), dim3(g.threads), 0, stream>>>(a);
  if (g.blocks > 1) route_finish_kernel<<<dim3(1), dim3(1024), 0, stream>>>(a, g.blocks);
}
template <bool BF, int V>
void enqueue(const RouteArgs& a, bool backward, bool whole, hipStream_t stream) {
  whole ? enqueue<BF, V, true>(a, backward, stream) : enqueue<BF, V, false>(a, backward, stream);
}
template <bool BF>
void enqueue(const RouteArgs& a, bool backward, bool whole, hipStream_t stream) {
  if (a.E <= 64) enqueue<BF, 4>(a, backward, whole, stream);
  else if (a.E <= 128) enqueue<BF, 8>(a, backward, whole, stream);
  else enqueue<BF, 16>(a, backward, whole, stream);
}
hipError_t enqueue(const RouteArgs& a, bool backward, int dtype, bool whole, hipStream_t stream) {
  dtype == 0 ? enqueue<false>(a, backward, whole, stream) : enqueue<true>(a, backward, whole, stream);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route(const RouteArgs& a, int dtype, hipStream_t stream) {
  return enqueue(a, false, dtype, whole_fours(a.logits, a.ld, a.E, dtype), stream);
}
hipError_t launch_route_backward(const RouteArgs& a, int dtype, hipStream_t stream) {
  return enqueue(a, true, dtype, whole_fours(a.logits, a.ld, a.E, dtype) && whole_fours(a.dlogits, a.ldd, a.E, dtype), stream);
}

}  // namespace fmoe
