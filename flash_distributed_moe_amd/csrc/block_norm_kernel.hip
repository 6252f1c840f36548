// The norms around a block, fused with what joins it to the residual stream:
//   z = post * branch / rms(branch)  (or the branch as it is),  y = alpha x + beta gate z,  h = next * y / rms(y)
// with rms(v) = sqrt(mean v^2 + eps), and the gradients. Without a branch y = x: the norm in front of a block alone.
//
// Backward, with u = branch / rms and v = y / rms(y), both rebuilt from the inputs (what was rounded into y is not used again):
//   t = dy + (next dh - v mean(next dh v)) / rms(y),  dx = alpha t,  d = beta t
//   dgate = d z,  dpost = sum d gate u,  dbranch = (q - u mean(q u)) / rms(branch) with q = d gate post,  dnext = sum dh v
// A gate a channel and the post norm's weight have one sum between them: with S = sum d u, dgate = post S and dpost = gate S.
// With a gate a token sum q u = gate sum d z, so its gradient needs no sum of its own.
//
// Bound by memory: every array is read or written once, rows stay in registers between the two norms. A row belongs to one
// wave or to several, which exchange their sums through LDS; the backward pass's column sums stay in registers over all rows of a
// workgroup and are joined by a second kernel, in one order.
#include "ffn_device.h"
#include "lane_device.h"
#include "layer_params.h"

namespace fmoe {
namespace {

template <bool BF>
constexpr int kPiece = BF ? 8 : 4;  // values in 16 bytes

// V pieces of a row: piece i of a lane is number i * lanes + lane of the row's.
template <int V>
struct Pieces {
  u32x4 u[V];
};
template <bool BF, int V>
__device__ __forceinline__ Pieces<V> load_pieces(const void* p, size_t at, int first, int apart, int count) {
  Pieces<V> r;
  const char* base = reinterpret_cast<const char*>(p) + at * (BF ? 2 : 4);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int n = first + i * apart;
    r.u[i] = n < count ? *reinterpret_cast<const u32x4*>(base + static_cast<size_t>(n) * 16) : u32x4{0, 0, 0, 0};
  }
  return r;
}
template <bool BF>
__device__ __forceinline__ float piece_value(const u32x4& u, int j) {
  if constexpr (BF) return __uint_as_float(j & 1 ? u[j >> 1] & 0xFFFF0000u : u[j >> 1] << 16);
  return __uint_as_float(u[j]);
}
template <bool BF>
__device__ __forceinline__ u32x4 pack_piece(const float* v) {
  if constexpr (BF) return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])};
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
template <bool BF, int V>
__device__ __forceinline__ void store_pieces(void* p, size_t at, int first, int apart, int count, const float* v) {
  char* base = reinterpret_cast<char*>(p) + at * (BF ? 2 : 4);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int n = first + i * apart;
    if (n < count) *reinterpret_cast<u32x4*>(base + static_cast<size_t>(n) * 16) = pack_piece<BF>(v + i * kPiece<BF>);
  }
}
template <bool BF>
__device__ __forceinline__ float one_value(const void* p, size_t at) {
  if constexpr (BF) return __uint_as_float(unsigned(reinterpret_cast<const unsigned short*>(p)[at]) << 16);
  return reinterpret_cast<const float*>(p)[at];
}
template <bool BF>
__device__ __forceinline__ void put_value(void* p, size_t at, float v) {
  if constexpr (BF) reinterpret_cast<unsigned short*>(p)[at] = static_cast<unsigned short>(pack_bf16(v, v));
  else reinterpret_cast<float*>(p)[at] = v;
}

// The sum over a row's waves; `room` has a place for each wave of the workgroup. Every wave comes by.
__device__ __forceinline__ float row_sum(float v, int waves, float* room) {
  v = wave_sum(v);
  if (waves == 1) return v;
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) room[wave] = v;
  __syncthreads();
  const int first = wave & ~(waves - 1);
  float sum = 0.0f;
  for (int i = 0; i < waves; ++i) sum += room[first + i];
  return sum;
}

__device__ __forceinline__ size_t gate_row(const NormArgs& a, long long row) {
  return a.gate_kind == GATE_CHANNEL ? 0 : a.gate_kind == GATE_GROUP ? row / a.shared : row;
}

template <bool BF, int V>
__global__ void norm_kernel(NormArgs a, int waves) {
  constexpr int P = kPiece<BF>, N = V * P;
  __shared__ float room[2][16];
  const int lanes = waves * 64, first = threadIdx.x & (lanes - 1), count = a.H / P;
  const int at_once = blockDim.x / lanes;
  for (long long start = static_cast<long long>(blockIdx.x) * at_once; start < a.T; start += static_cast<long long>(gridDim.x) * at_once) {
    const long long want = start + threadIdx.x / lanes, row = min(want, a.T - 1LL);
    const Pieces<V> x = load_pieces<BF, V>(a.x, row * a.ldx, first, lanes, count);
    float y[N];
    if (a.branch != nullptr) {
      const Pieces<V> b = load_pieces<BF, V>(a.branch, row * a.ldb, first, lanes, count);
      float scale = a.beta;
      if (a.post != nullptr) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(piece_value<BF>(b.u[i / P], i % P), piece_value<BF>(b.u[i / P], i % P), s);
        const float rms = rsqrtf(row_sum(s, waves, room[0]) / a.H + a.eps);
        if (first == 0 && want < a.T && a.branch_rms != nullptr) a.branch_rms[row] = rms;
        const Pieces<V> w = load_pieces<BF, V>(a.post, 0, first, lanes, count);
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(b.u[i / P], i % P) * rms * piece_value<BF>(w.u[i / P], i % P);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(b.u[i / P], i % P);
      }
      if (a.gate_kind == GATE_TOKEN) {
        scale *= one_value<BF>(a.gate, row);
      } else if (a.gate_kind != GATE_NONE) {
        const Pieces<V> g = load_pieces<BF, V>(a.gate, gate_row(a, row) * a.H, first, lanes, count);
#pragma unroll
        for (int i = 0; i < N; ++i) y[i] *= piece_value<BF>(g.u[i / P], i % P);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = fmaf(scale, y[i], a.alpha * piece_value<BF>(x.u[i / P], i % P));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = piece_value<BF>(x.u[i / P], i % P);
    }
    if (a.y != nullptr && want < a.T) store_pieces<BF, V>(a.y, row * a.H, first, lanes, count, y);
    if (a.next != nullptr) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(y[i], y[i], s);
      const float rms = rsqrtf(row_sum(s, waves, room[1]) / a.H + a.eps);
      if (first == 0 && want < a.T && a.y_rms != nullptr) a.y_rms[row] = rms;
      const Pieces<V> w = load_pieces<BF, V>(a.next, 0, first, lanes, count);
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = y[i] * rms * piece_value<BF>(w.u[i / P], i % P);
      if (want < a.T) store_pieces<BF, V>(a.h, row * a.H, first, lanes, count, y);
    }
    // a wave that is ahead writes its next sums where another may still read these
    if (waves > 1 && (a.post == nullptr || a.next == nullptr)) __syncthreads();
  }
}

// The workgroup's column sums: each row's waves have one, and they are added in one order.
template <bool BF>
__device__ __forceinline__ void join_rows(float* acc, float* room, int lanes, int first, int count, float* to, void* rounded) {
  constexpr int P = kPiece<BF>, V = kNormLane / P;
  const int mine = threadIdx.x / lanes, rows = kNormThreads / lanes;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int n = first + i * lanes;
    if (n < count) {
#pragma unroll
      for (int j = 0; j < P; ++j) room[mine * count * P + n * P + j] = acc[i * P + j];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < count * P; c += kNormThreads) {
    float s = 0.0f;
    for (int r = 0; r < rows; ++r) s += room[r * count * P + c];
    if (rounded != nullptr) put_value<BF>(rounded, c, s);
    else to[c] = s;
  }
}

template <bool BF, int GATE>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(NormArgs a) {
  constexpr int P = kPiece<BF>, V = kNormLane / P, N = kNormLane;
  __shared__ float room[2][16];
  extern __shared__ __align__(16) float columns[];
  const int waves = norm_waves(a.H), lanes = waves * 64, first = threadIdx.x & (lanes - 1), count = a.H / P;
  const int at_once = kNormThreads / lanes, mine = threadIdx.x / lanes;
  const bool next = a.next != nullptr && a.dh != nullptr, post = a.post != nullptr, branch = a.branch != nullptr;
  float sum_next[N], sum_post[GATE == GATE_CHANNEL ? 1 : N], sum_gate[GATE == GATE_CHANNEL || GATE == GATE_GROUP ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum_next[i] = 0.0f;
    if constexpr (GATE != GATE_CHANNEL) sum_post[i] = 0.0f;
    if constexpr (GATE == GATE_CHANNEL || GATE == GATE_GROUP) sum_gate[i] = 0.0f;
  }
  Pieces<V> wn{}, wp{}, g{};
  if (next) wn = load_pieces<BF, V>(a.next, 0, first, lanes, count);
  if (post) wp = load_pieces<BF, V>(a.post, 0, first, lanes, count);
  if constexpr (GATE == GATE_CHANNEL) g = load_pieces<BF, V>(a.gate, 0, first, lanes, count);

  // the rows of this workgroup: of all, or of one group after the other
  long long group = 0, groups = 1;
  if constexpr (GATE == GATE_GROUP) {
    if (a.parts > 0) group = blockIdx.x / a.parts;
    else group = static_cast<long long>(blockIdx.x) * a.groups, groups = min(static_cast<long long>(a.groups), a.T / a.shared - group);
  }
  for (const long long last = group + groups; group < last; ++group) {
    long long start = static_cast<long long>(blockIdx.x) * at_once, end = a.T, step = static_cast<long long>(gridDim.x) * at_once;
    if constexpr (GATE == GATE_GROUP) {
      start = group * a.shared, end = start + a.shared, step = at_once;
      if (a.parts > 0) {
        const long long part = (a.shared + a.parts - 1LL) / a.parts;
        start = min(start + blockIdx.x % a.parts * part, end);
        end = min(start + part, end);
      }
      g = load_pieces<BF, V>(a.gate, group * a.H, first, lanes, count);
    }
    for (; start < end; start += step) {
      const long long want = start + mine, row = min(want, end - 1);
      const bool real = want < end;  // rows behind the last one are taken for a second time, and count for nothing
      const Pieces<V> xs = load_pieces<BF, V>(a.x, row * a.ldx, first, lanes, count);
      Pieces<V> bs{}, dys{}, dhs{};
      if (branch) bs = load_pieces<BF, V>(a.branch, row * a.ldb, first, lanes, count);
      if (next) dhs = load_pieces<BF, V>(a.dh, row * a.lddh, first, lanes, count);
      if (a.dy != nullptr) dys = load_pieces<BF, V>(a.dy, row * a.lddy, first, lanes, count);
      if constexpr (GATE == GATE_FULL) g = load_pieces<BF, V>(a.gate, row * a.H, first, lanes, count);
      const float scalar = GATE == GATE_TOKEN ? one_value<BF>(a.gate, row) : 1.0f;
      const float rb = post ? a.branch_rms[row] : 1.0f, ry = next ? a.y_rms[row] : 0.0f;
      const auto gate_of = [&](int i) {
        if constexpr (GATE == GATE_NONE) return 1.0f;
        if constexpr (GATE == GATE_TOKEN) return scalar;
        return piece_value<BF>(g.u[i / P], i % P);
      };
      float t[N], s = 0.0f;
      if (next) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float y = piece_value<BF>(xs.u[i / P], i % P);
          if (branch) {
            const float u = piece_value<BF>(bs.u[i / P], i % P) * rb, z = post ? u * piece_value<BF>(wp.u[i / P], i % P) : u;
            y = fmaf(a.beta * gate_of(i), z, a.alpha * y);
          }
          const float v = y * ry, dh = piece_value<BF>(dhs.u[i / P], i % P);
          sum_next[i] = real ? fmaf(dh, v, sum_next[i]) : sum_next[i];
          t[i] = v;
          s = fmaf(dh * piece_value<BF>(wn.u[i / P], i % P), v, s);
        }
        const float mean = row_sum(s, waves, room[0]) / a.H;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float q = piece_value<BF>(dhs.u[i / P], i % P) * piece_value<BF>(wn.u[i / P], i % P);
          t[i] = fmaf(ry, q - t[i] * mean, piece_value<BF>(dys.u[i / P], i % P));
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = piece_value<BF>(dys.u[i / P], i % P);
      }
      float out[N];
      if (a.dx != nullptr && real) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = a.alpha * t[i];
        store_pieces<BF, V>(a.dx, row * a.H, first, lanes, count, out);
      }
      if (!branch) {
        if (waves > 1) __syncthreads();
        continue;
      }
      s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = a.beta * t[i], u = piece_value<BF>(bs.u[i / P], i % P) * rb, w = post ? piece_value<BF>(wp.u[i / P], i % P) : 1.0f;
        if constexpr (GATE == GATE_CHANNEL) sum_gate[i] = real ? fmaf(d, u, sum_gate[i]) : sum_gate[i];
        if constexpr (GATE == GATE_GROUP) sum_gate[i] = real ? fmaf(d, u * w, sum_gate[i]) : sum_gate[i];
        if constexpr (GATE != GATE_CHANNEL) sum_post[i] = real ? fmaf(d * gate_of(i), u, sum_post[i]) : sum_post[i];
        if constexpr (GATE == GATE_FULL) out[i] = d * u * w;
        s = fmaf(GATE == GATE_TOKEN ? d * w : d * w * gate_of(i), u, s);
        t[i] = d * gate_of(i) * w;
      }
      if constexpr (GATE == GATE_FULL) {
        if (a.dgate != nullptr && real) store_pieces<BF, V>(a.dgate, row * a.H, first, lanes, count, out);
      }
      if (post || GATE == GATE_TOKEN) {
        s = row_sum(s, waves, room[1]);
        if constexpr (GATE == GATE_TOKEN) {
          if (a.dgate != nullptr && real && first == 0) put_value<BF>(a.dgate, row, s);
          s *= scalar;
        }
      }
      if (post) {
        const float mean = s / a.H;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = rb * (t[i] - piece_value<BF>(bs.u[i / P], i % P) * rb * mean);
      }
      if (a.dbranch != nullptr && real) store_pieces<BF, V>(a.dbranch, row * a.H, first, lanes, count, t);
      if (waves > 1 && !(next && (post || GATE == GATE_TOKEN))) __syncthreads();
    }
    if constexpr (GATE == GATE_GROUP) {
      if (a.dgate != nullptr) {
        float* to = a.partial + (static_cast<size_t>(2) * a.blocks + blockIdx.x) * a.H;
        void* whole = a.parts > 0 ? nullptr : static_cast<char*>(a.dgate) + group * a.H * (BF ? 2 : 4);
        join_rows<BF>(sum_gate, columns, lanes, first, count, to, whole);
#pragma unroll
        for (int i = 0; i < N; ++i) sum_gate[i] = 0.0f;
      }
    }
  }
  float* to = a.partial + static_cast<size_t>(blockIdx.x) * a.H;
  if (next && a.dnext != nullptr) join_rows<BF>(sum_next, columns, lanes, first, count, to, nullptr);
  to += static_cast<size_t>(a.blocks) * a.H;
  if constexpr (GATE == GATE_CHANNEL) {
    if (a.dgate != nullptr || a.dpost != nullptr) join_rows<BF>(sum_gate, columns, lanes, first, count, to, nullptr);
  } else {
    if (a.dpost != nullptr) join_rows<BF>(sum_post, columns, lanes, first, count, to, nullptr);
  }
}

// Column sums of the workgroups: 64 columns by sixteen threads each. y: 0 the next norm's weight, 1 the post norm's (and the
// gate's of a channel), 2 + g group g's gate.
template <bool BF>
__global__ __launch_bounds__(1024) void norm_finish_kernel(NormArgs a) {
  __shared__ float room[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
  const int which = blockIdx.y < 2 ? blockIdx.y : 2;
  const int rows = which < 2 ? a.blocks : a.parts;
  const float* from = a.partial + static_cast<size_t>(which) * a.blocks * a.H;
  if (which == 2) from += static_cast<size_t>(blockIdx.y - 2) * a.parts * a.H;
  float s = 0.0f;
  if (c < a.H) {
#pragma unroll 4
    for (int r = part; r < rows; r += 16) s += from[static_cast<size_t>(r) * a.H + c];
  }
  room[part][threadIdx.x & 63] = s;
  __syncthreads();
  if (part != 0 || c >= a.H) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += room[i][threadIdx.x & 63];
  if (which == 0) {
    // without a gradient of h nothing reaches its norm's weight
    if (a.dnext != nullptr) put_value<BF>(a.dnext, c, a.dh != nullptr ? s : 0.0f);
  } else if (which == 2) {
    put_value<BF>(a.dgate, static_cast<size_t>(blockIdx.y - 2) * a.H + c, s);
  } else if (a.gate_kind == GATE_CHANNEL) {
    if (a.dgate != nullptr) put_value<BF>(a.dgate, c, a.post != nullptr ? s * one_value<BF>(a.post, c) : s);
    if (a.dpost != nullptr) put_value<BF>(a.dpost, c, s * one_value<BF>(a.gate, c));
  } else if (a.dpost != nullptr) {
    put_value<BF>(a.dpost, c, s);
  }
}

template <bool BF>
void enqueue_forward(const NormArgs& a, hipStream_t stream) {
  constexpr int P = kPiece<BF>, M = 32 / P;  // pieces of up to 32 values a lane
  const int pieces = a.H / P;
  // few rows are spread over as many lanes as they have pieces, many over as few waves as hold them
  const bool few = a.T < 1024;
  int waves = 1;
  while (waves < (few ? 16 : 8) && waves * 64 * (few ? 1 : M) < pieces) waves *= 2;
  const int threads = waves > 4 ? waves * 64 : 256, at_once = threads / (waves * 64);
  const long long blocks = (a.T + at_once - 1LL) / at_once;
  const dim3 grid(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), block(threads);
  const int each = (pieces + waves * 64 - 1) / (waves * 64);
  if (each <= 1) norm_kernel<BF, 1><<<grid, block, 0, stream>>>(a, waves);
  else if (each <= 2) norm_kernel<BF, 2><<<grid, block, 0, stream>>>(a, waves);
  else if (each <= 4) norm_kernel<BF, 4><<<grid, block, 0, stream>>>(a, waves);
  else if constexpr (!BF) norm_kernel<BF, 8><<<grid, block, 0, stream>>>(a, waves);
}

template <bool BF>
void enqueue_backward(const NormArgs& a, hipStream_t stream) {
  const int rows = kNormThreads / 64 / norm_waves(a.H);
  const size_t room = static_cast<size_t>(rows) * a.H * 4;
  const dim3 grid(a.blocks), block(kNormThreads);
  switch (a.gate_kind) {
    case GATE_NONE: norm_backward_kernel<BF, GATE_NONE><<<grid, block, room, stream>>>(a); break;
    case GATE_CHANNEL: norm_backward_kernel<BF, GATE_CHANNEL><<<grid, block, room, stream>>>(a); break;
    case GATE_GROUP: norm_backward_kernel<BF, GATE_GROUP><<<grid, block, room, stream>>>(a); break;
    case GATE_TOKEN: norm_backward_kernel<BF, GATE_TOKEN><<<grid, block, room, stream>>>(a); break;
    default: norm_backward_kernel<BF, GATE_FULL><<<grid, block, room, stream>>>(a); break;
  }
  const bool parts = a.gate_kind == GATE_GROUP && a.parts > 0 && a.dgate != nullptr;
  if (a.dnext != nullptr || a.dpost != nullptr || parts || (a.gate_kind == GATE_CHANNEL && a.dgate != nullptr))
    norm_finish_kernel<BF><<<dim3((a.H + 63) / 64, 2 + (parts ? a.T / a.shared : 0)), dim3(1024), 0, stream>>>(a);
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, int dtype, hipStream_t stream) {
  dtype == 0 ? enqueue_forward<false>(a, stream) : enqueue_forward<true>(a, stream);
  return hipGetLastError();
}
hipError_t launch_norm_backward(const NormArgs& a, int dtype, hipStream_t stream) {
  dtype == 0 ? enqueue_backward<false>(a, stream) : enqueue_backward<true>(a, stream);
  return hipGetLastError();
}

}  // namespace fmoe
