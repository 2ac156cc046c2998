// Group norm with an activation on feature maps that lie channels last, several levels behind one another, for gfx950.  For a batch element, a level of
// K keys and a group of C / G channels, with n = K C / G elements:
//
//   m = mean x,  v = mean (x - m)^2,  xhat = (x - m) / sqrt(v + eps),  u = xhat w + b,  y = act(u)
//   dz = dy act'(u),  db = sum dz,  dw = sum dz xhat  (over batch elements, levels and keys)
//   dx = (dz w - (S1 + xhat S2) / n) / sqrt(v + eps),  S1 = sum dz w,  S2 = sum dz w xhat  (over the group)
//
// Levels begin where `level_start` says and end where the next one begins: the k-th level is the k-th smallest start, whatever the table's order, so every key
// from the smallest on belongs to one level and no table can send a kernel outside the tensor.  Keys before that belong to none: their y and dx are zero.
//
// A tile is a run of keys of one batch element, all channels (or a block of them); it holds parts of one level or more, part (tile t, level k) in slot t + k,
// which is another one for every part.  Three launches each way: sums of the parts, the statistics from those, the results; one more each where the gradients' parts of
// a group or the channels' sums of the batch elements are too many to be added up one after the other.
// The parts' sums of squares are about their own means (kept in registers), and are joined by the counts' formula for two samples, so a large mean costs no
// digits.  Bound by memory: x is read twice, dy twice.
#include <algorithm>

#include "../../include/dfa3d.h"
#include "dfa3d_launch.h"
#include "dfa3d_rows.h"

namespace dfa3d {

constexpr int kNormBlock = 256;
constexpr int kSmallBlock = 1024;
// Elements of a batch element's group, all levels, forward and backward, and of the tensor, up to which one workgroup per batch element, level and group does
// it all.  us a pass, small and tiles: 2 x 1500 x 256, 32 groups forward 8.5, 14.6, training 77, 87; 2400 x 64, 4 groups (38400 elements) 9.8, 14.3 and 79,
// 88; 4800 x 256, 32 groups (38400) 15.0, 14.2 and 77, 87; 3 x 3295 x 120, 6 groups (65900) on the device alone 16, 14 and 40, 21.  (What training passes of
// this size take is mostly the launches' share of the host's time.)
// And only as many workgroups: in the backward, of 1024 threads, two a CU (256 x 100 x 64, 8 groups, training 110 us, tiles 66; 64 x 60 x 64, 512 workgroups, 57 and
// 57); forward 512 x 8 x 64, 4096 workgroups, 12.3 and 14.5, 130 x 60 x 256, 4160, 13.8 and 16.3, 250 x 30 x 256, 8000, 22.4 and 18.3, 2048 x 8 x 64 40 and 18.
constexpr long long kSmallElements[2] = {1 << 15, 1 << 16}, kSmallTotal = 1 << 21, kSmallUnits[2] = {5 << 10, 1 << 9};

struct NormDims {
  int B, S, C, G, L;
  int cols, at_once;                   // threads of a key's pieces in a workgroup, and keys at once
  float per_col;                       // 1 / cols
  int tile, tiles, slots;              // keys of a tile, tiles and slots of a batch element
  unsigned first;                      // tile of the first batch element and on that the launch begins with
  float per_piece;                     // 1 / group
  int group, abreast, cells, blocks;   // pieces of a group and groups side by side; the statistics' parts of a tile: one per group, or per block of a group's pieces where those are more than a workgroup
};

// x / n of whole numbers below 2^11, `per` being 1 / n: x + 0.5 is at least 0.5 / n away from a multiple.  (By divisions of integers the
// statistics' parts of 6 x 30825 x 256 in bfloat16 take 22.6 us, so 21.7.)
__device__ __forceinline__ int part_of(int x, float per) { return (int)(((float)x + 0.5f) * per); }

// First keys of the levels, ascending; s_first[L] = S.  All threads of the workgroup come here; a barrier follows.
__device__ __forceinline__ void sort_levels(const int64_t *__restrict__ level_start, int L, int S, int *s_first) {
  for (int l = threadIdx.x; l <= L; l += blockDim.x) {
    if (l == L) {
      s_first[L] = S;
    } else if (level_start == nullptr) {
      s_first[l] = 0;
    } else {
      const int64_t mine = level_start[l];
      int rank = 0;
      for (int k = 0; k < L; ++k) {
        const int64_t s = level_start[k];
        rank += s < mine || (s == mine && k < l);
      }
      s_first[rank] = (int)min(max(mine, (int64_t)0), (int64_t)S);
    }
  }
  __syncthreads();
}

// 1 / (1 + exp(-u)).  In float by the hardware's power of two and reciprocal: the rounding of u log2(e) weighs no more than that of u itself, which has been computed (both
// |u| 2^-24 of the gate, 5e-6 at u = -80); below u = -87 the gate is less than the least float that is not subnormal, and zero.  (The
// library's exponential and a correct division: 6 x 30825 x 256 in bfloat16 61 us for 41.)
__device__ __forceinline__ float gate_of(float u) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.44269504088896341f)); }
__device__ __forceinline__ double gate_of(double u) { return 1.0 / (1.0 + exp(-u)); }
template <int ACT, typename A> __device__ __forceinline__ A activated(A u) {
  if (ACT == DFA3D_ACT_RELU) return u > 0 ? u : u != u ? u : (A)0;
  if (ACT == DFA3D_ACT_SILU) return u * gate_of(u);
  return u;
}
// d * act'(u)
template <int ACT, typename A> __device__ __forceinline__ A through_activation(A d, A u) {
  if (ACT == DFA3D_ACT_RELU) return u > 0 ? d : (A)0;
  if (ACT == DFA3D_ACT_SILU) {
    const A gate = gate_of(u);
    return d * (gate * (1 + u * (1 - gate)));
  }
  return d;
}

// Two samples' count, mean and sum of squares about the mean as one's (T. Chan, G. Golub, R. LeVeque, 1979).  Where one is empty (its mean is zero) it is the other: the square
// of the other one's mean may be infinite, which times no elements is not a number.
template <typename A> struct Moments { A n, mean, m2; };
template <typename A> __device__ __forceinline__ Moments<A> joined(const Moments<A> &a, const Moments<A> &b) {
  if (b.n == 0) return a;
  const A n = a.n + b.n, d = b.mean - a.mean, part = b.n / n;
  return Moments<A>{n, a.mean + d * part, a.m2 + b.m2 + (a.n != 0 ? d * d * a.n * part : (A)0)};
}

// parts (B, slots, cells): mean and sum of squares about it of a part's keys and a group's channels (or a block's of them)
template <typename T, int VEC, int KEYS>
__global__ __launch_bounds__(kNormBlock) void norm_parts_kernel(const T *__restrict__ x, const int64_t *__restrict__ level_start,
                                                                typename Sum<T>::type *__restrict__ parts, NormDims d) {
  typedef typename Sum<T>::type A;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ Moments<A> s_part[kNormBlock];
  const int row = part_of(threadIdx.x, d.per_col), col = threadIdx.x - row * d.cols;
  // whole groups side by side, or a block of one group's pieces
  int piece = blockIdx.y * d.cols + col, pieces = d.group;
  if (d.blocks > 1) {
    const int block = blockIdx.y % d.blocks;
    piece = blockIdx.y / d.blocks * d.group + block * d.cols + col;
    pieces = min(d.group - block * d.cols, d.cols);
  }
  const bool on = row < d.at_once && piece < d.C / VEC && (d.blocks == 1 || col < pieces);
  const unsigned block = d.first + blockIdx.x;
  const long long b = block / d.tiles;
  const int tile = (int)(block - (unsigned)b * d.tiles), k0 = tile * d.tile, k1 = min(k0 + d.tile, d.S);
  const T *from = x + (b * d.S) * d.C + (long long)piece * VEC;
  A v[KEYS][VEC];
#pragma unroll
  for (int i = 0; i < KEYS; ++i) {
    const int k = k0 + i * d.at_once + row;
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[i][c] = 0;
    if (on && k < k1) load_row<T, VEC>(from + (long long)k * d.C, v[i]);
  }
  sort_levels(level_start, d.L, d.S, s_first);               // (the keys are on their way)
  const int nth = d.blocks == 1 ? part_of(col, d.per_piece) : 0, at = col - nth * d.group;         // which group, and which of its (or the block's) pieces
  for (int l = 0; l < d.L; ++l) {
    const int f0 = max(s_first[l], k0), f1 = min(s_first[l + 1], k1);
    if (f0 >= f1) continue;                                  // uniform
    A n = 0, mean = 0, m2 = 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int k = k0 + i * d.at_once + row;
      if (k >= f0 && k < f1) {
        n += VEC;
#pragma unroll
        for (int c = 0; c < VEC; ++c) mean += v[i][c];
      }
    }
    if (!on) n = 0;
    if (n != 0) mean /= n;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      const int k = k0 + i * d.at_once + row;
      if (k >= f0 && k < f1)
#pragma unroll
        for (int c = 0; c < VEC; ++c) m2 += (v[i][c] - mean) * (v[i][c] - mean);
    }
    Moments<A> mine = {n, mean, m2};
    for (int left = d.at_once; left > 1;) {                  // the keys side by side, halved
      const int half = (left + 1) / 2;
      s_part[threadIdx.x] = mine;
      __syncthreads();
      if (row + half < left) mine = joined(mine, s_part[threadIdx.x + half * d.cols]);
      __syncthreads();
      left = half;
    }
    for (int left = pieces; left > 1;) {                     // then the pieces
      const int half = (left + 1) / 2;
      if (row == 0) s_part[threadIdx.x] = mine;
      __syncthreads();
      if (row == 0 && at + half < left) mine = joined(mine, s_part[threadIdx.x + half]);
      __syncthreads();
      left = half;
    }
    if (row == 0 && on && at == 0) {
      A *to = parts + ((b * d.slots + tile + l) * d.cells + blockIdx.y * d.abreast + nth) * 2;
      to[0] = mine.mean;
      to[1] = mine.m2;
    }
  }
}

// x summed over the workgroup's threads, in every thread
template <int THREADS> __device__ __forceinline__ double block_sum(double x, double *s_part) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) s_part[threadIdx.x / kWave] = x;
  __syncthreads();
  x = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) x += s_part[w];
  return x;
}

// Neighbouring units on one XCD (workgroups go to the eight of them in turn), as what they read shares cache lines.
__device__ __forceinline__ long long side_by_side(long long turn, long long units) { return units % 8 == 0 ? turn % 8 * (units / 8) + turn / 8 : turn; }

// x summed over a unit's LANES threads, in each of them
template <int LANES> __device__ __forceinline__ double unit_sum(double x, double *s_part) {
  if constexpr (LANES > kWave) return block_sum<LANES>(x, s_part);
#pragma unroll
  for (int off = (LANES < kWave ? LANES : kWave) / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}
// Threads of a unit, of which there is one per batch element, level and group: a workgroup, or fewer where units are so many that workgroups would take turns
// and what is left of them still holds at once what a unit has.  (2000 x 16 x 256, 32 groups, forward: workgroups 213 us,
// 4 threads each 25.)
static int unit_lanes(long long units, long long each, int held) {
  int lanes = kNormBlock;
  while (lanes > 4 && units * lanes > (1 << 19) && each <= (long long)(lanes / 4) * held) lanes /= 4;
  return lanes;
}

// stats (B, L, G): mean and 1 / sqrt(variance + eps).  The mean of the parts' means first, then their sums of squares and what their means are off by.  In double:
// it is little, and the counts of a large map leave float's whole numbers.
// The parts of a group are few bytes of each line: what bounds this is that they come.  (6 x 30825 x 256 in float, four levels, neighbouring
// groups anywhere and parts asked for in turn 12.3 us, groups side by side 9.6, parts asked for at once 6.7.  With a part for every piece of a group's channels
// instead of one for all of them large groups are many parts: 30000 x 1023, three groups, forward 2690 us, now 102.)
constexpr int kHeldParts = 8;
template <typename A, int LANES>
__global__ __launch_bounds__(kNormBlock) void norm_stats_kernel(const A *__restrict__ parts, const int64_t *__restrict__ level_start, A *__restrict__ stats, NormDims d,
                                                                int vec, double eps) {
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ double s_part[kNormBlock / kWave];
  sort_levels(level_start, d.L, d.S, s_first);
  const int group = d.group, at = threadIdx.x % LANES;
  const long long units = (long long)d.B * d.L * d.G;
  for (long long turn = (long long)blockIdx.x * (kNormBlock / LANES) + threadIdx.x / LANES; turn < units; turn += (long long)gridDim.x * (kNormBlock / LANES)) {
    const long long unit = LANES == kNormBlock ? side_by_side(turn, units) : turn;
    const int g = (int)(unit % d.G), l = (int)(unit / d.G % d.L);
    const long long b = unit / d.G / d.L;
    const int f0 = s_first[l], f1 = s_first[l + 1];
    const int t0 = f0 / d.tile, n = f0 < f1 ? ((f1 - 1) / d.tile - t0 + 1) * d.blocks : 0;
    const A *from = parts + ((b * d.slots + t0 + l) * d.cells + g * d.blocks) * 2;
    // part k: tile t0 + k / blocks, block k % blocks
    auto part = [&](int k) { return from + (d.blocks == 1 ? (long long)k * d.cells : (long long)(k / d.blocks) * d.cells + k % d.blocks) * 2; };
    // up to kHeldParts stay in registers, asked for at once
    A held[kHeldParts][2];
#pragma unroll
    for (int i = 0; i < kHeldParts; ++i) {
      const int k = at + i * LANES;
      held[i][0] = held[i][1] = 0;
      if (k < n) {
        held[i][0] = part(k)[0];
        held[i][1] = part(k)[1];
      }
    }
    const double count = (double)(f1 - f0) * vec * group;
    double mean = 0, m2 = 0;
    for (int pass = 0; pass < 2; ++pass) {
      double sum = 0;
      auto add = [&](int k, A part_mean, A part_m2) {
        const int t = t0 + (d.blocks == 1 ? k : k / d.blocks), pieces = d.blocks == 1 ? group : min(group - k % d.blocks * kNormBlock, kNormBlock);
        const double have = (double)(min(f1, (t + 1) * d.tile) - max(f0, t * d.tile)) * (pieces * vec), off = (double)part_mean - mean;
        sum += pass == 0 ? have * off : (double)part_m2 + have * off * off;
      };
#pragma unroll
      for (int i = 0; i < kHeldParts; ++i)
        if (at + i * LANES < n) add(at + i * LANES, held[i][0], held[i][1]);
#pragma unroll 4
      for (int k = at + kHeldParts * LANES; k < n; k += LANES) add(k, part(k)[0], part(k)[1]);
      sum = unit_sum<LANES>(sum, s_part);
      if (n > 0) (pass == 0 ? mean : m2) = sum / count;
    }
    if (at == 0) {
      stats[unit * 2] = (A)mean;
      stats[unit * 2 + 1] = n > 0 ? (A)(1.0 / sqrt(m2 + eps)) : (A)0;
    }
  }
}

// the channels' weights and biases of a piece
template <int VEC, typename A>
__device__ __forceinline__ void channel_params(const A *__restrict__ weight, const A *__restrict__ bias, int c0, A (&w)[VEC], A (&b)[VEC]) {
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    w[c] = weight != nullptr ? weight[c0 + c] : (A)1;
    b[c] = bias != nullptr ? bias[c0 + c] : (A)0;
  }
}

// grad_weight and grad_bias: the channels' sums over batch elements and levels
struct ParamGrads {
  const double *channels;              // (B, L, C, 2)
  void *weight, *bias;                 // or nullptr
  int BL, C, blocks;
};
template <typename A> __device__ __forceinline__ void param_grads(const ParamGrads &p, int c) {
  if (c >= p.C) return;
  double s1 = 0, s2 = 0;
#pragma unroll 8
  for (int k = 0; k < p.BL; ++k) {
    s1 += p.channels[((long long)k * p.C + c) * 2];
    s2 += p.channels[((long long)k * p.C + c) * 2 + 1];
  }
  if (p.bias != nullptr) ((A *)p.bias)[c] = (A)s1;
  if (p.weight != nullptr) ((A *)p.weight)[c] = (A)s2;
}

// Results of a tile.  BACK: dx from dy and sums (B, L, G, 2), the means of dz w and dz w xhat, and in the first workgroups the gradients of weight and bias;
// otherwise y.
template <typename T, int VEC, int ACT, bool BACK>
__global__ __launch_bounds__(kNormBlock) void norm_apply_kernel(const T *__restrict__ x, const T *__restrict__ dy, const typename Sum<T>::type *__restrict__ weight,
                                                                const typename Sum<T>::type *__restrict__ bias, const int64_t *__restrict__ level_start,
                                                                const typename Sum<T>::type *__restrict__ stats, const typename Sum<T>::type *__restrict__ sums,
                                                                T *__restrict__ out, NormDims d, ParamGrads params) {
  typedef typename Sum<T>::type A;
  constexpr int kAhead = 4;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  if (BACK && (int)blockIdx.x < params.blocks) {             // uniform
    if (blockIdx.y == 0) param_grads<A>(params, blockIdx.x * kNormBlock + threadIdx.x);
    return;
  }
  const int per = d.C / VEC, row = part_of(threadIdx.x, d.per_col), piece = blockIdx.y * d.cols + threadIdx.x - row * d.cols;
  const bool on = row < d.at_once && piece < per;
  // the tiles that were read last first: what of them is still in the caches need not come from memory again
  const unsigned block = d.first + gridDim.x - 1 - blockIdx.x;
  const long long b = block / d.tiles;
  const int tile = (int)(block - (unsigned)b * d.tiles), k0 = tile * d.tile, k1 = min(k0 + d.tile, d.S);
  const long long at = (b * d.S) * d.C + (long long)piece * VEC;
  // kAhead keys at once, the next ones on their way while these are worked on (the first ones while the levels are sorted)
  Raw<T, VEC> xs[2][kAhead], gs[2][BACK ? kAhead : 1];
  auto ask = [&](int turn, int k) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const long long o = at + (long long)(k + i * d.at_once) * d.C;
      if (on && k + i * d.at_once < k1) {
        xs[turn][i] = load_raw<T, VEC>(x + o);
        if (BACK) gs[turn][BACK ? i : 0] = load_raw<T, VEC>(dy + o);
      }
    }
  };
  ask(0, k0 + row);
  A w[VEC], bb[VEC], scale[VEC];
  if (on) channel_params<VEC>(weight, bias, piece * VEC, w, bb);
  sort_levels(level_start, d.L, d.S, s_first);
  if (!on) return;
  const int g = piece * VEC / (d.C / d.G);
  int l = -2, f1 = 0;                                        // the level of the key in hand (-1: none) and its end
  A mean = 0, rstd = 0, m1 = 0, m2 = 0;
  auto work = [&](int turn, int k) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i, k += d.at_once) {
      if (k >= k1) return;
      if (k >= f1) {
        do f1 = s_first[++l + 1];
        while (k >= f1);
        if (l >= 0) {
          const long long s = ((b * d.L + l) * d.G + g) * 2;
          mean = stats[s];
          rstd = stats[s + 1];
          if (BACK) { m1 = sums[s]; m2 = sums[s + 1]; }
        }
#pragma unroll
        for (int c = 0; c < VEC; ++c) scale[c] = rstd * w[c];
      }
      A v[VEC], dz[VEC];
      unpack<T, VEC>(xs[turn][i], v);
      if (BACK) unpack<T, VEC>(gs[turn][BACK ? i : 0], dz);
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        if (BACK) {
          const A xhat = (v[c] - mean) * rstd;
          dz[c] = through_activation<ACT>(dz[c], xhat * w[c] + bb[c]);
          v[c] = rstd * (dz[c] * w[c] - m1 - xhat * m2);
        } else {
          v[c] = activated<ACT>((v[c] - mean) * scale[c] + bb[c]);
        }
        if (l < 0) v[c] = 0;                                 // a key of no level
      }
      store_row<T, VEC, true>(out + at + (long long)k * d.C, v);
    }
  };
  const int step = kAhead * d.at_once;
  for (int k = k0 + row; k < k1; k += 2 * step) {
    ask(1, k + step);
    work(0, k);
    ask(0, k + 2 * step);
    work(1, k + step);
  }
}

// parts (B, slots, C): the sums of dz and of dz xhat over a part's keys
template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kNormBlock) void norm_grad_parts_kernel(const T *__restrict__ x, const T *__restrict__ dy, const typename Sum<T>::type *__restrict__ weight,
                                                                     const typename Sum<T>::type *__restrict__ bias, const int64_t *__restrict__ level_start,
                                                                     const typename Sum<T>::type *__restrict__ stats, typename Sum<T>::type *__restrict__ parts, NormDims d) {
  typedef typename Sum<T>::type A;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ A s_sum[kNormBlock * 2];
  sort_levels(level_start, d.L, d.S, s_first);
  const int per = d.C / VEC, row = part_of(threadIdx.x, d.per_col), piece = blockIdx.y * d.cols + threadIdx.x - row * d.cols;
  const bool on = row < d.at_once && piece < per;
  const unsigned block = d.first + blockIdx.x;
  const long long b = block / d.tiles;
  const int tile = (int)(block - (unsigned)b * d.tiles), k0 = tile * d.tile, k1 = min(k0 + d.tile, d.S);
  const int g = on ? piece * VEC / (d.C / d.G) : 0;
  A w[VEC], bb[VEC];
  channel_params<VEC>(weight, bias, on ? piece * VEC : 0, w, bb);
  const long long at = (b * d.S) * d.C + (long long)piece * VEC;
  for (int l = 0; l < d.L; ++l) {
    const int f0 = max(s_first[l], k0), f1 = min(s_first[l + 1], k1);
    if (f0 >= f1) continue;                                  // uniform
    const long long s = ((b * d.L + l) * d.G + g) * 2;
    const A mean = stats[s], rstd = stats[s + 1];
    A sum[VEC][2];
#pragma unroll
    for (int c = 0; c < VEC; ++c) sum[c][0] = sum[c][1] = 0;
    if (on) {
#pragma unroll 4
      for (int k = f0 + row; k < f1; k += d.at_once) {
        const long long o = at + (long long)k * d.C;
        A v[VEC], g_[VEC];
        load_row<T, VEC>(x + o, v);
        load_row<T, VEC>(dy + o, g_);
#pragma unroll
        for (int c = 0; c < VEC; ++c) {
          const A xhat = (v[c] - mean) * rstd;
          const A dz = through_activation<ACT>(g_[c], xhat * w[c] + bb[c]);
          sum[c][0] += dz;
          sum[c][1] += dz * xhat;
        }
      }
    }
    // the keys side by side, one channel after the other
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      for (int left = d.at_once; left > 1;) {
        const int half = (left + 1) / 2;
        s_sum[threadIdx.x * 2] = sum[c][0];
        s_sum[threadIdx.x * 2 + 1] = sum[c][1];
        __syncthreads();
        if (row + half < left) {
          sum[c][0] += s_sum[(threadIdx.x + half * d.cols) * 2];
          sum[c][1] += s_sum[(threadIdx.x + half * d.cols) * 2 + 1];
        }
        __syncthreads();
        left = half;
      }
    }
    if (row == 0 && on) {
      A *to = parts + ((b * d.slots + tile + l) * d.C + piece * VEC) * 2;
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        to[c * 2] = sum[c][0];
        to[c * 2 + 1] = sum[c][1];
      }
    }
  }
}

// Many parts of few channels' sums are added up in K ranges first: in (slots of a batch element, C, 2) -> out (B, L, K, C, 2).
template <typename In>
__global__ __launch_bounds__(kNormBlock) void norm_fold_kernel(const In *__restrict__ in, const int64_t *__restrict__ level_start, double *__restrict__ out, NormDims d, int K) {
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  sort_levels(level_start, d.L, d.S, s_first);
  const int e = blockIdx.y * kNormBlock + threadIdx.x;
  if (e >= d.C * 2) return;
  const int k = blockIdx.x % K, l = blockIdx.x / K % d.L;
  const long long b = blockIdx.x / K / d.L;
  const int f0 = s_first[l], f1 = s_first[l + 1], t0 = f0 / d.tile, tiles = f0 < f1 ? (f1 - 1) / d.tile - t0 + 1 : 0;
  const int from = t0 + (int)((long long)tiles * k / K), to = t0 + (int)((long long)tiles * (k + 1) / K);
  const In *part = in + (b * d.slots + l) * d.C * 2 + e;
  double sum = 0;
#pragma unroll 8
  for (int t = from; t < to; ++t) sum += (double)part[(long long)t * d.C * 2];
  out[(long long)blockIdx.x * d.C * 2 + e] = sum;
}

// For a batch element, a level and a group: channels (B, L, C, 2), the channels' sums over all parts, and sums (B, L, G, 2), the means of dz w and
// dz w xhat over the group.  `parts` are the tiles', or K ranges of them.  A workgroup of THREADS has as many channels side by side as there are, and as many parts
// at once as there is room for; fewer LANES than a workgroup's take all parts of a channel one after the other.  In double.
template <typename A, typename In, int LANES, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_grad_sums_kernel(const In *__restrict__ parts, const int64_t *__restrict__ level_start, const A *__restrict__ weight,
                                                                 double *__restrict__ channels, A *__restrict__ sums, NormDims d, int K) {
  constexpr bool kWhole = LANES == THREADS;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ double s_sum[kWhole ? THREADS : 1][2];
  __shared__ double s_part[THREADS / kWave];
  sort_levels(level_start, d.L, d.S, s_first);
  const int n = d.C / d.G, side = min(n, LANES), at_once = kWhole ? LANES / side : 1, lane = threadIdx.x % LANES, row = lane / side, at = lane - row * side;
  const long long units = (long long)d.B * d.L * d.G;
  for (long long turn = (long long)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES; turn < units; turn += (long long)gridDim.x * (THREADS / LANES)) {
    const long long unit = kWhole ? side_by_side(turn, units) : turn;
    const int g = (int)(unit % d.G), l = (int)(unit / d.G % d.L);
    const long long b = unit / d.G / d.L;
    const int f0 = s_first[l], f1 = s_first[l + 1], t0 = f0 / d.tile;
    const int count = f0 >= f1 ? 0 : K > 0 ? K : (f1 - 1) / d.tile - t0 + 1;
    const In *from = parts + (K > 0 ? (b * d.L + l) * K : b * d.slots + t0 + l) * d.C * 2;
    double m1 = 0, m2 = 0;
    for (int c0 = 0; c0 < n; c0 += side) {
      const int c = g * n + c0 + at;
      double s1 = 0, s2 = 0;
      if (row < at_once && c0 + at < n) {
#pragma unroll 4
        for (int t = row; t < count; t += at_once) {
          const In *part = from + ((long long)t * d.C + c) * 2;
          s1 += (double)part[0];
          s2 += (double)part[1];
        }
      }
      if constexpr (kWhole)
        for (int left = at_once; left > 1;) {
          const int half = (left + 1) / 2;
          __syncthreads();
          s_sum[threadIdx.x][0] = s1;
          s_sum[threadIdx.x][1] = s2;
          __syncthreads();
          if (row + half < left) {
            s1 += s_sum[threadIdx.x + half * side][0];
            s2 += s_sum[threadIdx.x + half * side][1];
          }
          left = half;
        }
      if (row == 0 && c0 + at < n) {
        double *to = channels + ((b * d.L + l) * d.C + c) * 2;
        to[0] = s1;
        to[1] = s2;
        const double w = weight != nullptr ? (double)weight[c] : 1.0;
        m1 += s1 * w;
        m2 += s2 * w;
      }
    }
    m1 = unit_sum<LANES>(m1, s_part);
    m2 = unit_sum<LANES>(m2, s_part);
    if (lane == 0) {
      const double all = (double)(f1 - f0) * n;
      sums[unit * 2] = f0 < f1 ? (A)(m1 / all) : (A)0;
      sums[unit * 2 + 1] = f0 < f1 ? (A)(m2 / all) : (A)0;
    }
  }
}

// Small maps: a workgroup per batch element, level and group does it all, its elements (a group's channels of a level's keys) read again from the caches for
// each of its passes: one launch for three, and backward two, or one where there is one batch element and level.
struct SmallUnit { int g, l, f0, f1; long long b, at; };
// Neighbouring groups share cache lines: they are put on one XCD (workgroups go to the eight of them in turn).
__device__ __forceinline__ SmallUnit small_unit(const NormDims &d, const int *s_first) {
  const int units = gridDim.x;
  const int unit = units % 8 == 0 ? (int)(blockIdx.x % 8) * (units / 8) + (int)(blockIdx.x / 8) : (int)blockIdx.x;
  SmallUnit u;
  u.g = unit % d.G;
  u.l = unit / d.G % d.L;
  u.b = unit / d.G / d.L;
  u.f0 = s_first[u.l];
  u.f1 = s_first[u.l + 1];
  u.at = u.b * d.S * d.C + (long long)u.g * (d.C / d.G);
  return u;
}
// keys of no level
template <typename T, int VEC, int THREADS>
__device__ __forceinline__ void small_zeros(T *__restrict__ out, const SmallUnit &u, const NormDims &d, int first, int pieces) {
  typename Sum<T>::type zero[VEC] = {};
  if (u.l == 0)
    for (int k = threadIdx.x; k < first * pieces; k += THREADS) store_row<T, VEC>(out + u.at + (long long)(k / pieces) * d.C + k % pieces * VEC, zero);
}

constexpr int kHeld = 4;               // keys that a thread holds in registers from the first pass to the last, where those are all

template <typename T, int VEC, int ACT, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_small_kernel(const T *__restrict__ x, const typename Sum<T>::type *__restrict__ weight,
                                                             const typename Sum<T>::type *__restrict__ bias, const int64_t *__restrict__ level_start,
                                                             typename Sum<T>::type *__restrict__ stats, T *__restrict__ y, NormDims d, double eps) {
  typedef typename Sum<T>::type A;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ double s_part[THREADS / kWave];
  sort_levels(level_start, d.L, d.S, s_first);
  const SmallUnit u = small_unit(d, s_first);
  const int n = d.C / d.G, pieces = n / VEC, at_once = THREADS / pieces, row = threadIdx.x / pieces, piece = threadIdx.x - row * pieces;
  const bool on = row < at_once, held = u.f1 - u.f0 <= kHeld * at_once;       // (held: uniform)
  const T *from = x + u.at + piece * VEC;
  const double count = (double)(u.f1 - u.f0) * n;
  A v[kHeld][VEC], w[VEC], bb[VEC];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) {
    const int k = u.f0 + row + i * at_once;
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[i][c] = 0;
    if (on && k < u.f1) load_row<T, VEC>(from + (long long)k * d.C, v[i]);
  }
  channel_params<VEC>(weight, bias, u.g * n + piece % pieces * VEC, w, bb);
  small_zeros<T, VEC, THREADS>(y, u, d, s_first[0], pieces);
  // a pass for the mean, one for the squares about it
  A mean = 0, rstd = 0;
  for (int pass = 0; pass < 2; ++pass) {
    A sum = 0;
    auto add = [&](const A (&v)[VEC]) {
      A some = 0;
#pragma unroll
      for (int c = 0; c < VEC; ++c) some += pass == 0 ? v[c] : (v[c] - mean) * (v[c] - mean);
      sum += some;
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (on && u.f0 + row + i * at_once < u.f1) add(v[i]);
    if (on && !held)
#pragma unroll 4
      for (int k = u.f0 + row + kHeld * at_once; k < u.f1; k += at_once) {
        A more[VEC];
        load_row<T, VEC>(from + (long long)k * d.C, more);
        add(more);
      }
    const double all = block_sum<THREADS>((double)sum, s_part);
    if (u.f0 < u.f1) {
      if (pass == 0) mean = (A)(all / count);
      else rstd = (A)(1.0 / sqrt(all / count + eps));
    }
  }
  if (threadIdx.x == 0) {
    A *to = stats + ((u.b * d.L + u.l) * d.G + u.g) * 2;
    to[0] = mean;
    to[1] = rstd;
  }
  if (!on) return;
  auto finish = [&](A (&v)[VEC], int k) {
#pragma unroll
    for (int c = 0; c < VEC; ++c) v[c] = activated<ACT>((v[c] - mean) * rstd * w[c] + bb[c]);
    store_row<T, VEC>(y + u.at + piece * VEC + (long long)k * d.C, v);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (u.f0 + row + i * at_once < u.f1) finish(v[i], u.f0 + row + i * at_once);
  if (!held)
#pragma unroll 4
    for (int k = u.f0 + row + kHeld * at_once; k < u.f1; k += at_once) {
      A more[VEC];
      load_row<T, VEC>(from + (long long)k * d.C, more);
      finish(more, k);
    }
}

template <typename T, int VEC, int ACT>
__global__ __launch_bounds__(kSmallBlock) void norm_small_grad_kernel(const T *__restrict__ x, const T *__restrict__ dy, const typename Sum<T>::type *__restrict__ weight,
                                                                      const typename Sum<T>::type *__restrict__ bias, const int64_t *__restrict__ level_start,
                                                                      const typename Sum<T>::type *__restrict__ stats, double *__restrict__ channels,
                                                                      typename Sum<T>::type *__restrict__ grad_weight, typename Sum<T>::type *__restrict__ grad_bias,
                                                                      T *__restrict__ dx, NormDims d) {
  typedef typename Sum<T>::type A;
  __shared__ int s_first[DFA3D_MAX_LEVELS + 1];
  __shared__ double s_part[kSmallBlock / kWave];
  __shared__ double s_sum[kSmallBlock][2];
  sort_levels(level_start, d.L, d.S, s_first);
  const SmallUnit u = small_unit(d, s_first);
  const int n = d.C / d.G, pieces = n / VEC, at_once = kSmallBlock / pieces, row = threadIdx.x / pieces, piece = threadIdx.x - row * pieces;
  const bool on = row < at_once;
  const long long at = u.at + piece * VEC;
  const A mean = stats[((u.b * d.L + u.l) * d.G + u.g) * 2], rstd = stats[((u.b * d.L + u.l) * d.G + u.g) * 2 + 1];
  A w[VEC], bb[VEC], sum[VEC][2];
  channel_params<VEC>(weight, bias, u.g * n + piece * VEC, w, bb);
#pragma unroll
  for (int c = 0; c < VEC; ++c) sum[c][0] = sum[c][1] = 0;
  if (on)
#pragma unroll 4
    for (int k = u.f0 + row; k < u.f1; k += at_once) {
      A v[VEC], g[VEC];
      load_row<T, VEC>(x + at + (long long)k * d.C, v);
      load_row<T, VEC>(dy + at + (long long)k * d.C, g);
#pragma unroll
      for (int c = 0; c < VEC; ++c) {
        const A xhat = (v[c] - mean) * rstd, dz = through_activation<ACT>(g[c], xhat * w[c] + bb[c]);
        sum[c][0] += dz;
        sum[c][1] += dz * xhat;
      }
    }
  double m1 = 0, m2 = 0;
#pragma unroll
  for (int c = 0; c < VEC; ++c) {
    double s1 = sum[c][0], s2 = sum[c][1];
    m1 += s1 * (double)w[c];
    m2 += s2 * (double)w[c];
    if (channels != nullptr || grad_weight != nullptr || grad_bias != nullptr) {         // the keys side by side, one channel after the other
      for (int left = at_once; left > 1;) {
        const int half = (left + 1) / 2;
        __syncthreads();
        s_sum[threadIdx.x][0] = s1;
        s_sum[threadIdx.x][1] = s2;
        __syncthreads();
        if (row + half < left) {
          s1 += s_sum[threadIdx.x + half * pieces][0];
          s2 += s_sum[threadIdx.x + half * pieces][1];
        }
        left = half;
      }
      if (row == 0 && on) {
        const int channel = u.g * n + piece * VEC + c;
        if (channels != nullptr) {
          double *to = channels + ((u.b * d.L + u.l) * d.C + channel) * 2;
          to[0] = s1;
          to[1] = s2;
        } else {                                             // there is one batch element and level
          if (grad_bias != nullptr) grad_bias[channel] = (A)s1;
          if (grad_weight != nullptr) grad_weight[channel] = (A)s2;
        }
      }
    }
  }
  if (dx == nullptr) return;                                 // uniform
  m1 = block_sum<kSmallBlock>(m1, s_part);
  m2 = block_sum<kSmallBlock>(m2, s_part);
  small_zeros<T, VEC, kSmallBlock>(dx, u, d, s_first[0], pieces);
  if (!on || u.f0 >= u.f1) return;
  const double count = (double)(u.f1 - u.f0) * n;
  const A a1 = (A)(m1 / count), a2 = (A)(m2 / count);
#pragma unroll 4
  for (int k = u.f0 + row; k < u.f1; k += at_once) {
    A v[VEC], g[VEC];
    load_row<T, VEC>(x + at + (long long)k * d.C, v);
    load_row<T, VEC>(dy + at + (long long)k * d.C, g);
#pragma unroll
    for (int c = 0; c < VEC; ++c) {
      const A xhat = (v[c] - mean) * rstd, dz = through_activation<ACT>(g[c], xhat * w[c] + bb[c]);
      v[c] = rstd * (dz * w[c] - a1 - xhat * a2);
    }
    store_row<T, VEC>(dx + at + (long long)k * d.C, v);
  }
}

template <typename A> __global__ __launch_bounds__(kNormBlock) void norm_grad_params_kernel(ParamGrads p) {
  param_grads<A>(p, blockIdx.x * kNormBlock + threadIdx.x);
}

// ---------------------------------------------------------------------------------------------------------------------------------------------

// Whether a workgroup per batch element, level and group does it all.  (The pieces of a key stand side by side in it.)
static bool is_small(const NormArgs &a, int vec, bool back) {
  const long long n = a.C / a.G;
  return n / vec <= kSmallBlock && a.S * n <= kSmallElements[back] && (long long)a.B * a.S * a.C <= kSmallTotal && (long long)a.B * a.L * a.G <= kSmallUnits[back];
}
// Keys of a tile that a thread of the results takes, of 16 bytes a piece.  (6 x 30825 x 256, training in float: 8 254.7 us, 16 257.5; inference with silu in
// bfloat16: 72.4, 67.6.)
static int most_apply_keys(int elem_size) { return elem_size == 2 ? 16 : 8; }
// Keys of a tile that a thread of the statistics keeps in registers: 32 elements.  (6 x 30825 x 256 in bfloat16, 8 to a piece: 8 keys 24.1 us, 4 21.8; in float,
// 4 to a piece: 8 keys 34.5, 4 34.4, and their parts' sums 6.7 and 9.9.)
constexpr int norm_keys(int vec) { return vec == 8 ? 4 : 8; }
constexpr int kGradKeys = 32;          // keys of a tile that a thread of the gradients' sums takes

// keys of a tile that a thread of the gradients' sums takes: many, for few parts to be written and read, while that leaves two workgroups a CU
static int keys_for(const NormArgs &a, int vec, int keys, int least, int workgroups) {
  const int at_once = kNormBlock / std::min(a.C / vec, kNormBlock);
  while (keys > least && (long long)a.B * ((a.S + at_once * keys - 1) / (at_once * keys)) < workgroups) keys /= 2;
  return keys;
}
static int grad_keys(const NormArgs &a, int vec) { return keys_for(a, vec, kGradKeys, 4, 512); }
static int apply_keys(const NormArgs &a, int vec, int elem_size) { return keys_for(a, vec, most_apply_keys(elem_size), 2, 1024); }
static NormDims norm_dims(const NormArgs &a, int vec, int per_thread) {
  NormDims d{};
  d.B = a.B; d.S = a.S; d.C = a.C; d.G = a.G; d.L = a.L;
  const int per = a.C / vec;
  d.cols = std::min(per, kNormBlock);
  d.at_once = kNormBlock / d.cols;
  d.per_col = 1.0f / d.cols;
  d.tile = d.at_once * per_thread;
  d.tiles = (int)(((long long)a.S + d.tile - 1) / d.tile);
  d.slots = d.tiles + a.L - 1;
  return d;
}
// the same for the statistics' parts: whole groups side by side
static NormDims parts_dims(const NormArgs &a, int vec) {
  NormDims d = norm_dims(a, vec, 1);
  d.group = a.C / a.G / vec;
  d.per_piece = 1.0f / d.group;
  d.blocks = (d.group + kNormBlock - 1) / kNormBlock;
  d.cells = a.G * d.blocks;
  d.abreast = d.blocks > 1 ? 1 : std::min(a.G, kNormBlock / d.group);
  d.cols = d.blocks > 1 ? kNormBlock : d.abreast * d.group;
  d.per_col = 1.0f / d.cols;
  d.at_once = kNormBlock / d.cols;
  d.tile = d.at_once * norm_keys(vec);
  d.tiles = (int)(((long long)a.S + d.tile - 1) / d.tile);
  d.slots = d.tiles + a.L - 1;
  return d;
}
static unsigned most_blocks(long long blocks) { return (unsigned)std::min(blocks, 1LL << 20); }
// launch(d, grid) for all tiles of all batch elements, `columns` workgroups each: in turns, as a grid holds fewer than 2^32 threads.
constexpr long long kTurn = 1 << 23;
template <typename F> static hipError_t in_turns(NormDims d, int columns, F launch) {
  const long long all = (long long)d.B * d.tiles;
  for (long long first = 0; first < all; first += kTurn) {
    d.first = (unsigned)first;
    launch(d, dim3((unsigned)std::min(kTurn, all - first), columns));
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}
static int parts_columns(const NormDims &d) { return (d.cells + d.abreast - 1) / d.abreast; }
static int norm_columns(const NormDims &d, int vec) { return (d.C / vec + d.cols - 1) / d.cols; }

constexpr int kSerialParts = 8;
// Ranges in which the gradients' parts are added up first, for few groups of many of them; 0: not.  (One after the other, and in
// ranges, the sums on the device: 131072 x 256 of 32 groups, 32 turns of a workgroup, 7.8 us and 10.1, 262144, 64 turns, 11.0 and 12.1, 20000 x 64 of one group, 40 turns,
// 12.9 and 8.0, 16000 x 256 of one group 86 and 12, 4000 x 1024 386 and 14.)
static int fold_ranges(const NormDims &d) {
  const int n = d.C / d.G, side = std::min(n, kNormBlock);
  const long long at_once = kNormBlock / side, turns = (d.tiles + at_once - 1) / at_once * ((n + side - 1) / side);
  if (turns <= 32 || (long long)d.B * d.L * d.G > 4096) return 0;
  int K = 1;
  while (K < 256 && (long long)K * K * ((n + side - 1) / side) < d.tiles) ++K;
  return K;
}
// Ranges in which the channels' sums of many batch elements and levels are added up first; 0: not.  (They are added up while the
// results are formed.  Backward of B x S x 256, on the device: 250 x 200 at once 54 us, in ranges first 57, 1000 x 50 88 and 56.)
static int param_rows(const NormArgs &a) {
  const long long BL = (long long)a.B * a.L;
  if (BL <= 256) return 0;
  int K = 8;
  while (K < 256 && (long long)K * K < BL) ++K;
  return K;
}
// the channels' sums as parts of one batch element and level
static NormDims channel_dims(const NormArgs &a) {
  NormDims d{};
  d.B = d.L = d.G = 1;
  d.S = d.slots = d.tiles = a.B * a.L;
  d.C = a.C;
  d.tile = 1;
  return d;
}
static size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
static size_t norm_parts_bytes(const NormArgs &a, int vec, size_t elem) {
  const NormDims d = parts_dims(a, vec);
  return (size_t)d.B * d.slots * d.cells * 2 * elem;
}
static size_t grad_parts_bytes(const NormArgs &a, int vec, size_t elem) {
  const NormDims d = norm_dims(a, vec, grad_keys(a, vec));
  return rounded((size_t)d.B * d.slots * a.C * 2 * elem);
}
size_t norm_workspace_bytes(const NormArgs &a, int dtype, bool back) {
  // (whatever the operands' alignment turns out to be)
  const size_t elem = dtype == DFA3D_F64 ? 8 : 4;
  size_t most = 0;
  for (int vec = 1; vec <= 8; vec *= 2)
    if (a.C / a.G % vec == 0) most = std::max(most, back ? grad_parts_bytes(a, vec, elem) : norm_parts_bytes(a, vec, elem));
  if (!back) return most;
  size_t ranges = (size_t)param_rows(a);
  for (int vec = 1; vec <= 8; vec *= 2)
    if (a.C / a.G % vec == 0) ranges = std::max(ranges, (size_t)a.B * a.L * fold_ranges(norm_dims(a, vec, grad_keys(a, vec))));
  return most + rounded((size_t)a.B * a.L * a.C * 2 * sizeof(double)) + rounded((size_t)a.B * a.L * a.G * 2 * elem) + ranges * a.C * 2 * sizeof(double);
}

template <typename T, int VEC, int ACT>
static hipError_t norm_forward(const NormArgs &a, hipStream_t stream) {
  typedef typename Sum<T>::type A;
  const NormDims d = parts_dims(a, VEC);
  if (is_small(a, VEC, false)) {
    auto launch = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, dim3(d.B * d.L * d.G), dim3(threads), 0, stream, (const T *)a.x, (const A *)a.weight, (const A *)a.bias, a.level_start, (A *)a.stats,
                         (T *)a.y, d, a.eps);
      return hipGetLastError();
    };
    // four wavefronts where they hold all of a group
    const int pieces = a.C / a.G / VEC;
    return pieces <= kNormBlock && a.S <= kHeld * (kNormBlock / pieces) ? launch(norm_small_kernel<T, VEC, ACT, kNormBlock>, kNormBlock)
                                                                       : launch(norm_small_kernel<T, VEC, ACT, kSmallBlock>, kSmallBlock);
  }
  const NormDims k = norm_dims(a, VEC, apply_keys(a, VEC, (int)sizeof(T)));
  auto parts = [&](const NormDims &d, dim3 grid) {
    hipLaunchKernelGGL((norm_parts_kernel<T, VEC, norm_keys(VEC)>), grid, dim3(kNormBlock), 0, stream, (const T *)a.x, a.level_start, (A *)a.workspace, d);
  };
  if (hipError_t e = in_turns(d, parts_columns(d), parts)) return e;
  const long long units = (long long)d.B * d.L * d.G;
  const int lanes = unit_lanes(units, (long long)d.tiles * d.blocks, kHeldParts);
  auto stats = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(most_blocks((units * lanes + kNormBlock - 1) / kNormBlock)), dim3(kNormBlock), 0, stream, (const A *)a.workspace, a.level_start,
                       (A *)a.stats, d, VEC, a.eps);
    return hipGetLastError();
  };
  if (hipError_t e = lanes == 4 ? stats(norm_stats_kernel<A, 4>) : lanes == 16 ? stats(norm_stats_kernel<A, 16>) : lanes == 64 ? stats(norm_stats_kernel<A, 64>)
                                                                                                        : stats(norm_stats_kernel<A, kNormBlock>)) return e;
  return in_turns(k, norm_columns(k, VEC), [&](const NormDims &k, dim3 grid) {
    hipLaunchKernelGGL((norm_apply_kernel<T, VEC, ACT, false>), grid, dim3(kNormBlock), 0, stream, (const T *)a.x, (const T *)nullptr, (const A *)a.weight, (const A *)a.bias,
                       a.level_start, (const A *)a.stats, (const A *)nullptr, (T *)a.y, k, ParamGrads{});
  });
}
template <typename T, int VEC, int ACT>
static hipError_t norm_backward(const NormArgs &a, hipStream_t stream) {
  typedef typename Sum<T>::type A;
  const NormDims d = norm_dims(a, VEC, grad_keys(a, VEC)), k = norm_dims(a, VEC, apply_keys(a, VEC, (int)sizeof(T)));
  A *parts = (A *)a.workspace;
  double *channels = (double *)((char *)a.workspace + grad_parts_bytes(a, VEC, sizeof(A)));
  A *sums = (A *)((char *)channels + rounded((size_t)a.B * a.L * a.C * 2 * sizeof(double)));
  double *folded = (double *)((char *)sums + rounded((size_t)a.B * a.L * a.G * 2 * sizeof(A)));
  const bool of_params = a.grad_weight != nullptr || a.grad_bias != nullptr, small = is_small(a, VEC, true);
  if (small) {
    const bool one = a.B * a.L == 1;
    hipLaunchKernelGGL((norm_small_grad_kernel<T, VEC, ACT>), dim3(d.B * d.L * d.G), dim3(kSmallBlock), 0, stream, (const T *)a.x, (const T *)a.grad_y, (const A *)a.weight,
                       (const A *)a.bias, a.level_start, (const A *)a.stats, of_params && !one ? channels : nullptr, one ? (A *)a.grad_weight : nullptr,
                       one ? (A *)a.grad_bias : nullptr, (T *)a.grad_x, d);
    if (one) return hipGetLastError();
  } else {
    auto grad_parts = [&](const NormDims &d, dim3 grid) {
      hipLaunchKernelGGL((norm_grad_parts_kernel<T, VEC, ACT>), grid, dim3(kNormBlock), 0, stream, (const T *)a.x, (const T *)a.grad_y, (const A *)a.weight, (const A *)a.bias,
                         a.level_start, (const A *)a.stats, parts, d);
    };
    if (hipError_t e = in_turns(d, norm_columns(d, VEC), grad_parts)) return e;
    const int K = fold_ranges(d);
    if (K > 0) {
      hipLaunchKernelGGL((norm_fold_kernel<A>), dim3((unsigned)(d.B * d.L * K), (d.C * 2 + kNormBlock - 1) / kNormBlock), dim3(kNormBlock), 0, stream, parts, a.level_start,
                         folded, d, K);
      if (hipError_t e = hipGetLastError()) return e;
    }
    const long long units = (long long)d.B * d.L * d.G;
    const int n = d.C / d.G, lanes = d.tiles <= kSerialParts ? unit_lanes(units, n, 1) : kNormBlock;
    auto launch = [&](auto kernel, const auto *in, int threads) {
      hipLaunchKernelGGL(kernel, dim3(most_blocks((units * std::min(lanes, threads) + threads - 1) / threads)), dim3(threads), 0, stream, in, a.level_start,
                         (const A *)a.weight, channels, sums, d, K);
    };
    if (K > 0 && n > kNormBlock) {
      hipLaunchKernelGGL((norm_grad_sums_kernel<A, double, kSmallBlock, kSmallBlock>), dim3(most_blocks(units)), dim3(kSmallBlock), 0, stream, folded, a.level_start,
                         (const A *)a.weight, channels, sums, d, K);
    } else if (K > 0) {
      launch(norm_grad_sums_kernel<A, double, kNormBlock, kNormBlock>, folded, kNormBlock);
    } else if (lanes == kNormBlock) {
      launch(norm_grad_sums_kernel<A, A, kNormBlock, kNormBlock>, parts, kNormBlock);
    } else if (lanes == 64) {
      launch(norm_grad_sums_kernel<A, A, 64, kNormBlock>, parts, kNormBlock);
    } else if (lanes == 16) {
      launch(norm_grad_sums_kernel<A, A, 16, kNormBlock>, parts, kNormBlock);
    } else {
      launch(norm_grad_sums_kernel<A, A, 4, kNormBlock>, parts, kNormBlock);
    }
  }
  if (hipError_t e = hipGetLastError()) return e;
  const int rows = of_params ? param_rows(a) : 0;
  if (rows > 0) {
    const NormDims all = channel_dims(a);
    hipLaunchKernelGGL((norm_fold_kernel<double>), dim3(rows, (d.C * 2 + kNormBlock - 1) / kNormBlock), dim3(kNormBlock), 0, stream, channels, (const int64_t *)nullptr, folded, all,
                       rows);
    if (hipError_t e = hipGetLastError()) return e;
  }
  ParamGrads params = {rows > 0 ? folded : channels, a.grad_weight, a.grad_bias, rows > 0 ? rows : d.B * d.L, d.C, of_params ? (d.C + kNormBlock - 1) / kNormBlock : 0};
  if (of_params && (small || a.grad_x == nullptr)) {
    hipLaunchKernelGGL((norm_grad_params_kernel<A>), dim3(params.blocks), dim3(kNormBlock), 0, stream, params);
    return hipGetLastError();
  }
  if (small || a.grad_x == nullptr) return hipSuccess;
  return in_turns(k, norm_columns(k, VEC), [&](const NormDims &k, dim3 grid) {
    grid.x += params.blocks;
    hipLaunchKernelGGL((norm_apply_kernel<T, VEC, ACT, true>), grid, dim3(kNormBlock), 0, stream, (const T *)a.x, (const T *)a.grad_y, (const A *)a.weight, (const A *)a.bias,
                       a.level_start, (const A *)a.stats, sums, (T *)a.grad_x, k, params);
    params.blocks = 0;                                       // (formed)
  });
}

template <typename T, int VEC>
static hipError_t norm_act(const NormArgs &a, bool back, hipStream_t stream) {
  switch (a.act) {
    case DFA3D_ACT_NONE: return back ? norm_backward<T, VEC, DFA3D_ACT_NONE>(a, stream) : norm_forward<T, VEC, DFA3D_ACT_NONE>(a, stream);
    case DFA3D_ACT_RELU: return back ? norm_backward<T, VEC, DFA3D_ACT_RELU>(a, stream) : norm_forward<T, VEC, DFA3D_ACT_RELU>(a, stream);
    case DFA3D_ACT_SILU: return back ? norm_backward<T, VEC, DFA3D_ACT_SILU>(a, stream) : norm_forward<T, VEC, DFA3D_ACT_SILU>(a, stream);
  }
  return hipErrorInvalidValue;
}
// pieces of one group's channels
template <typename T>
static hipError_t norm_typed(const NormArgs &a, bool back, hipStream_t stream) {
  const int vec = row_vec(a.C / a.G, (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.grad_y | (uintptr_t)a.grad_x, sizeof(T));
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return norm_act<T, 8>(a, back, stream);
  if constexpr (sizeof(T) <= 4)
    if (vec == 4) return norm_act<T, 4>(a, back, stream);
  return vec == 2 ? norm_act<T, 2>(a, back, stream) : norm_act<T, 1>(a, back, stream);
}
static hipError_t norm_any(const NormArgs &a, int dtype, bool back, hipStream_t stream) {
  if (dtype == DFA3D_F32) return norm_typed<float>(a, back, stream);
  if (dtype == DFA3D_F64) return norm_typed<double>(a, back, stream);
  if (dtype == DFA3D_BF16) return norm_typed<__hip_bfloat16>(a, back, stream);
  return hipErrorInvalidValue;
}
hipError_t launch_norm(const NormArgs &a, int dtype, hipStream_t stream) { return norm_any(a, dtype, false, stream); }
hipError_t launch_norm_grad(const NormArgs &a, int dtype, hipStream_t stream) { return norm_any(a, dtype, true, stream); }

}  // namespace dfa3d
