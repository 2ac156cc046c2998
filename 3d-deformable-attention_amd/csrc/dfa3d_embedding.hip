// Rows looked up in a learned table, scaled and summed, for gfx950:
//
//   out[r, n, :] = plus[r, n, :] + mul * sum over h of scale[r, n, h] * table[index[n], h, :]
//
// and its gradients.  index lists N places (N entries of a camera's list, N tokens), shared by R batch elements; the table holds V entries of H
// rows of E elements.  A place outside [0, V) (the padding of a list) adds nothing and has no gradient.
//
//   embedding_kernel         the sum
//   embedding_scale_kernel   grad_scale[r, n, h] = mul * <table[index[n], h], g[r, n]>
//   embedding_order_kernel   the places of every entry, in ascending order, in one launch
//   embedding_digits_kernel, embedding_tiles_kernel, embedding_sort_kernel, embedding_starts_kernel
//                            the same for more places or a larger table, sorted by digits
//   embedding_table_kernel   grad_table[v, h, :] = mul * sum over those and r of scale[r, n, h] g[r, n, :], in that order: no atomics, the same result
//   embedding_join_kernel    every time; entries with very many places are summed in pieces that the last kernel joins
//
// All of them stream rows: bound by memory.
#include <algorithm>

#include "../../include/dfa3d.h"
#include "dfa3d_launch.h"
#include "dfa3d_rows.h"

namespace dfa3d {

constexpr int kEmbBlock = 256;

// the place's entry, or -1
template <typename I> __device__ __forceinline__ int entry_of(const I *__restrict__ index, long long n, int V) {
  const I v = index[n];
  return v >= 0 && v < (I)V ? (int)v : -1;
}

// One thread per VEC elements of a row of out.
template <typename T, typename I, int VEC>
__global__ __launch_bounds__(kEmbBlock) void embedding_kernel(const T *__restrict__ table, const I *__restrict__ index,
                                                              const typename Sum<T>::type *__restrict__ scale, const T *__restrict__ plus, T *__restrict__ out,
                                                              long long rows, Pieces places, int V, int H, int E, typename Sum<T>::type mul, Pieces pieces) {
  typedef typename Sum<T>::type A;
  const long long total = rows * pieces.per;
  for (long long t = (long long)blockIdx.x * kEmbBlock + threadIdx.x; t < total; t += (long long)gridDim.x * kEmbBlock) {
    long long row;
    int piece;
    pieces.place(t, row, piece);
    const int e = piece * VEC;
    long long r;
    int n;
    places.place(row, r, n);
    const int v = entry_of(index, n, V);
    A sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0;
    if (v >= 0) {
      const T *from = table + (long long)v * H * E + e;
#pragma unroll 8
      for (int h = 0; h < H; ++h) {
        A r[VEC];
        load_row<T, VEC>(from + (long long)h * E, r);
        const A s = scale != nullptr ? scale[row * H + h] : (A)1;
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += s * r[i];
      }
    }
    if (plus != nullptr) {
      A add[VEC];
      load_row<T, VEC>(plus + row * E + e, add);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] = v >= 0 ? add[i] + mul * sum[i] : add[i];
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] = v >= 0 ? mul * sum[i] : (A)0;
    }
    store_row<T, VEC, true>(out + row * E + e, sum);
  }
}

// A wavefront per row: a lane's share of each head's product, then the lanes' sum.
template <typename T, typename I, int VEC>
__global__ __launch_bounds__(kEmbBlock) void embedding_scale_kernel(const T *__restrict__ table, const I *__restrict__ index, const T *__restrict__ grad,
                                                                    typename Sum<T>::type *__restrict__ grad_scale, long long rows, Pieces places, int V, int H,
                                                                    int E, typename Sum<T>::type mul) {
  typedef typename Sum<T>::type A;
  const int lane = threadIdx.x % kWave;
  const long long waves = (long long)gridDim.x * (kEmbBlock / kWave);
  for (long long row = (long long)blockIdx.x * (kEmbBlock / kWave) + threadIdx.x / kWave; row < rows; row += waves) {
    long long r;
    int n;
    places.place(row, r, n);
    const int v = entry_of(index, n, V);                     // uniform
    for (int h0 = 0; h0 < H; h0 += 8) {
      A dot[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) dot[h] = 0;
      if (v >= 0)
        for (int e = lane * VEC; e < E; e += kWave * VEC) {
          A g[VEC];
          load_row<T, VEC>(grad + row * E + e, g);
#pragma unroll
          for (int h = 0; h < 8; ++h) {
            A r[VEC];
            load_row<T, VEC>(table + ((long long)v * H + min(h0 + h, H - 1)) * E + e, r);
#pragma unroll
            for (int i = 0; i < VEC; ++i) dot[h] += g[i] * r[i];
          }
        }
#pragma unroll
      for (int h = 0; h < 8; ++h) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) dot[h] += __shfl_xor(dot[h], off, kWave);
        if (lane == 0 && h0 + h < H) grad_scale[row * H + h0 + h] = v >= 0 ? mul * dot[h] : (A)0;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------
// Places are numbered on beyond the index where its batch elements are places of their own (spread_over): place n has the index of place n % period.
// The places of every entry, in ascending order: order (N), and where each entry's begin in it, starts (V + 1).  Entries of more than `chunk` places are
// listed, in any order (many).
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <bool SPREAD> __device__ __forceinline__ uint32_t in_index(long long n, int period) { return SPREAD ? (uint32_t)n % (uint32_t)period : (uint32_t)n; }
struct Many { int entry, from, to; };  // an entry of many places, and which they are

// Where 64 keys, a lane's each, go if equal ones keep their order: `count` says where the next one of a key goes, and is moved on.  Lanes with the same key find
// each other by a vote on each of the keys' `bits`.
__device__ __forceinline__ int next_place(uint32_t key, bool on, int bits, int *count) {
  const int lane = threadIdx.x % kWave;
  unsigned long long same = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const bool set = (key >> b & 1) != 0;
    const unsigned long long those = __ballot(set);
    same &= set ? those : ~those;
  }
  const int leader = on ? __ffsll(same) - 1 : 0;
  int at = 0;
  if (on && lane == leader) at = atomicAdd(&count[key], __popcll(same));
  return __shfl(at, leader, kWave) + __popcll(same & ((1ull << lane) - 1));
}

// Not too many places, in a table that is not too large: one launch.  A workgroup keeps the entries [first, first + per); each of its wavefronts reads a share
// of the index, counts what is the workgroup's, and what belongs before it (which says where the workgroup's begin: no workgroup waits for another), and
// keeps those places in LDS; once the counts say where each entry's and each wavefront's go, it writes them there, or, where they were too many to keep,
// reads its share again.  A wavefront's places of one entry ascend, and so do the wavefronts' shares.
//   Every workgroup reads the whole index, from the second-level caches, so that a place costs as many instructions as there are workgroups: as many of those as
// there are CUs do best.  49200 places of 40000 entries: 512 workgroups, one place at a time, twice 46 us, 256, four at a time, twice 18, and once 12.
constexpr int kOrderWaves = 16, kOrderBlock = kOrderWaves * kWave;
constexpr int kOrderGroups = 256, kXcds = 8;
constexpr int kOrderPer = 512;         // (32 KB of counts)
constexpr int kOrderAhead = 8;         // places of a lane asked for at once
constexpr int kOrderLds = 60 << 10;    // for the counts, and for the places that the wavefronts keep from their first reading for the second: 256 to 576 each

// A place as it stands in the index, in 32 bits: what lies outside the table comes out as no entry of it and not before any.
template <bool SPREAD, typename I> __device__ __forceinline__ uint32_t raw_entry(const I *__restrict__ index, long long n, int period) {
  const I v = index[in_index<SPREAD>(n, period)];
  if constexpr (sizeof(I) == 4) return (uint32_t)v;
  else return (uint32_t)((uint64_t)v >> 32) != 0 ? 0xFFFFFFFFu : (uint32_t)v;
}

template <typename I, bool SPREAD>
__global__ __launch_bounds__(kOrderBlock) void embedding_order_kernel(const I *__restrict__ index, int *__restrict__ order, int *__restrict__ starts,
                                                                      Many *__restrict__ many, int *__restrict__ many_count, int N, int period, int V, int per, int bits, int keep, int chunk,
                                                                      uint32_t *__restrict__ grad_scale, long long R, int words) {
  extern __shared__ int s_count[];     // (kOrderWaves, per): how many of an entry a wavefront has, then where its next one goes
  int *const s_place = s_count + kOrderWaves * per;                          // (kOrderWaves, keep): the places kept, and their entries
  uint16_t *const s_entry = (uint16_t *)(s_place + kOrderWaves * keep);
  __shared__ int s_before[kOrderWaves], s_all[kOrderWaves], s_many;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t first = blockIdx.x * per, mine = min((uint32_t)per, V - first);
  const int share = (int)((((long long)N + kOrderWaves - 1) / kOrderWaves + kWave - 1) / kWave * kWave);
  const long long n0 = (long long)wave * share, n1 = min(n0 + share, (long long)N);
  for (int k = threadIdx.x; k < kOrderWaves * per; k += kOrderBlock) s_count[k] = 0;
  if (threadIdx.x == 0) s_many = 0;
  __syncthreads();
  int *const count = s_count + wave * per;
  // Each line of the index is asked for once in each second-level cache before all of its workgroups want it at once: an index that comes from memory, 40000 places
  // of 64 bits, 18.8 -> 12.2 us; 49200 of 32 13.2 -> 12.3.
  constexpr int kLine = 128 / sizeof(I);
  const int nth = blockIdx.x / kXcds, of = (gridDim.x + kXcds - 1) / kXcds;
  I touched = 0;
  for (long long n = ((long long)threadIdx.x * of + nth) * kLine; n < period; n += (long long)of * kOrderBlock * kLine) touched ^= index[n];
  int before = 0, kept = 0;            // (kept: uniform)
  for (long long n = n0; n < n1; n += kOrderAhead * kWave) {
    uint32_t v[kOrderAhead];
#pragma unroll
    for (int a = 0; a < kOrderAhead; ++a) {
      const long long at = n + a * kWave + lane;
      v[a] = at < n1 ? raw_entry<SPREAD>(index, at, period) : 0xFFFFFFFFu;
    }
#pragma unroll
    for (int a = 0; a < kOrderAhead; ++a) {
      before += v[a] < first;
      v[a] -= first;
      const unsigned long long on = __ballot(v[a] < mine);
      if (on == 0) continue;                                 // uniform
      const int at = kept + __popcll(on & ((1ull << lane) - 1));
      kept += __popcll(on);
      if (v[a] < mine) {
        atomicAdd(&count[v[a]], 1);
        if (at < keep) {
          s_place[wave * keep + at] = (int)(n + a * kWave + lane);
          s_entry[wave * keep + at] = (uint16_t)v[a];
        }
      }
    }
  }
  asm volatile("" : : "v"(touched));                         // (and no earlier)
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) before += __shfl_xor(before, off, kWave);
  if (lane == 0) s_before[wave] = before;
  __syncthreads();
  // where each wavefront's places of each entry begin: entries in order, an entry's wavefronts in order
  int base = 0;
  for (int w = 0; w < kOrderWaves; ++w) base += s_before[w];
  for (uint32_t k0 = 0; k0 < mine; k0 += kOrderBlock) {
    const uint32_t k = k0 + threadIdx.x;
    int all = 0;
    if (k < mine)
      for (int w = 0; w < kOrderWaves; ++w) all += s_count[w * per + k];
    int upto = all;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int u = __shfl_up(upto, off, kWave);
      if (lane >= off) upto += u;
    }
    if (lane == kWave - 1) s_all[wave] = upto;
    __syncthreads();
    int at = base + upto - all;
    for (int w = 0; w < wave; ++w) at += s_all[w];
    if (k < mine) {
      starts[first + k] = at;
      if (first + k == (uint32_t)V - 1) starts[V] = at + all;
      if (all > chunk) many[first + atomicAdd(&s_many, 1)] = Many{(int)(first + k), at, at + all};
      for (int w = 0; w < kOrderWaves; ++w) {
        const int c = s_count[w * per + k];
        s_count[w * per + k] = at;
        at += c;
      }
    }
    for (int w = 0; w < kOrderWaves; ++w) base += s_all[w];
    __syncthreads();
  }
  if (threadIdx.x == 0) many_count[blockIdx.x] = s_many;
  if (kept <= keep) {                                        // uniform
    for (int i = 0; i < kept; i += kWave) {
      const bool on = i + lane < kept;
      const int to = next_place(on ? s_entry[wave * keep + i + lane] : 0, on, bits, count);
      if (on) order[to] = s_place[wave * keep + i + lane];
    }
  } else {
    for (long long n = n0; n < n1; n += kOrderAhead * kWave) {
      uint32_t v[kOrderAhead];
#pragma unroll
      for (int a = 0; a < kOrderAhead; ++a) {
        const long long at = n + a * kWave + lane;
        v[a] = (at < n1 ? raw_entry<SPREAD>(index, at, period) : 0xFFFFFFFFu) - first;
      }
#pragma unroll
      for (int a = 0; a < kOrderAhead; ++a) {
        const bool on = v[a] < mine;
        if (__ballot(on) == 0) continue;                     // uniform
        const int to = next_place(v[a], on, bits, count);
        if (on) order[to] = (int)(n + a * kWave + lane);
      }
    }
  }
  // places of no entry, a share of them: what the table kernel does not write of grad_scale
  if (grad_scale != nullptr)
    for (long long n = (long long)blockIdx.x * kOrderBlock + threadIdx.x; n < N; n += (long long)gridDim.x * kOrderBlock)
      if (entry_of(index, in_index<SPREAD>(n, period), V) < 0)
        for (long long r = 0; r < R; ++r)
          for (int w = 0; w < words; ++w) grad_scale[(r * N + n) * words + w] = 0;
}

// Many places, or a large table: sorted by digits of up to kDigitBits bits, the lowest first, equal ones in their order: how many of each digit each tile of places
// has, where the tiles' go, and they go there; then where each entry's begin.  Places of no entry are left out from the first digit on.
constexpr int kDigitBits = 10, kDigits = 1 << kDigitBits;
constexpr int kSortWaves = 8, kSortBlock = kSortWaves * kWave;
constexpr int kSortSteps = 8, kSortTile = kSortBlock * kSortSteps;           // places of a lane, places of a tile
struct SortPass {
  const void *index;                   // first digit: the index itself
  const uint32_t *keys;                // further ones: what the one before has left, `valid` of them
  const int *places;
  uint32_t *keys_out;
  int *places_out, *counts, *totals, *valid, *many_count;       // counts (digits, tiles), totals (digits)
  int N, period, V, tiles, shift, bits;        // this digit's bits
  bool first;
};
// a wavefront's places: step k's lane has the place first + k * 64 + lane of the sequence
template <typename I, bool SPREAD>
__device__ __forceinline__ bool sort_key(const SortPass &p, long long at, int valid, uint32_t &key, int &place) {
  if (at >= valid) return false;
  if (p.first) {
    const int v = entry_of((const I *)p.index, in_index<SPREAD>(at, p.period), p.V);
    key = (uint32_t)v;
    place = (int)at;
    return v >= 0;
  }
  key = p.keys[at];
  place = p.places[at];
  return true;
}
template <typename I, bool SPREAD>
__global__ __launch_bounds__(kSortBlock) void embedding_digits_kernel(SortPass p, uint32_t *__restrict__ grad_scale, long long R, int words) {
  __shared__ int s_count[kDigits];
  const int digits = 1 << p.bits, valid = p.first ? p.N : *p.valid;
  for (int k = threadIdx.x; k < digits; k += kSortBlock) s_count[k] = 0;
  if (p.first && blockIdx.x == 0 && threadIdx.x == 0) p.many_count[0] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortSteps; ++k) {
    const long long at = (long long)blockIdx.x * kSortTile + k * kSortBlock + threadIdx.x;
    uint32_t key = 0;
    int place;
    if (sort_key<I, SPREAD>(p, at, valid, key, place)) atomicAdd(&s_count[key >> p.shift & (digits - 1)], 1);
    else if (p.first && at < valid && grad_scale != nullptr)                 // (what the table kernel does not write)
      for (long long r = 0; r < R; ++r)
        for (int w = 0; w < words; ++w) grad_scale[(r * p.N + at) * words + w] = 0;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < digits; k += kSortBlock) p.counts[(long long)k * p.tiles + blockIdx.x] = s_count[k];
}
// A wavefront per digit: what the tiles before have of it, and how many there are.
__global__ __launch_bounds__(kEmbBlock) void embedding_tiles_kernel(SortPass p) {
  const int lane = threadIdx.x % kWave, digit = blockIdx.x * (kEmbBlock / kWave) + threadIdx.x / kWave;
  if (digit >= 1 << p.bits) return;
  int *counts = p.counts + (long long)digit * p.tiles, before = 0;
#pragma unroll 4
  for (int t = 0; t < p.tiles; t += kWave) {
    const int have = t + lane < p.tiles ? counts[t + lane] : 0;
    int upto = have;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int u = __shfl_up(upto, off, kWave);
      if (lane >= off) upto += u;
    }
    if (t + lane < p.tiles) counts[t + lane] = before + upto - have;
    before += __shfl(upto, kWave - 1, kWave);
  }
  if (lane == 0) p.totals[digit] = before;
}
template <typename I, bool SPREAD>
__global__ __launch_bounds__(kSortBlock) void embedding_sort_kernel(SortPass p) {
  extern __shared__ int s_next[];      // (kSortWaves, digits): how many of a digit a wavefront has, then where its next one goes
  __shared__ int s_part[kSortWaves];
  const int digits = 1 << p.bits, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, valid = p.first ? p.N : *p.valid;
  for (int k = threadIdx.x; k < kSortWaves * digits; k += kSortBlock) s_next[k] = 0;
  __syncthreads();
  int *const next = s_next + wave * digits;
  uint32_t key[kSortSteps];
  int place[kSortSteps];
  bool on[kSortSteps];
#pragma unroll
  for (int k = 0; k < kSortSteps; ++k) {
    key[k] = 0;
    place[k] = 0;
    on[k] = sort_key<I, SPREAD>(p, (long long)blockIdx.x * kSortTile + (wave * kSortSteps + k) * kWave + lane, valid, key[k], place[k]);
  }
#pragma unroll
  for (int k = 0; k < kSortSteps; ++k)
    if (on[k]) atomicAdd(&next[key[k] >> p.shift & (digits - 1)], 1);
  __syncthreads();
  // digits before, tiles before, wavefronts before
  int base = 0;
  for (int k0 = 0; k0 < digits; k0 += kSortBlock) {
    const int k = k0 + threadIdx.x;
    const int all = k < digits ? p.totals[k] : 0, tiles_before = k < digits ? p.counts[(long long)k * p.tiles + blockIdx.x] : 0;
    int upto = all;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int u = __shfl_up(upto, off, kWave);
      if (lane >= off) upto += u;
    }
    if (lane == kWave - 1) s_part[wave] = upto;
    __syncthreads();
    int at = base + upto - all + tiles_before;
    for (int w = 0; w < wave; ++w) at += s_part[w];
    if (k < digits)
      for (int w = 0; w < kSortWaves; ++w) {
        const int c = s_next[w * digits + k];
        s_next[w * digits + k] = at;
        at += c;
      }
    for (int w = 0; w < kSortWaves; ++w) base += s_part[w];
    __syncthreads();
  }
  if (p.first && blockIdx.x == 0 && threadIdx.x == 0) *p.valid = base;
#pragma unroll
  for (int k = 0; k < kSortSteps; ++k) {
    const int to = next_place(key[k] >> p.shift & (digits - 1), on[k], p.bits, next);
    if (on[k]) {
      p.keys_out[to] = key[k];
      p.places_out[to] = place[k];
    }
  }
}
// starts (V + 1) from the sorted keys, by halving; EACH > 1: where a workgroup's entries begin and end first, and those of each in between, if there are any.  And
// the entries of many places.
template <int EACH>
__global__ __launch_bounds__(kEmbBlock) void embedding_starts_kernel(const uint32_t *__restrict__ keys, const int *__restrict__ valid, int *__restrict__ starts,
                                                                     Many *__restrict__ many, int *__restrict__ many_count, int V, int chunk) {
  constexpr int kSpan = EACH * kEmbBlock;
  __shared__ int s_start[kSpan + 1];
  __shared__ int s_range[2];
  auto first_of = [&](long long v, int lo, int hi) {         // the first key from lo on that is not below v
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if ((long long)keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  for (long long v0 = (long long)blockIdx.x * kSpan; v0 <= V; v0 += (long long)gridDim.x * kSpan) {
    int lo = 0, hi = *valid;
    if constexpr (EACH > 1) {
      if (threadIdx.x < 2) s_range[threadIdx.x] = first_of(v0 + (int)threadIdx.x * kSpan, lo, hi);
      __syncthreads();
      lo = s_range[0];
      hi = s_range[1];
    }
    if (lo < hi) {                                           // uniform
#pragma unroll
      for (int k = threadIdx.x; k < kSpan; k += kEmbBlock) s_start[k] = first_of(v0 + k, lo, hi);
      if (threadIdx.x == 0) s_start[kSpan] = EACH > 1 ? hi : first_of(v0 + kSpan, lo, hi);
      __syncthreads();
    }
#pragma unroll
    for (int k = threadIdx.x; k < kSpan; k += kEmbBlock) {
      const long long v = v0 + k;
      const int from = lo < hi ? s_start[k] : lo, to = lo < hi ? s_start[k + 1] : lo;
      if (v <= V) starts[v] = from;
      if (v < V && to - from > chunk) many[atomicAdd(many_count, 1)] = Many{(int)v, from, to};
    }
    __syncthreads();
  }
}
// Which way.  The one launch's time grows with the places times the workgroups, as each of them reads the whole index; the digits' with their launches, four
// for each digit but one, at the least.  65536 places of 128000 entries at random: the one launch 40 us, two digits 61 to 90; most of them the same few entries, 105 to 117 and
// 94.  131072 places: the digits the same or better in both.  49200 places: the one launch in all (12 us).  More entries than the workgroups' counts have
// room for leave the digits: 1000 places of 9000000 entries, three digits 43 us and the begins 20 of a backward of 157, whose zeros take 97.
static bool ordered_at_once(int N, int V) { return V <= kOrderGroups * kOrderPer && N <= (1 << 16); }

// ---------------------------------------------------------------------------------------------------------------------------------------------
// The table's gradient, and with it (SCALED) that of the scales: bound by memory (40000 entries of 8 rows of 256 floats, read and written, and 49200 g rows,
// 706 MB, 137 us).  A wavefront's lanes stand side by side on a row's pieces (`lanes` a power of two of
// them), as many entries at once as 64 lanes have room for, HB heads of an entry at once: an entry's g rows are read once for all of them, and its rows of the
// table once for all of its places.  A wavefront takes up to kRunOf entries one after the other, whose begins it has read at once: most of a table's entries have no
// place and are zeros to be written.  (Heads at once, that case: 2 243 us with the forward, 4 231, 8 236; the registers decide, as they do for places at
// once, 2 253, 1 233.)  Entries with more than `chunk` places are left to the pieces: the sorted places are cut every `chunk`, and a cut piece holds parts of
// at most two such entries, at its begin and at its end.
// ---------------------------------------------------------------------------------------------------------------------------------------------
template <int HB> constexpr int kRunOf = HB == 1 ? 8 : 4;      // entries that a wavefront takes at the most
constexpr int places_at_once(int hb) { return hb == 1 ? 4 : 1; }

struct TableGrad {
  const void *table, *index, *scale, *grad;
  void *grad_table, *grad_scale;
  const int *order, *starts;
  const Many *many;
  const int *many_count;               // entries of more than `chunk` places: order_groups lists, a list's from the (its number * order_per)-th of `many` on
  int order_groups, order_per;
  void *parts;                         // (chunks, 2, H, E)
  long long R;
  int N, period, V, H, E;
  int chunk, chunks;                   // chunks 0: no entry can have more than `chunk` places
  int lanes, slices, head_blocks, run;
  double mul;
};

// HB values of each of `lanes` neighbouring lanes (a power of two, at least HB), summed over them: the lane gets the sum of one of the values, the `head`.  Halves of
// the values change sides with halves of the lanes: HB + log2(lanes / HB) exchanges, not HB log2(lanes).
template <int HB, typename A>
__device__ __forceinline__ A lanes_sums(A (&x)[HB], int lanes, int at, int &head) {
  int off = lanes / 2;
  head = 0;
#pragma unroll
  for (int n = HB / 2; n > 0; n /= 2) {
    const bool upper = (at & off) != 0;
#pragma unroll
    for (int h = 0; h < n; ++h) {
      const A other = __shfl_xor(upper ? x[h] : x[h + n], off, kWave);
      x[h] = (upper ? x[h + n] : x[h]) + other;
    }
    head += upper ? n : 0;
    off /= 2;
  }
  for (; off > 0; off /= 2) x[0] += __shfl_xor(x[0], off, kWave);
  return x[0];
}

// Adds the places order[from, to) of an entry to `sum` for one slice of a row; `first` is order[from].  SCALED: the products of the entry's rows `t` and the
// places' g rows go to grad_scale, on top of what the slices before have put there.
template <typename T, int VEC, int HB, bool SCALED>
__device__ __forceinline__ void add_places(const TableGrad &a, int from, int to, int first, int h0, int slice, int at, const typename Sum<T>::type (&t)[HB][VEC],
                                           typename Sum<T>::type (&sum)[HB][VEC]) {
  typedef typename Sum<T>::type A;
  constexpr int kAtOnce = places_at_once(HB);                // (with and without SCALED: it is the order of the sum)
  const A *scale = (const A *)a.scale;
  const int e = (slice * a.lanes + at) * VEC;
  const bool on = e < a.E, all_heads = h0 + HB <= a.H;
  int n[kAtOnce], n_next[kAtOnce];                           // (the next places are asked for before the rows of these)
#pragma unroll
  for (int u = 0; u < kAtOnce; ++u) n_next[u] = u == 0 ? first : a.order[min(from + u, to - 1)];
  for (int k = from; k < to; k += kAtOnce) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      n[u] = n_next[u];
      n_next[u] = a.order[min(k + kAtOnce + u, to - 1)];
    }
    for (long long r = 0; r < a.R; ++r) {
      A g[kAtOnce][VEC], s[kAtOnce][HB];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u > 0 && k + u >= to) continue;                  // (the same for all lanes of an entry)
        const long long row = r * a.N + n[u];
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[u][i] = 0;
        if (on) load_row<T, VEC>((const T *)a.grad + row * a.E + e, g[u]);
#pragma unroll
        for (int h = 0; h < HB; ++h) s[u][h] = 1;
        if (scale != nullptr) {
          if (all_heads) {
#pragma unroll
            for (int h = 0; h < HB; ++h) s[u][h] = scale[row * a.H + h0 + h];
          } else {
#pragma unroll
            for (int h = 0; h < HB; ++h) s[u][h] = scale[row * a.H + min(h0 + h, a.H - 1)];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (u > 0 && k + u >= to) continue;
#pragma unroll
        for (int h = 0; h < HB; ++h)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[h][i] += s[u][h] * g[u][i];
        if constexpr (SCALED) {
          A dot[HB];
#pragma unroll
          for (int h = 0; h < HB; ++h) {
            dot[h] = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) dot[h] += t[h][i] * g[u][i];
          }
          int head;
          const A whole = (A)a.mul * lanes_sums<HB>(dot, a.lanes, at, head);
          if (at % (a.lanes / HB) == 0 && h0 + head < a.H) {
            A *to_scale = (A *)a.grad_scale + (r * a.N + n[u]) * a.H + h0 + head;
            *to_scale = whole + (slice > 0 ? *to_scale : (A)0);
          }
        }
      }
    }
  }
}

// the lanes' elements of HB rows of an entry
template <typename T, int VEC, int HB>
__device__ __forceinline__ void load_entry(const TableGrad &a, long long v, int h0, int e, typename Sum<T>::type (&t)[HB][VEC]) {
#pragma unroll
  for (int h = 0; h < HB; ++h) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[h][i] = 0;
    if (e < a.E) load_row<T, VEC, true>((const T *)a.table + (v * a.H + min(h0 + h, a.H - 1)) * a.E + e, t[h]);
  }
}
template <int HB, int VEC, typename A> __device__ __forceinline__ void clear(A (&sum)[HB][VEC]) {
#pragma unroll
  for (int h = 0; h < HB; ++h)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[h][i] = 0;
}

template <typename T, typename I, int VEC, int HB, bool SCALED>
__global__ __launch_bounds__(kEmbBlock) void embedding_table_kernel(TableGrad a, long long piece_units, long long units) {
  typedef typename Sum<T>::type A;
  const int lane = threadIdx.x % kWave, side = lane / a.lanes, at = lane - side * a.lanes, sides = kWave / a.lanes;
  const long long waves = (long long)gridDim.x * (kEmbBlock / kWave);
  const int slices_here = SCALED ? a.slices : 1, slices_apart = SCALED ? 1 : a.slices;
  // units, the longest first: (piece, slice, heads), `sides` pieces at once, then (run of entries, slice, heads) by `sides` neighbouring entries; SCALED: all slices
  for (long long w = (long long)blockIdx.x * (kEmbBlock / kWave) + threadIdx.x / kWave; w < units; w += waves) {
    const bool whole = w >= piece_units;                     // uniform
    long long u = whole ? w - piece_units : w;
    const int h0 = (int)(u % a.head_blocks) * HB;
    u /= a.head_blocks;
    const int slice0 = (int)(u % slices_apart);
    u /= slices_apart;
    A sum[HB][VEC], t[HB][VEC];
    if (whole) {
      // lane k of an entry's lanes reads where the k-th one's places begin, and the first of them
      const long long v0 = u * a.run * sides + side, ahead = min(v0 + min(at, a.run - 1) * sides, (long long)a.V - 1);
      const int from_ahead = a.starts[ahead], to_ahead = a.starts[ahead + 1], first_ahead = a.order[max(min(from_ahead, to_ahead - 1), 0)];
#pragma unroll 1
      for (int k = 0; k < a.run; ++k) {
        const long long v = v0 + k * sides;
        const int from = __shfl(from_ahead, lane - at + k, kWave), to = __shfl(to_ahead, lane - at + k, kWave), first = __shfl(first_ahead, lane - at + k, kWave);
        if (v >= a.V || (a.chunks > 0 && to - from > a.chunk)) continue;
        for (int s = 0; s < slices_here; ++s) {
          const int slice = slice0 + s, e = (slice * a.lanes + at) * VEC;
          clear(sum);
          if (to > from) {
            if constexpr (SCALED) load_entry<T, VEC, HB>(a, v, h0, e, t);
            add_places<T, VEC, HB, SCALED>(a, from, to, first, h0, slice, at, t, sum);
          }
#pragma unroll
          for (int h = 0; h < HB; ++h) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[h][i] *= to > from ? (A)a.mul : (A)0;      // (a mul of infinity adds nothing to an entry without a place)
            if (e < a.E && h0 + h < a.H) store_row<T, VEC, true>((T *)a.grad_table + (v * a.H + h0 + h) * a.E + e, sum[h]);
          }
        }
      }
    } else {
      u = u * sides + side;
      if (u >= a.chunks) continue;
      const int total = a.starts[a.V], c0 = (int)min(u * a.chunk, (long long)total), c1 = (int)min((u + 1) * a.chunk, (long long)total);
      if (c0 >= c1) continue;
      const I *index = (const I *)a.index;
      const int v[2] = {(int)index[in_index<true>(a.order[c0], a.period)], (int)index[in_index<true>(a.order[c1 - 1], a.period)]};
      for (int part = 0; part < (v[1] == v[0] ? 1 : 2); ++part) {
        const int begin = a.starts[v[part]], end = a.starts[v[part] + 1];
        if (end - begin <= a.chunk) continue;
        const int from = max(begin, c0), to = min(end, c1);
        for (int s = 0; s < slices_here; ++s) {
          const int slice = slice0 + s, e = (slice * a.lanes + at) * VEC;
          clear(sum);
          if constexpr (SCALED) load_entry<T, VEC, HB>(a, v[part], h0, e, t);
          add_places<T, VEC, HB, SCALED>(a, from, to, a.order[from], h0, slice, at, t, sum);
#pragma unroll
          for (int h = 0; h < HB; ++h)
            if (e < a.E && h0 + h < a.H) store_row<A, VEC>((A *)a.parts + (((u * 2 + part) * a.H + h0 + h) * a.E + e), sum[h]);
        }
      }
    }
  }
}

// Entries of many places: a workgroup takes every gridDim.x-th of those listed and a slice of its H * E sums (blockIdx.y); its wavefronts add up shares of
// the entry's pieces, in order.  (Four wavefronts with four times the workgroups and sixteen: a backward of 65536 places of 500 entries of 8 x 128 bf16 126 us and
// 149, both passes of 16384 places of 50000 entries of 1024 65 and 69, one entry with all of 1048576 places 301 and 253.)
constexpr int kJoinWaves = 4, kJoinBlock = kJoinWaves * kWave;
template <typename T>
__global__ __launch_bounds__(kJoinBlock) void embedding_join_kernel(TableGrad a) {
  typedef typename Sum<T>::type A;
  __shared__ A s_sum[kJoinWaves][kWave];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, HE = a.H * a.E;
  int before = 0;                                            // of the list, in the workgroups before
  int haves[kOrderGroups / kWave];
#pragma unroll
  for (int i = 0; i < kOrderGroups / kWave; ++i) haves[i] = i * kWave + lane < a.order_groups ? a.many_count[i * kWave + lane] : 0;
#pragma unroll
  for (int i = 0; i < kOrderGroups / kWave; ++i) {           // every wavefront does the same
    const int w0 = i * kWave, have = haves[i];
    int upto = have;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int u = __shfl_up(upto, off, kWave);
      if (lane >= off) upto += u;
    }
    const int all = __shfl(upto, kWave - 1, kWave);
    // the next number of the list that is this workgroup's
    const int G = (int)gridDim.x;
    for (int nth = before + ((int)blockIdx.x - before % G + G) % G; nth < before + all; nth += G) {      // uniform over the workgroup
      const unsigned long long not_yet = __ballot(before + upto <= nth);
      const int l = __popcll(not_yet);
      const int at = nth - before - __shfl(upto - have, l, kWave);
      const Many of = a.many[(long long)(w0 + l) * a.order_per + at];
      const int c = of.from / a.chunk, pieces = (of.to - 1) / a.chunk - c + 1, share = (pieces + kJoinWaves - 1) / kJoinWaves;
      const int p0 = wave * share, p1 = min(p0 + share, pieces);
      const int first_slot = of.from > c * a.chunk;          // (another entry begins its first piece)
      for (int e0 = blockIdx.y * kWave; e0 < HE; e0 += gridDim.y * kWave) {
        const int e = e0 + lane;
        A sum = 0;
        if (e < HE) {
          const A *part = (const A *)a.parts + e;
#pragma unroll 16
          for (int p = p0; p < p1; ++p) sum += part[((long long)(c + p) * 2 + (p == 0 ? first_slot : 0)) * HE];
        }
        s_sum[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && e < HE) {
#pragma unroll
          for (int w = 1; w < kJoinWaves; ++w) sum += s_sum[w][lane];
          Elem<T>::st((T *)a.grad_table + (long long)of.entry * HE + e, sum * (A)a.mul);
        }
        __syncthreads();
      }
    }
    before += all;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------------------------

static int table_lanes(int E, int vec) {
  int lanes = 4;                       // (as many as heads at once)
  while (lanes < kWave && lanes * vec < E) lanes *= 2;
  return lanes;
}
static int heads_at_once(int H) { return H >= 4 ? 4 : H >= 2 ? 2 : 1; }
// Places of an entry that the lanes of a row add up, and more than which make it an entry of many: pieces for some 4096 wavefronts, of 16 places at the least
// (65536 places of 500 entries of 8 x 128 bf16: 32 at the least 126 us of a backward, 16 95).
static int table_chunk(int N, int H, int E, int vec) {
  const int lanes = table_lanes(E, vec), sides = kWave / lanes, slices = (E + lanes * vec - 1) / (lanes * vec), hb = heads_at_once(H);
  const long long units = (long long)slices * ((H + hb - 1) / hb);
  long long chunk = 16;
  while (chunk < 1024 && chunk * 4096 * sides < N * units) chunk *= 2;
  return (int)chunk;
}
// Whether the batch elements of a place are places of their own, which are ordered and cut into pieces as others: where there are too few entries to keep the chip
// at work while wavefronts add up one after the other many batch elements of each of an entry's places.  (Batch elements x places of entries x heads x elements in
// float, gradients on the device: 1000 x 5 of 100 x 256 188 us of a pass and 47, 500 x 100 of 50 x 8 x 32 1912 and 62, 256 x 256 of 256 x 768 100 and 66, 64 x 250 of
// 1000 x 256 31 and 26; 64 x 1000 of 1000 x 256 36 and 48, 32 x 300 of 300 x 8 x 256 37 and 44, 16 x 1000 of 1000 x 256 15 and 24.)
// With more than 2^20 places in all, ordering them costs as well: there both sides' times are weighed.  A wavefront's step takes some 1.2 us (bfloat16 by eights 2.5); one after
// the other it makes them for all batch elements of an entry's or a piece's places; as places of their own a million takes 80 us to order, then g for all heads at the
// rate of a copy or a piece's steps, and the join 1 us for 64 pieces of an entry.  (Likewise: 20000 x 100 of 100 x 256 10191 and 433, 1020 x 16747 of 266 x 8 x 68 15878 and
// 3265, 300 x 4000 of 300 x 16 1512 and 104, 147 x 52107 of 323 x 4 817 and 475, 9 x 131072 of 900 x 2 x 4 145 and 125; 64 x 20000 of 100 x 256 290 and 340, 8 x 200000 of
// 1000 x 4 107 and 143, 12 x 100000 of 100 x 8 x 64 244 and 362, 239 x 15296 of one of 16 634 and 1031.)  And more than 2^20 batch elements always, as one float adds
// up those of a place that are not places of their own.
constexpr long long kMostPlaces = 1LL << 30, kSerialElements = 1LL << 20;
static bool spread_over(long long R, int N, int V, int H, int E, int vec) {
  if (R < 8 || R > kMostPlaces / N) return false;
  if (R > kSerialElements) return true;
  const int lanes = table_lanes(E, vec), slices = (E + lanes * vec - 1) / (lanes * vec), hb = heads_at_once(H), head_blocks = (H + hb - 1) / hb, entries = std::min(N, V);
  if (R * N <= (1 << 20)) return R * N / entries >= 128 && (long long)entries * slices * head_blocks / (kWave / lanes) < 1024;
  const double all = (double)R * N, step = vec == 8 ? 2.5 : 1.2;
  auto steps = [&](int places) { return (places + places_at_once(hb) - 1) / places_at_once(hb); };
  const int chunk = table_chunk((int)(R * N), H, E, vec);
  const double serial = step * R * steps(std::min((N + entries - 1) / entries, table_chunk(N, H, E, vec)));
  const double own = 25 + 80e-6 * all + std::max(all * head_blocks * E * 4 / 5.1e6, step * steps(chunk)) + all / chunk / entries / 64;
  return serial > own;
}
// Batch elements that would have to be places of their own, and are more than can be.
bool embedding_too_many(long long R, int N) { return R > kSerialElements && R > kMostPlaces / N; }
static size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }
// What the ordering leaves and what it works in, from `ws` on (or nullptr: how large that is).
struct OrderPlan {
  int *order, *starts, *many_count, *valid, *counts, *totals, *places[2];
  uint32_t *keys[2];
  Many *many;
  int per, groups, tiles, passes, bits;
  size_t bytes;
};
static OrderPlan order_plan(int N, int V, char *ws) {
  OrderPlan p{};
  auto take = [&](size_t bytes) { char *at = ws == nullptr ? nullptr : ws + p.bytes; p.bytes += rounded(bytes); return at; };
  p.starts = (int *)take((size_t)(V + 1LL) * 4);
  if (ordered_at_once(N, V)) {
    p.per = (V + kOrderGroups - 1) / kOrderGroups;
    p.groups = (V + p.per - 1) / p.per;
    while ((1 << p.bits) < p.per) ++p.bits;
    p.order = (int *)take((size_t)N * 4);
    p.many_count = (int *)take((size_t)p.groups * 4);
    p.many = (Many *)take((size_t)V * sizeof(Many));
    return p;
  }
  int bits = 1;
  while (bits < 31 && (1LL << bits) < V) ++bits;
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tiles = (N + kSortTile - 1) / kSortTile;
  p.groups = 1;
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = (uint32_t *)take((size_t)N * 4);
    p.places[k] = (int *)take((size_t)N * 4);
  }
  p.order = p.places[(p.passes - 1) % 2];
  p.counts = (int *)take(((size_t)p.tiles << p.bits) * 4);
  p.totals = (int *)take((size_t)4 << p.bits);
  p.valid = (int *)take(4);
  p.many_count = (int *)take(4);
  p.many = (Many *)take((size_t)(N / 16 + 1) * sizeof(Many));          // (no fewer than 16 places make an entry of many)
  return p;
}
size_t embedding_workspace_bytes(long long R, int one, int V, int H, int E, int dtype) {
  // (whatever the operands' alignment turns out to be)
  const size_t elem = dtype == DFA3D_F64 ? 8 : 4;
  size_t most = 0;
  for (int vec = 1; vec <= (dtype == DFA3D_BF16 ? 8 : dtype == DFA3D_F32 ? 4 : 2); vec *= 2) {
    const int N = spread_over(R, one, V, H, E, vec) ? (int)(R * one) : one, chunk = table_chunk(N, H, E, vec);
    most = std::max(most, order_plan(N, V, nullptr).bytes + (N > chunk ? (size_t)((N + chunk - 1) / chunk) * 2 * H * E * elem : 0));
  }
  return most;
}

static unsigned emb_grid(long long threads) {
  const long long blocks = (threads + kEmbBlock - 1) / kEmbBlock;
  return (unsigned)(blocks < 1 ? 1 : blocks > (1 << 20) ? 1 << 20 : blocks);
}

template <typename T, typename I, int VEC>
static hipError_t embedding_cfg(const EmbeddingArgs &a, hipStream_t stream) {
  typedef typename Sum<T>::type A;
  const long long rows = a.R * a.N;
  const Pieces pieces(rows, a.E / VEC);
  hipLaunchKernelGGL((embedding_kernel<T, I, VEC>), dim3(emb_grid(rows * pieces.per)), dim3(kEmbBlock), 0, stream, (const T *)a.table, (const I *)a.index,
                     (const A *)a.scale, (const T *)a.plus, (T *)a.out, rows, Pieces(a.R, a.N), a.V, a.H, a.E, (A)a.mul, pieces);
  return hipGetLastError();
}
template <typename T, typename I, int VEC>
static hipError_t scale_cfg(const EmbeddingArgs &a, hipStream_t stream) {
  typedef typename Sum<T>::type A;
  const long long rows = a.R * a.N;
  hipLaunchKernelGGL((embedding_scale_kernel<T, I, VEC>), dim3(emb_grid(rows * kWave)), dim3(kEmbBlock), 0, stream, (const T *)a.table, (const I *)a.index,
                     (const T *)a.grad, (A *)a.grad_scale, rows, Pieces(a.R, a.N), a.V, a.H, a.E, (A)a.mul);
  return hipGetLastError();
}
template <typename T, typename I, int VEC, int HB, bool SCALED>
static hipError_t table_launch(TableGrad &t, hipStream_t stream) {
  const int sides = kWave / t.lanes;
  const long long per = (long long)(SCALED ? 1 : t.slices) * t.head_blocks;
  // one after the other only where that leaves wavefronts for all of the chip: where entries are few, they have places
  t.run = (int)std::max(std::min(t.V * per / (sides * 8192LL), (long long)std::min(kRunOf<HB>, t.lanes)), 1LL);
  const long long piece_units = ((long long)t.chunks + sides - 1) / sides * per, units = piece_units + ((long long)t.V + sides * t.run - 1) / (sides * t.run) * per;
  hipLaunchKernelGGL((embedding_table_kernel<T, I, VEC, HB, SCALED>), dim3(emb_grid(units * kWave)), dim3(kEmbBlock), 0, stream, t, piece_units, units);
  if (hipError_t e = hipGetLastError()) return e;
  if (t.chunks == 0) return hipSuccess;
  // workgroups for 1024 entries and slices at once; where no entry has many places all find the list empty.  (Both passes of 16384 places of 50000 entries of 1024 bf16:
  // 4096 63.4 us, 2048 60.5, 1024 57.5, 512 58.5, 256 60.8; a backward of 65536 places of 500 entries of 8 x 128 89, 87, 85, 92, 115.)
  const int slices = std::min((t.H * t.E + kWave - 1) / kWave, 512);
  hipLaunchKernelGGL((embedding_join_kernel<T>), dim3(std::min(t.chunks, std::max(1024 / slices, 16)), slices), dim3(kJoinBlock), 0, stream, t);
  return hipGetLastError();
}
template <typename A, typename I, bool SPREAD>
static hipError_t launch_order(const EmbeddingArgs &a, const OrderPlan &p, int period, int chunk, hipStream_t stream) {
  uint32_t *grad_scale = (uint32_t *)a.grad_scale;
  const int words = (int)(a.H * sizeof(A) / 4);
  if (p.per > 0) {
    const int keep = (kOrderLds / kOrderWaves - p.per * 4) / 6 / kWave * kWave;
    hipLaunchKernelGGL((embedding_order_kernel<I, SPREAD>), dim3(p.groups), dim3(kOrderBlock), (size_t)kOrderWaves * (p.per * 4 + keep * 6), stream, (const I *)a.index, p.order,
                       p.starts, p.many, p.many_count, a.N, period, a.V, p.per, p.bits, keep, chunk, grad_scale, a.R, words);
    return hipGetLastError();
  }
  for (int k = 0; k < p.passes; ++k) {
    const SortPass s = {a.index, p.keys[(k + 1) % 2], p.places[(k + 1) % 2], p.keys[k % 2], p.places[k % 2], p.counts, p.totals, p.valid, p.many_count,
                        a.N, period, a.V, p.tiles, k * p.bits, p.bits, k == 0};
    hipLaunchKernelGGL((embedding_digits_kernel<I, SPREAD>), dim3(p.tiles), dim3(kSortBlock), 0, stream, s, grad_scale, a.R, words);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(embedding_tiles_kernel, dim3(((1 << p.bits) + kEmbBlock / kWave - 1) / (kEmbBlock / kWave)), dim3(kEmbBlock), 0, stream, s);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((embedding_sort_kernel<I, SPREAD>), dim3(p.tiles), dim3(kSortBlock), (size_t)kSortWaves * sizeof(int) << p.bits, stream, s);
    if (hipError_t e = hipGetLastError()) return e;
  }
  // (us: 256k places of 256000 entries one at a time 8.9, eight 23.8; 256k of 9000000 102 and 41, 1000 of 9000000 53 and 20)
  auto starts = [&](auto kernel, int span) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((a.V + (long long)span) / span)), dim3(kEmbBlock), 0, stream, p.keys[(p.passes - 1) % 2], p.valid, p.starts, p.many, p.many_count,
                       a.V, chunk);
  };
  a.V > (1 << 21) ? starts(embedding_starts_kernel<8>, 8 * kEmbBlock) : starts(embedding_starts_kernel<1>, kEmbBlock);
  return hipGetLastError();
}
template <typename T, typename I, int VEC>
static hipError_t table_cfg(const EmbeddingArgs &given, hipStream_t stream) {
  typedef typename Sum<T>::type A;
  EmbeddingArgs a = given;
  if (spread_over(a.R, a.N, a.V, a.H, a.E, VEC)) {
    a.N = (int)(a.R * a.N);
    a.R = 1;
  }
  const OrderPlan plan = order_plan(a.N, a.V, (char *)a.workspace);
  TableGrad t{};
  t.lanes = table_lanes(a.E, VEC);
  t.slices = (a.E + t.lanes * VEC - 1) / (t.lanes * VEC);
  t.chunk = table_chunk(a.N, a.H, a.E, VEC);
  t.chunks = a.N > t.chunk ? (a.N + t.chunk - 1) / t.chunk : 0;
  t.order = plan.order; t.starts = plan.starts; t.many = plan.many; t.many_count = plan.many_count; t.order_per = plan.per; t.order_groups = plan.groups;
  t.parts = (char *)a.workspace + plan.bytes;
  if (hipError_t e = a.N > given.N ? launch_order<A, I, true>(a, plan, given.N, t.chunk, stream) : launch_order<A, I, false>(a, plan, given.N, t.chunk, stream)) return e;
  t.table = a.table; t.index = a.index; t.scale = a.scale; t.grad = a.grad; t.grad_table = a.grad_table; t.grad_scale = a.grad_scale;
  t.R = a.R; t.N = a.N; t.period = given.N; t.V = a.V; t.H = a.H; t.E = a.E; t.mul = a.mul;
  const int hb = heads_at_once(a.H);
  t.head_blocks = (a.H + hb - 1) / hb;
  auto with = [&](auto h) {
    constexpr int HB = decltype(h)::value;
    return a.grad_scale != nullptr ? table_launch<T, I, VEC, HB, true>(t, stream) : table_launch<T, I, VEC, HB, false>(t, stream);
  };
  switch (hb) {
    case 4: return with(std::integral_constant<int, 4>());
    case 2: return with(std::integral_constant<int, 2>());
    default: return with(std::integral_constant<int, 1>());
  }
}

enum { kEmbForward, kEmbScale, kEmbTable };
template <typename T, typename I>
static hipError_t embedding_typed(const EmbeddingArgs &a, int what, hipStream_t stream) {
  // (the index is read place by place; what a kernel does not touch is NULL)
  const int vec = row_vec(a.E, (uintptr_t)a.table | (uintptr_t)a.plus | (uintptr_t)a.out | (uintptr_t)a.grad | (uintptr_t)a.grad_table, sizeof(T));      // (workspace: 256)
  auto with = [&](auto v) {
    constexpr int VEC = decltype(v)::value;
    return what == kEmbForward ? embedding_cfg<T, I, VEC>(a, stream) : what == kEmbScale ? scale_cfg<T, I, VEC>(a, stream) : table_cfg<T, I, VEC>(a, stream);
  };
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return with(std::integral_constant<int, 8>());
  if constexpr (sizeof(T) <= 4)
    if (vec == 4) return with(std::integral_constant<int, 4>());
  return vec == 2 ? with(std::integral_constant<int, 2>()) : with(std::integral_constant<int, 1>());
}
static hipError_t embedding_any(const EmbeddingArgs &a, int what, int dtype, hipStream_t stream) {
  auto typed = [&](auto t) {
    typedef decltype(t) T;
    return a.wide_index ? embedding_typed<T, int64_t>(a, what, stream) : embedding_typed<T, int32_t>(a, what, stream);
  };
  if (dtype == DFA3D_F32) return typed(float());
  if (dtype == DFA3D_F64) return typed(double());
  if (dtype == DFA3D_BF16) return typed(__hip_bfloat16());
  return hipErrorInvalidValue;
}
hipError_t launch_embedding(const EmbeddingArgs &a, int dtype, hipStream_t stream) { return embedding_any(a, kEmbForward, dtype, stream); }
hipError_t launch_embedding_grad_scale(const EmbeddingArgs &a, int dtype, hipStream_t stream) { return embedding_any(a, kEmbScale, dtype, stream); }
hipError_t launch_embedding_grad_table(const EmbeddingArgs &a, int dtype, hipStream_t stream) { return embedding_any(a, kEmbTable, dtype, stream); }

}  // namespace dfa3d
