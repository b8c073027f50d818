// What each row of (log) probabilities says: for x over V entries, with m = max x and s = sum e^(x - m),
//   log probability of a given token t   x_t - m - ln s
//   entropy                              ln s - (sum e^(x - m) (x - m)) / s
//   rank of t                            #{x_v > x_t} + #{v < t, x_v = x_t}
//   top k                                by value, equal values by the lowest index, as log probabilities
// Statistics are held in 32 bits whatever the input's type.
#include "scoring.h"

#include <algorithm>
#include <type_traits>

namespace tone {
namespace {

struct ScoreArgs {
  const void* x;
  int64_t stride, x_rows;
  const int64_t* rows;                  // row of x per output row, or nullptr (row n)
  int64_t n;
  int vocab, k;
  const int32_t* tokens;                // or nullptr
  float *logprob, *entropy;
  int32_t* rank;
  float* top_lp;
  int32_t* top_ids;
};

constexpr float kLog2e = 1.4426950408889634f;
// e^z for z <= 0 (v_exp_f32; z log2 e is rounded once, so e^z is off by about |z| 2^-24 of its value: ln s, where each
// term counts as often as it is likely, by 2^-24 of the mean |z|, which is at most the entropy)
__device__ __forceinline__ float exp_neg(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

// total order of the values as integers: larger value = larger integer, -0 and +0 are one value, never INT_MIN or INT_MAX
// (1 can be added; the ends are NaN)
__device__ __forceinline__ int order_of(float v) {
  const int b = __float_as_int(v + 0.0f);
  return min(max(b < 0 ? b ^ 0x7fffffff : b, -0x7fffffff), 0x7ffffffe);
}
// larger value = larger key; equal values: the lower index has the larger key.  Never 0.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
  return ((uint64_t)((uint32_t)order_of(v) ^ 0x80000000u) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float value_of(int order) { return __int_as_float(order < 0 ? order ^ 0x7fffffff : order); }
__device__ __forceinline__ float key_value(uint64_t key) { return value_of((int)((uint32_t)(key >> 32) ^ 0x80000000u)); }
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(uint32_t)key; }

// lane ^ X of a 16-lane row without LDS (DPP); X = 16 or 32: ds_bpermute
template <int X>
__device__ __forceinline__ int xor_lane(int v) {
  if constexpr (X == 1) return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true);        // quad_perm 1 0 3 2
  else if constexpr (X == 2) return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true);   // quad_perm 2 3 0 1
  else if constexpr (X == 3) return __builtin_amdgcn_mov_dpp(v, 0x1b, 0xf, 0xf, true);   // quad_perm 3 2 1 0
  else if constexpr (X == 7) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true);  // row_half_mirror
  else if constexpr (X == 15) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true); // row_mirror
  else if constexpr (X == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xf, 0xf, true);  // row_ror 8
  else if constexpr (X < 7) return xor_lane<7 - X>(xor_lane<7>(v));
  else return __shfl_xor(v, X);
}
template <int X>
__device__ __forceinline__ float xor_lane(float v) { return __int_as_float(xor_lane<X>(__float_as_int(v))); }
template <int X>
__device__ __forceinline__ uint64_t xor_lane(uint64_t v) {
  return ((uint64_t)(uint32_t)xor_lane<X>((int)(v >> 32)) << 32) | (uint32_t)xor_lane<X>((int)(uint32_t)v);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ float read_lane(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

// a commutative operation over the wave's 64 lanes, in a fixed order; uniform
__device__ __forceinline__ int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
template <class V, class Op>
__device__ __forceinline__ V over_wave(V v, Op&& op) {
  v = op(v, xor_lane<1>(v));
  v = op(v, xor_lane<2>(v));
  v = op(v, xor_lane<7>(v));
  v = op(v, xor_lane<15>(v));
  return op(op(read_lane(v, 0), read_lane(v, 16)), op(read_lane(v, 32), read_lane(v, 48)));
}

// what a row that is none gives
__device__ __forceinline__ void write_none(const ScoreArgs& p, int64_t n, int first, int step) {
  if (first == 0) {
    if (p.tokens) {
      p.logprob[n] = 0.f;
      p.rank[n] = -1;
    }
    p.entropy[n] = 0.f;
  }
  for (int i = first; i < p.k; i += step) {
    p.top_lp[n * p.k + i] = -INFINITY;
    p.top_ids[n * p.k + i] = -1;
  }
}

// Rows of up to 64 entries (the 35-token head): 8 lanes per row, entry 8 e + lane in register e, 8 rows per wave.  Every
// entry's rank is counted against all others (the other lanes' registers come by DPP, lane ^ 1 .. 7), so one pass gives the
// given token's rank and the place of each of the top k, whatever k is, with no selection rounds and no LDS: 8 E^2
// compares per 8 rows.  They bound it: 40,960 rows of 35 (9.2 MB in and out, 2 us) take 8.2 us at some 700 vector
// instructions per wave, 187 rows 4.1, of which two are the launch.
template <typename T, int E>
__global__ void __launch_bounds__(256) scores_short_kernel(ScoreArgs p) {
  const int sub = threadIdx.x & 7;
  const int64_t n = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool in = n < p.n;
  const int64_t row = !in ? -1 : p.rows ? p.rows[n] : n;
  const bool here = row >= 0 && row < p.x_rows;
  if (in && !here) write_none(p, n, sub, 8);
  if (!here) return;                     // whole groups of 8 lanes: the DPP exchanges below stay inside a group
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  const int t = p.tokens ? p.tokens[n] : -1;
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 8 * e + sub < p.vocab ? load_elem(x + 8 * e + sub) : -INFINITY;
  float m = -3.402823466e38f;            // finite, so that -inf - m is -inf and a row of -inf sums up to 0
#pragma unroll
  for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
  m = fmaxf(m, xor_lane<1>(m));
  m = fmaxf(m, xor_lane<2>(m));
  m = fmaxf(m, xor_lane<7>(m));
  float s = 0.f, u = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float z = v[e] - m, ex = exp_neg(z);
    s += ex;
    u = fmaf(ex, fmaxf(z, -200.f), u);   // e^-200 is 0 in fp32: the bound keeps 0 x -inf out
  }
  s += xor_lane<1>(s);
  u += xor_lane<1>(u);
  s += xor_lane<2>(s);
  u += xor_lane<2>(u);
  s += xor_lane<7>(s);
  u += xor_lane<7>(u);
  const bool left = s != 0.f;            // a NaN counts as something left
  const float ls = logf(s);
  if (sub == 0) {
    p.entropy[n] = left ? ls - u / s : 0.f;
    if (p.tokens && !(t >= 0 && t < p.vocab)) {
      p.logprob[n] = 0.f;
      p.rank[n] = -1;
    }
  }
  if (!p.k && !p.tokens) return;
  int o[E], above[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    o[e] = 8 * e + sub < p.vocab ? order_of(v[e]) : -0x7fffffff - 1;    // entries that are none are below all
    above[e] = 0;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int f = 0; f < E; ++f)
      if (f != e) above[e] += f < e ? o[f] >= o[e] : o[f] > o[e];
  auto against = [&](const int (&w)[E], int lower) {   // lower: 1 where the other lane is below this one
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int f = 0; f < E; ++f) above[e] += f < e ? w[f] >= o[e] : f > e ? w[f] > o[e] : w[f] + lower > o[e];
    }
  };
  auto with = [&](auto x_) {
    constexpr int X = decltype(x_)::value;
    int w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = xor_lane<X>(o[e]);
    against(w, (sub ^ X) < sub);
  };
  with(std::integral_constant<int, 1>{});
  with(std::integral_constant<int, 2>{});
  with(std::integral_constant<int, 3>{});
  with(std::integral_constant<int, 4>{});
  with(std::integral_constant<int, 5>{});
  with(std::integral_constant<int, 6>{});
  with(std::integral_constant<int, 7>{});
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = 8 * e + sub;
    if (i >= p.vocab) continue;
    const float lp = left ? v[e] - m - ls : -INFINITY;
    if (i == t && p.tokens) {
      p.logprob[n] = lp;
      p.rank[n] = above[e];
    }
    if (above[e] < p.k) {
      p.top_lp[n * p.k + above[e]] = lp;
      p.top_ids[n * p.k + above[e]] = i;
    }
  }
}

// The 64 best keys of a wave, one per lane in descending order (0: none).
struct Best {
  uint64_t key;
  uint64_t floor;                        // the k-th best; keys at or below it do not matter

  __device__ __forceinline__ void clear() { key = floor = 0; }
  __device__ __forceinline__ bool any() const { return read_lane(key, 0) != 0; }
  // another list, in ascending order
  __device__ __forceinline__ void join(uint64_t other, int lane) {
    key = key > other ? key : other;
    step<32>(lane);
    step<16>(lane);
    step<8>(lane);
    step<4>(lane);
    step<2>(lane);
    step<1>(lane);
  }
  // the wave's keys, one per lane, as the first list: a bitonic sort
  __device__ __forceinline__ void sort(uint64_t mine, int lane, int k) {
    key = mine;
    merge<2>(lane);
    merge<4>(lane);
    merge<8>(lane);
    merge<16>(lane);
    merge<32>(lane);
    merge<64>(lane);
    floor = read_lane(key, k - 1);
  }
  // one key per lane: those above the floor go in one after the other
  __device__ __forceinline__ void take(uint64_t mine, int lane, int k) {
    uint64_t todo = __ballot(mine > floor);
    while (todo) {
      const uint64_t c = read_lane(mine, __builtin_ctzll(todo));
      const int at = __builtin_popcountll(__ballot(key > c));
      const uint64_t moved = ((uint64_t)(uint32_t)__builtin_amdgcn_mov_dpp((int)(key >> 32), 0x138, 0xf, 0xf, true) << 32) |
                             (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)key, 0x138, 0xf, 0xf, true);   // wave_shr 1
      key = lane < at ? key : lane == at ? c : moved;
      floor = read_lane(key, k - 1);
      todo &= todo - 1;
      todo &= __ballot(mine > floor);
    }
  }

 private:
  template <int N>
  __device__ __forceinline__ void merge(int lane) {   // sorted runs of N / 2 -> sorted runs of N
    flip<N>(lane);
    if constexpr (N >= 64) step<16>(lane);
    if constexpr (N >= 32) step<8>(lane);
    if constexpr (N >= 16) step<4>(lane);
    if constexpr (N >= 8) step<2>(lane);
    if constexpr (N >= 4) step<1>(lane);
  }
  template <int N>
  __device__ __forceinline__ void flip(int lane) {
    const uint64_t other = xor_lane<N - 1>(key);
    key = ((lane & (N / 2)) == 0) == (key > other) ? key : other;
  }
  template <int D>
  __device__ __forceinline__ void step(int lane) {
    const uint64_t other = xor_lane<D>(key);
    key = ((lane & D) == 0) == (key > other) ? key : other;
  }
};

// the k-th largest of the wave's 64 values, bit by bit from the top
__device__ __forceinline__ float kth_of(float v, int k) {
  const uint32_t mine = (uint32_t)order_of(v) ^ 0x80000000u;
  uint32_t at = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__builtin_popcountll(__ballot(mine >= (at | bit))) >= k) at |= bit;
  return value_of((int)(at ^ 0x80000000u));
}

// 16 bytes of a row
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  union {
    uint4 raw;
    T e[N];
  };
  __device__ Vec() {}
};

// One wave's part of a row, in batches of Q steps of N entries per lane, in ascending order.  The maximum is the wave's, so
// every e^(x - m) is at most 1 and all terms of the entropy's sum have one sign; a batch that brings no new maximum and
// nothing above the k-th best entry (one compare of the lanes' largest against the floor) adds up its terms and nothing else.
struct Part {
  float m = -3.402823466e38f, s = 0.f, u = 0.f;
  int above = 0;                         // of the lane's entries
  float floor = -INFINITY;               // value of the k-th best, or the maximum for k = 0
  bool full = false;                     // k entries seen
  Best best;
  int* shared;                           // the largest floor of the row's waves, as order_of

  // x[q][j]: entry base + (64 q + lane) N + j; those of lanes from valid[q] on are none (-inf).  ALL: there are no such lanes
  template <bool ALL, int Q, int N>
  __device__ __forceinline__ void batch(const float (&x)[Q][N], int base, const int (&valid)[Q], int lane, int k, float xt, int t) {
    float top[Q], most;
#pragma unroll
    for (int q = 0; q < Q; ++q) {        // steps of which no lane has an entry are left out here and below
      if (!ALL && q && valid[q] <= 0) continue;
      top[q] = x[q][0];
#pragma unroll
      for (int j = 1; j < N; ++j) top[q] = fmaxf(top[q], x[q][j]);
      most = q ? fmaxf(most, top[q]) : top[q];
    }
    const float other = shared ? value_of(*static_cast<volatile int*>(shared)) : -INFINITY;
    // (a NaN is not below `other`: lanes of nothing else fill a list that is not full)
    if ((!full || __ballot(most > floor)) && (k == 0 || __ballot(!(most < other))))
      news<ALL, Q, N>(x, top, most, other, base, valid, lane, k);
    else if (__ballot(most > m)) larger(most);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      if (!ALL && q && valid[q] <= 0) continue;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float z = x[q][j] - m, e = exp_neg(z);
        s += e;
        u = fmaf(e, fmaxf(z, -200.f), u);   // as in the short form
      }
    }
    // entries above x_t; equal ones count below index t.  A step without any is passed over: a token worth asking for is
    // among the best (2048 rows over 65,537 entries, bf16: 47 us without tokens, 48 with likely ones, 56 with random ones)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int b = base + q * 64 * N;
      if (t < 0 || (!ALL && q && valid[q] <= 0) || __ballot(top[q] >= xt) == 0) continue;
      if (t >= b + 64 * N) {
#pragma unroll
        for (int j = 0; j < N; ++j) above += x[q][j] >= xt && (ALL || lane < valid[q]);
      } else if (t < b) {
#pragma unroll
        for (int j = 0; j < N; ++j) above += x[q][j] > xt;
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) above += (ALL || lane < valid[q]) && (x[q][j] > xt || (x[q][j] == xt && b + lane * N + j < t));
      }
    }
  }

  __device__ __forceinline__ void larger(float most) {
    const float w = over_wave(most, [](float p_, float q_) { return fmaxf(p_, q_); });
    if (w > m) {
      // s and u to the new maximum: e^(x - w) = e^(x - m) e^d, (x - w) = (x - m) + d; d bounded as in the sums
      const float d = fmaxf(m - w, -200.f), f = exp_neg(d);
      u = f * fmaf(d, s, u);
      s *= f;
      m = w;
    }
  }

  template <bool ALL, int Q, int N>
  __device__ __forceinline__ void news(const float (&x)[Q][N], const float (&top)[Q], float most, float other, int base, const int (&valid)[Q], int lane,
                                       int k) {
    if (__ballot(most > m)) larger(most);
    if (k == 0) {
      floor = m;
      full = true;
      return;
    }
    int best_at = -1;
    // where many lanes have news (rows that ascend), k entries of this batch are at or above `enough`, and others need not go
    // in: 2048 ascending rows over 65,537 entries take 373 us instead of 1130, others 1 us more (k = 10)
    float enough = -INFINITY;
    const int hits = __builtin_popcountll(__ballot(most >= fmaxf(floor, other)));
    if (best.floor && hits >= k && hits > 16) enough = kth_of(most, k);
    if (!best.any()) {
      // nothing held yet: the lanes' largest first, which sets a floor close to the final one
      best_at = 0;                       // (a lane of NaN: its first entry)
      float largest = x[0][0];
#pragma unroll
      for (int q = Q - 1; q >= 0; --q) {
        if (!ALL && q && valid[q] <= 0) continue;
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
          if (x[q][j] == most) {
            best_at = q * N + j;
            largest = most;
          }
      }
      best.sort(ALL || lane < valid[0] ? key_of(largest, base + (best_at / N * 64 + lane) * N + best_at % N) : 0, lane, k);
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      // nothing below another wave's floor can be among the row's k best; what equals it can, by its index
      const float low = fmaxf(fmaxf(best.floor ? key_value(best.floor) : -INFINITY, other), enough);
      if ((!ALL && q && valid[q] <= 0) || (best.floor && __ballot(top[q] >= low) == 0)) continue;      // (a NaN is above no floor, but fills a list)
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!best.floor || __ballot(x[q][j] >= low))
          best.take((ALL || lane < valid[q]) && q * N + j != best_at ? key_of(x[q][j], base + (q * 64 + lane) * N + j) : 0, lane, k);
    }
    full = best.floor != 0;
    if (full) {
      floor = key_value(best.floor);
      if (shared && lane == 0) atomicMax(shared, order_of(floor));
    }
  }
};

// Longer rows: W waves per row, each a contiguous part of it in 16-byte loads from the first aligned entry on (the entries in
// front of it and behind the last whole vector are single loads of the first and the last wave), joined in LDS.  2048 rows over
// 65,537 bf16 entries (268 MB) take 47 us for the entropy alone, 5.7 TB/s, where memory bounds it; the rank of random tokens
// costs 9 us more and ten alternatives 28, of which each of some 35 insertions per row stalls its wave for half a
// microsecond.  One row over 65,536 takes 19.5 us: the first sort, the join and a sixteenth of the row per wave.
template <typename T, int W, int ROWS>
__global__ void __launch_bounds__(64 * W * ROWS) scores_long_kernel(ScoreArgs p) {
  constexpr int N = Vec<T>::N, Q = 4;
  __shared__ float part_f[W * ROWS][3];
  __shared__ int part_i[W * ROWS];
  __shared__ uint64_t part_k[W > 1 ? W / 2 : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = W > 1 ? wave : 0;
  const int64_t n = (int64_t)blockIdx.x * ROWS + (W > 1 ? 0 : wave);
  const bool in = n < p.n;
  const int64_t row = !in ? -1 : p.rows ? p.rows[n] : n;
  const bool here = row >= 0 && row < p.x_rows;
  if (!here) {                           // the whole workgroup, or (W = 1) the wave alone
    if (in && wr == 0) write_none(p, n, lane, 64);
    return;
  }
  __shared__ int s_floor;
  Part a;
  a.best.clear();
  a.shared = nullptr;
  if constexpr (W > 1) {
    if (threadIdx.x == 0) s_floor = order_of(-INFINITY);
    __syncthreads();
    a.shared = &s_floor;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  int t = p.tokens ? p.tokens[n] : -1;
  if (t < 0 || t >= p.vocab) t = -1;
  const float xt = t >= 0 ? load_elem(x + t) : 0.f;
  const int head = min(p.vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (p.vocab - head) / N, each = (vecs + W - 1) / W;
  const int v0 = min(vecs, wr * each), v1 = min(vecs, v0 + each);
  const uint4* base = reinterpret_cast<const uint4*>(x + head);
  Vec<T> v[Q];
  auto load = [&](int c) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = c + 64 * q + lane;
      if (i < v1) v[q].raw = base[i];
    }
  };
  load(v0);
  for (int c = v0; c < v1; c += 64 * Q) {
    float f[Q][N];
    int valid[Q];
    if (c + 64 * Q <= v1) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int j = 0; j < N; ++j) f[q][j] = load_elem(&v[q].e[j]);
      load(c + 64 * Q);
      a.batch<true, Q, N>(f, head + c * N, valid, lane, p.k, xt, t);
    } else {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        valid[q] = v1 - (c + 64 * q);
#pragma unroll
        for (int j = 0; j < N; ++j) f[q][j] = lane < valid[q] ? load_elem(&v[q].e[j]) : -INFINITY;
      }
      a.batch<false, Q, N>(f, head + c * N, valid, lane, p.k, xt, t);
    }
  }
  const int tail = head + vecs * N;
  if (wr == W - 1 && tail < p.vocab) {
    const int valid[1] = {p.vocab - tail};
    const float one[1][1] = {{lane < valid[0] ? load_elem(x + tail + lane) : -INFINITY}};
    a.batch<false, 1, 1>(one, tail, valid, lane, p.k, xt, t);
  }
  if (wr == 0 && head) {
    const int valid[1] = {head};
    const float one[1][1] = {{lane < head ? load_elem(x + lane) : -INFINITY}};
    a.full = false;                      // lower indices than what is held: equal values have to be looked at
    a.batch<false, 1, 1>(one, 0, valid, lane, p.k, xt, t);
  }
  a.s = over_wave(a.s, [](float p_, float q_) { return p_ + q_; });
  a.u = over_wave(a.u, [](float p_, float q_) { return p_ + q_; });
  a.above = over_wave(a.above, [](int p_, int q_) { return p_ + q_; });
  if constexpr (W > 1) {
    if (lane == 0) {
      part_f[wave][0] = a.m;
      part_f[wave][1] = a.s;
      part_f[wave][2] = a.u;
      part_i[wave] = a.above;
    }
    // the waves' lists in pairs: of two lists in descending order, the larger of each entry and the other's mirror image
    // are the 64 best, in an order that log2(64) exchanges sort
#pragma unroll
    for (int w = W / 2; w >= 1; w /= 2) {
      if (p.k) {
        if (wave >= w && wave < 2 * w) part_k[wave - w][63 - lane] = a.best.key;
        __syncthreads();
        if (wave < w) a.best.join(part_k[wave][lane], lane);
        if (w > 1) __syncthreads();
      }
    }
    if (!p.k) __syncthreads();
    if (wr != 0) return;
    float m = a.m;
    for (int w = 1; w < W; ++w) m = fmaxf(m, part_f[w][0]);
    float s = 0.f, u = 0.f;
    a.above = 0;
    for (int w = 0; w < W; ++w) {
      const float d = fmaxf(part_f[w][0] - m, -200.f), f = exp_neg(d);
      u += f * fmaf(d, part_f[w][1], part_f[w][2]);
      s += f * part_f[w][1];
      a.above += part_i[w];
    }
    a.m = m;
    a.s = s;
    a.u = u;
  }
  const bool left = a.s != 0.f;
  const float ls = logf(a.s);
  if (lane == 0) {
    p.entropy[n] = left ? ls - a.u / a.s : 0.f;
    if (p.tokens) {
      p.logprob[n] = t < 0 ? 0.f : left ? xt - a.m - ls : -INFINITY;
      p.rank[n] = t < 0 ? -1 : a.above;
    }
  }
  if (lane < p.k) {
    p.top_lp[n * p.k + lane] = left ? key_value(a.best.key) - a.m - ls : -INFINITY;
    p.top_ids[n * p.k + lane] = key_index(a.best.key);
  }
}

template <typename T, int E>
void short_as(const ScoreArgs& p, hipStream_t st) {
  hipLaunchKernelGGL((scores_short_kernel<T, E>), dim3((unsigned)((p.n + 31) / 32)), dim3(256), 0, st, p);
}

template <typename T>
hipError_t launch_as(const ScoreArgs& p, hipStream_t st) {
  if (p.vocab <= 64) {
    switch ((p.vocab + 7) / 8) {
      case 1: short_as<T, 1>(p, st); break;
      case 2: short_as<T, 2>(p, st); break;
      case 3: short_as<T, 3>(p, st); break;
      case 4: short_as<T, 4>(p, st); break;
      case 5: short_as<T, 5>(p, st); break;
      case 6: short_as<T, 6>(p, st); break;
      case 7: short_as<T, 7>(p, st); break;
      default: short_as<T, 8>(p, st);
    }
    return hipGetLastError();
  }
  // Waves per row, by the 64-lane loads it takes (us, k = 10, with 1 / 4 / 16 waves).  Few rows are a matter of one row's time
  // (bf16 65,537: 1 row 79 / 31 / 19, 256 rows 93 / 35 / 22, 400 rows 92 / 40 / 40; 5000: 256 rows 17 / 10 / 11), and from some
  // 1500 rows on the card is full with one wave each, which sorts once per row instead of four times (bf16 65,537: 1024 rows
  // 77 / 51, 2048 88 / 90; 32,000: 1500 rows 54 / 47, 2600 64 / 73, 4096 77 / 102; 5000: 1024 rows 16 / 13, 2048 17 / 21,
  // 16,384 73 / 116; 2500: 600 rows 11 / 11, 2048 13 / 19).
  const int64_t steps = (p.vocab / Vec<T>::N + 63) / 64;
  if (steps >= 20 && p.n <= 256) hipLaunchKernelGGL((scores_long_kernel<T, 16, 1>), dim3((unsigned)p.n), dim3(1024), 0, st, p);
  else if (steps >= 4 && p.n <= (steps >= 16 ? 1536 : 1024))
    hipLaunchKernelGGL((scores_long_kernel<T, 4, 1>), dim3((unsigned)p.n), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((scores_long_kernel<T, 1, 4>), dim3((unsigned)((p.n + 3) / 4)), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_scores(const ScoreArgs& p, int type, hipStream_t st) {
  switch (type) {
    case TONE_TYPE_FP32: return launch_as<float>(p, st);
    case TONE_TYPE_FP16: return launch_as<__half>(p, st);
    default: return launch_as<Bf16>(p, st);
  }
}

}  // namespace
}  // namespace tone

using namespace tone;

extern "C" {

int tone_token_scores(int device, const void* x, int type, int64_t stride, int64_t x_rows, const int64_t* rows, int64_t n,
                      int vocab, const int32_t* tokens, int k, float* logprob, float* entropy, int32_t* rank,
                      float* top_logprob, int32_t* top_ids, void* stream) {
  const char* what = "tone_token_scores";
  if (n < 0 || x_rows < 0 || vocab <= 0 || vocab > (1 << 24)) return refuse(what, "n, x_rows or vocab out of range");
  if (!known_type(type)) return refuse(what, "unknown element type");
  if (k < 0 || k > TONE_SCORES_MAX_K || k > vocab) return refuse(what, "k must be in 0 .. min(vocab, TONE_SCORES_MAX_K)");
  if (n == 0) return TONE_OK;
  if ((!x && x_rows) || !entropy || (k && (!top_logprob || !top_ids))) return refuse(what, "null pointer");
  if (tokens && (!logprob || !rank)) return refuse(what, "tokens without logprob or rank");
  if (!rows && x_rows < n) return refuse(what, "fewer rows in x than outputs");
  if (stride < vocab && x_rows > 1) return refuse(what, "row stride < vocab");
  if (!aligned(x, type)) return refuse(what, "x not aligned to its element type");
  if (n > kMaxThreads / (vocab <= 64 ? 8 : 64) - 32) return refuse(what, "too many rows for one launch");
  ScoreArgs p{x, stride, x_rows, rows, n, vocab, k, tokens, tokens ? logprob : nullptr, entropy, tokens ? rank : nullptr,
              top_logprob, top_ids};
  return launch_on(device, what, [&] { return launch_scores(p, type, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
