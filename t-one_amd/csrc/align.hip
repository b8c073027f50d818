// CTC alignment of given token sequences.  A sequence of L tokens is the chain of 2L + 1 states blank, token 0, blank, ...,
// token L - 1, blank; a path holds one state per frame, starts in state 0 or 1, stays, moves on by one, or by two over the
// blank between two different tokens, and ends in one of the last two.  With e_t(s) the frame's log probability of the
// state's label
//   best_t(s)  = max(best_{t-1}(s), best_{t-1}(s - 1), best_{t-1}(s - 2) where allowed) + e_t(s)
//   total_t(s) = the same with log-sum-exp
// The first of equals is taken in that order, and the last blank before the last token at the end.  The sums are held in
// 64 bits: a minute of frames adds up 2000 terms, the paths' difference may be one rounding of a term, and the sequence
// of additions is the definition's, so the path is reproducible bit for bit.
//
// The recurrence is a chain of frame_lens dependent steps, so its latency is what counts.  The states live in the registers
// of W waves, R consecutive ones per lane: a step moves one 64-bit value from lane to lane (DPP) and needs no LDS and no
// barrier.  With W > 1 the waves' ranges overlap: a wave's first HL lanes repeat the last ones of the wave below, whose
// values they lack go wrong by at most two states per frame from the left edge on, and are set right from that wave through
// LDS every 32 frames.  The frames' log probabilities are staged in LDS some frames ahead, the columns being the vocabulary,
// or only the sequence's own labels where those are fewer.  Which predecessor was taken is one bit (blank) or two (token)
// per state, F frames of a lane to a word of the workspace; the path is read back by one wave, a lane's word at a time
// (v_readlane) with the state in scalar registers, so no load waits for the state it belongs to.
//
// The sum over paths runs in a workgroup of its own, beside the one that finds the best path.  Each state is a 32-bit mantissa
// and a 32-bit exponent of 2 (never a logarithm: no exp and log per state and frame, and no underflow, however unlikely a
// prefix is): three terms aligned to the largest exponent, added, times the label's probability, itself mantissa and exponent.
#include "scoring.h"

#include <algorithm>

namespace tone {
namespace {

struct AlignArgs {
  const void* x;                        // frame (b, t) at b * batch_stride + t * stride, or rows[b][t] * stride
  int type;
  int64_t stride, batch_stride, x_rows;
  const int64_t* rows;
  int batch, frames, vocab, blank;
  const int32_t* tokens;                // [batch][most]
  int most;
  const int32_t *token_lens, *frame_lens;
  float *score, *total;                 // total: or nullptr
  int32_t *labels, *spans;              // [batch][frames], [batch][most][2]
  uint32_t* words;                      // [batch][groups][W][64]
  int columns, direct;                  // columns staged per frame; direct: column = label, else 0 = blank, 1 + i = token i
  int ahead;                            // frames per stage
};

constexpr float kClosed = 6e4f;         // entries of this size and more (masks of lowest values) count as -inf
constexpr int kZero = -(1 << 30);       // exponents of probability 0 end here ...
constexpr int kShut = kZero / 2;        // ... after a factor of 0; what passes one stays below kZero / 4 and is taken for 0
constexpr int kRefresh = 32;            // frames between two refreshes of the waves' overlap
constexpr int kStage = 8;               // loads of the next stage a lane has in flight during a stage

template <int W_, int R_>
struct Shape {
  static constexpr int W = W_, R = R_;
  static constexpr int HL = W > 1 ? (2 * kRefresh + R - 1) / R : 0;   // lanes that repeat the wave below
  static constexpr int N = (64 - HL) * R;                              // states a wave adds
  static constexpr int kStates = (W - 1) * N + 64 * R;
  static constexpr int kBits = R / 2 * 3;
  static constexpr int F = 32 / kBits;                                 // frames per word
};

__device__ __forceinline__ double shift_in(double v, double edge) {   // lane i: lane i - 1's value, lane 0: edge
  const int64_t a = __double_as_longlong(v), e = __double_as_longlong(edge);
  const int lo = __builtin_amdgcn_update_dpp((int)e, (int)a, 0x138, 0xf, 0xf, false);   // wave_shr 1
  const int hi = __builtin_amdgcn_update_dpp((int)(e >> 32), (int)(a >> 32), 0x138, 0xf, 0xf, false);
  return __longlong_as_double(((int64_t)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ int shift_in(int v, int edge) { return __builtin_amdgcn_update_dpp(edge, v, 0x138, 0xf, 0xf, false); }
__device__ __forceinline__ float shift_in(float v, float edge) {
  return __int_as_float(shift_in(__float_as_int(v), __float_as_int(edge)));
}

// the larger of two numbers that are no NaN (fmax puts a quieting v_max in front of each operand)
__device__ __forceinline__ double larger(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// one bit more at the low end: word + word + carry, one v_addc behind the compare
__device__ __forceinline__ void push(uint32_t& word, bool bit) {
  unsigned out;
  word = __builtin_addc(word, word, (unsigned)bit, &out);
}

// a probability e^v as mantissa in [0.7, 1.42) and exponent: v log2 e in two terms, so the mantissa is off by a few 2^-24
// however large |v| is
struct Prob {
  float m;
  int e;
};
__device__ __forceinline__ Prob prob_of(float v) {
  if (v == -INFINITY) return {1.f, kShut};
  const float n = rintf(v * 1.44269502f);
  const float f = fmaf(v, 1.92596299e-8f, fmaf(v, 1.44269502f, -n));
  return {__builtin_amdgcn_exp2f(f), (int)n};
}

// The frames of a sequence, staged `ahead` at a time: stage() issues the loads of the next ones, put() writes what came.
template <class SH, bool SUM>
struct Frames {
  const AlignArgs p;
  const int b, n, lane, wave;
  const int32_t* tok;
  char* buf;                            // [2][ahead][columns + 1]: the last column is closed
  int64_t row, row_after;               // lane f: row of frame f of the stage under way / of the one behind it
  float got[kStage];

  static constexpr int kEntry = SUM ? 8 : 4;

  __device__ Frames(const AlignArgs& p_, int b_, int n_, char* buf_)
      : p(p_), b(b_), n(n_), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), tok(p_.tokens + (int64_t)b_ * p_.most), buf(buf_) {}

  __device__ __forceinline__ int per_frame() const { return (p.columns + 1) * kEntry; }
  __device__ __forceinline__ char* at(int stage, int f) const { return buf + ((stage & 1) * p.ahead + f) * per_frame(); }
  __device__ __forceinline__ int column(int i, int len) const {        // of token i of the sequence
    if (i >= len) return 0;                                            // a state behind the last: anything
    const int t = tok[i];
    return t < 0 || t >= p.vocab || t == p.blank ? p.columns : p.direct ? t : i + 1;
  }
  __device__ __forceinline__ int blank_column() const { return p.direct ? p.blank : 0; }
  __device__ __forceinline__ void rows_from(int t0) {
    row_after = -1;
    if (p.rows && lane < p.ahead && t0 + lane < n) row_after = p.rows[(int64_t)b * p.frames + t0 + lane];
  }
  __device__ __forceinline__ float value(int64_t off) const {
    float v;
    if (p.type == TONE_TYPE_FP32) v = load_elem(static_cast<const float*>(p.x) + off);
    else if (p.type == TONE_TYPE_FP16) v = load_elem(static_cast<const __half*>(p.x) + off);
    else v = load_elem(static_cast<const Bf16*>(p.x) + off);
    return v;
  }
  // The wave's part of a stage is the frames wave, wave + W, ... in blocks of 64 columns (the closed one among them), item by
  // item in that order.  The first kStage items are under way during the stage before; only wide frames have more.
  __device__ __forceinline__ float item(int t0, int f, int c0) const {
    const int c = c0 + lane;
    int64_t off = (int64_t)b * p.batch_stride + (int64_t)(t0 + f) * p.stride;
    bool here = c < p.columns;
    if (p.rows) {
      const int64_t r = ((int64_t)__builtin_amdgcn_readlane((int)(row >> 32), f) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)row, f);
      here = here && r >= 0 && r < p.x_rows;
      off = r * p.stride;
    }
    if (!here) return -INFINITY;
    const int label = p.direct ? c : c == 0 ? p.blank : tok[c - 1];
    return label >= 0 && label < p.vocab ? value(off + label) : -INFINITY;
  }
  __device__ __forceinline__ void write(int stage, int f, int c0, float v) const {
    const int c = c0 + lane;
    v = fabsf(v) < kClosed ? v : -INFINITY;
    if (c > p.columns) return;
    if constexpr (SUM) reinterpret_cast<Prob*>(at(stage, f))[c] = prob_of(v);
    else reinterpret_cast<float*>(at(stage, f))[c] = v;
  }
  __device__ __forceinline__ void load(int t0) {
    row = row_after;
    rows_from(t0 + p.ahead);
    int f = wave, c0 = 0;
#pragma unroll
    for (int j = 0; j < kStage; ++j) {
      if (f < p.ahead && t0 + f < n) got[j] = item(t0, f, c0);
      next(f, c0);
    }
  }
  __device__ __forceinline__ void put(int stage, int t0) {
    int f = wave, c0 = 0;
#pragma unroll
    for (int j = 0; j < kStage; ++j) {
      if (f < p.ahead && t0 + f < n) write(stage, f, c0, got[j]);
      next(f, c0);
    }
    while (f < p.ahead && t0 + f < n) {
      write(stage, f, c0, item(t0, f, c0));
      next(f, c0);
    }
  }
  __device__ __forceinline__ void next(int& f, int& c0) const {
    c0 += 64;
    if (c0 > p.columns) {
      c0 = 0;
      f += SH::W;
    }
  }
};

// one frame of the best path: the lane's states to the next frame's, highest first (each needs the ones below as they were)
template <class SH>
struct BestStep {
  double a[SH::R];
  double closed[SH::R / 2];             // 0 where token q may follow the token before it directly, else -inf
  int col[SH::R / 2];                   // byte offsets
  uint32_t word;

  __device__ __forceinline__ void step(const char* frame, int blank, double edge) {
    const double eb = *reinterpret_cast<const float*>(frame + blank);
    double et[SH::R / 2];
#pragma unroll
    for (int q = 0; q < SH::R / 2; ++q) et[q] = *reinterpret_cast<const float*>(frame + col[q]);
    const double below = shift_in(a[SH::R - 1], edge);
#pragma unroll
    for (int q = SH::R / 2 - 1; q >= 0; --q) {
      const double stay = a[2 * q + 1], one = a[2 * q], two = (q ? a[q ? 2 * q - 1 : 0] : below) + closed[q];
      const double m = larger(stay, one);
      push(word, one > stay);
      push(word, two > m);
      a[2 * q + 1] = larger(m, two) + et[q];
      const double from = q ? a[q ? 2 * q - 1 : 0] : below;
      push(word, from > one);
      a[2 * q] = larger(one, from) + eb;
    }
  }
};

// the same for the sum over paths
template <class SH>
struct SumStep {
  float m[SH::R];
  int e[SH::R];
  int closed[SH::R / 2];                // 0 or kShut
  int col[SH::R / 2];

  __device__ __forceinline__ void step(const char* frame, int blank, float edge_m, int edge_e) {
    const Prob pb = *reinterpret_cast<const Prob*>(frame + blank);
    Prob pt[SH::R / 2];
#pragma unroll
    for (int q = 0; q < SH::R / 2; ++q) pt[q] = *reinterpret_cast<const Prob*>(frame + col[q]);
    const float below_m = shift_in(m[SH::R - 1], edge_m);
    const int below_e = shift_in(e[SH::R - 1], edge_e);
#pragma unroll
    for (int q = SH::R / 2 - 1; q >= 0; --q) {
      const float fm = q ? m[q ? 2 * q - 1 : 0] : below_m;
      const int fe = q ? e[q ? 2 * q - 1 : 0] : below_e;
      {
        const int e2 = fe + closed[q], hi = max(max(e[2 * q + 1], e[2 * q]), e2);
        const float sum = (ldexpf(m[2 * q + 1], e[2 * q + 1] - hi) + ldexpf(m[2 * q], e[2 * q] - hi)) + ldexpf(fm, e2 - hi);
        m[2 * q + 1] = sum * pt[q].m;
        e[2 * q + 1] = max(hi + pt[q].e, kZero);
      }
      const int hi = max(e[2 * q], fe);
      m[2 * q] = (ldexpf(m[2 * q], e[2 * q] - hi) + ldexpf(fm, fe - hi)) * pb.m;
      e[2 * q] = max(hi + pb.e, kZero);
    }
  }
  // a frame multiplies a mantissa by 0.7 to 4.3, so 32 frames stay far inside fp32
  __device__ __forceinline__ void renormalize() {
#pragma unroll
    for (int r = 0; r < SH::R; ++r) {
      const int x = __builtin_amdgcn_frexp_expf(m[r]);
      m[r] = __builtin_amdgcn_frexp_mantf(m[r]);
      e[r] = max(e[r] + x, kZero);
    }
  }
};

// Runs `step(stage, frame)` for all frames of the sequence: stages the frames, and refreshes the overlap of the waves.
template <class SH, bool SUM, class Step, class Refresh>
__device__ __forceinline__ void over_frames(Frames<SH, SUM>& fr, bool active, Step&& step, Refresh&& refresh) {
  const int n = fr.n, ahead = fr.p.ahead;
  fr.rows_from(0);
  fr.load(0);
  fr.put(0, 0);
  __syncthreads();
  for (int t0 = 0, stage = 0; t0 < n; t0 += ahead, ++stage) {
    const bool more = t0 + ahead < n;
    if (more) fr.load(t0 + ahead);
    const int m = min(ahead, n - t0);
    if (active)
      for (int f = 0; f < m; ++f) step(stage, f, t0 + f);
    if (more) {
      fr.put(stage + 1, t0 + ahead);
      const bool now = ((t0 + ahead) & (kRefresh - 1)) == 0;
      if (now) refresh(true, ((t0 + ahead) / kRefresh) & 1);
      __syncthreads();
      if (now) refresh(false, ((t0 + ahead) / kRefresh) & 1);
    }
  }
}

template <class SH>
__device__ void best_path(const AlignArgs& p, int b, int L, int n, char* lds) {
  constexpr int W = SH::W, R = SH::R, HL = SH::HL;
  __shared__ double s_end[2];
  __shared__ double s_over[2][W][W > 1 ? HL * R : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), base = wave * SH::N + lane * R;
  const bool active = wave * SH::N <= 2 * L;
  const int64_t groups = (p.frames + SH::F - 1) / SH::F;
  uint32_t* words = p.words + (int64_t)b * groups * W * 64;
  int32_t* labels = p.labels + (int64_t)b * p.frames;
  int32_t* spans = p.spans + (int64_t)b * p.most * 2;
  const int32_t* tok = p.tokens + (int64_t)b * p.most;
  if (threadIdx.x < 2) s_end[threadIdx.x] = n == 0 && L == 0 && threadIdx.x == 0 ? 0.0 : -INFINITY;   // [0]: last blank, [1]: last token
  if (n > 0) {
    Frames<SH, false> fr(p, b, n, lds);
    BestStep<SH> st;
    st.word = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) st.a[r] = -INFINITY;
#pragma unroll
    for (int q = 0; q < R / 2; ++q) {
      const int i = (base >> 1) + q;
      st.col[q] = fr.column(i, L) * 4;
      st.closed[q] = i > 0 && i < L && tok[i] == tok[i - 1] ? -INFINITY : 0.0;
    }
    const int blank = fr.blank_column() * 4;
    int held = 0;
    uint32_t* out = words + wave * 64 + lane;
    // before the first frame: a state in front of the first, from which blank 0 (one on) and token 0 (two on) are reached
    double edge = wave == 0 ? 0.0 : -INFINITY;
    over_frames<SH, false>(
        fr, active,
        [&](int stage, int f, int t) {
          st.step(fr.at(stage, f), blank, edge);
          edge = -INFINITY;
          if (++held == SH::F || t == n - 1) {
            *out = st.word;
            out += W * 64;
            st.word = 0;
            held = 0;
          }
        },
        [&](bool write, int half) {
          if constexpr (W > 1) {
            if (write) {
              if (lane >= 64 - HL)
#pragma unroll
                for (int r = 0; r < R; ++r) s_over[half][wave][(lane - (64 - HL)) * R + r] = st.a[r];
            } else if (wave > 0 && lane < HL) {
#pragma unroll
              for (int r = 0; r < R; ++r) st.a[r] = s_over[half][wave - 1][lane * R + r];
            }
          }
        });
    __syncthreads();                     // s_end's first values are in place
    if (active && (wave == 0 || lane >= HL)) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (base + r == 2 * L) s_end[0] = st.a[r];
        if (base + r == 2 * L - 1) s_end[1] = st.a[r];
      }
    }
    __threadfence_block();
  }
  __syncthreads();
  const double at_blank = s_end[0], at_token = s_end[1], score = fmax(at_blank, at_token);
  const bool alive = score > -INFINITY;
  for (int t = (alive ? n : 0) + threadIdx.x; t < p.frames; t += 64 * W) labels[t] = -1;
  for (int i = (alive ? 2 * L : 0) + threadIdx.x; i < 2 * p.most; i += 64 * W) spans[i] = -1;
  if (threadIdx.x == 0) p.score[b] = (float)score;
  if (!alive || n == 0 || wave > 0) return;
  // the path from its end: the state is uniform, wave w_'s lane l_'s state r_
  int s = at_token > at_blank ? 2 * L - 1 : 2 * L, w_ = 0, l_, r_;
  {
    int rest = s;
    while (rest >= 64 * R) {
      rest -= SH::N;
      ++w_;
    }
    l_ = rest / R;
    r_ = rest - l_ * R;
  }
  int t = n - 1, path = 0, above = -1;
  constexpr int kAhead = 8;
  uint32_t cur[kAhead][W], nxt[kAhead][W];
  auto fetch = [&](uint32_t (&to)[kAhead][W], int g0) {     // groups g0, g0 - 1, ...
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int w = 0; w < W; ++w) to[i][w] = g0 - i >= 0 ? words[((int64_t)(g0 - i) * W + w) * 64 + lane] : 0;
  };
  int g = t / SH::F;
  fetch(cur, g);
  while (g >= 0) {
    fetch(nxt, g - kAhead);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (g - i < 0) continue;
      const int first = (g - i) * SH::F;
      int at = 0;                        // bits of the frames behind t in the word
      for (; t >= first; --t, at += SH::kBits) {
        uint32_t word = __builtin_amdgcn_readlane(cur[i][0], l_);
#pragma unroll
        for (int w = 1; w < W; ++w)
          if (w_ == w) word = __builtin_amdgcn_readlane(cur[i][w], l_);
        const uint32_t bits = word >> (at + 3 * (r_ >> 1));
        const int how = r_ & 1 ? (bits & 2 ? 2 : (bits >> 2) & 1) : bits & 1;
        path = lane == (t & 63) ? s : path;
        const int now = s;
        s -= how;
        r_ -= how;
        if (r_ < 0) {
          r_ += R;
          --l_;
          if (W > 1 && w_ > 0 && l_ < HL) {
            --w_;
            l_ += 64 - HL;
          }
        }
        if ((t & 63) == 0) {             // frames t .. t + 63 are known, and the state before them
          const int mine = t + lane, before = t ? s : -1;
          const int prev = shift_in(path, before);
          int next = __shfl_down(path, 1);
          if (lane == 63) next = above;
          if (mine == n - 1) next = -1;
          if (mine < n) {
            labels[mine] = path & 1 ? tok[path >> 1] : p.blank;
            if ((path & 1) && prev != path) spans[path & ~1] = mine;
            if ((path & 1) && next != path) spans[path | 1] = mine + 1;
          }
          above = now;
        }
      }
    }
    g -= kAhead;
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int w = 0; w < W; ++w) cur[i][w] = nxt[i][w];
  }
}

template <class SH>
__device__ void all_paths(const AlignArgs& p, int b, int L, int n, char* lds) {
  constexpr int W = SH::W, R = SH::R, HL = SH::HL;
  __shared__ float s_end_m[2];
  __shared__ int s_end_e[2];
  __shared__ float s_over_m[2][W][W > 1 ? HL * R : 1];
  __shared__ int s_over_e[2][W][W > 1 ? HL * R : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), base = wave * SH::N + lane * R;
  const bool active = wave * SH::N <= 2 * L;
  const int32_t* tok = p.tokens + (int64_t)b * p.most;
  if (n == 0) {
    if (threadIdx.x == 0) p.total[b] = L == 0 ? 0.f : -INFINITY;
    return;
  }
  if (threadIdx.x < 2) {
    s_end_m[threadIdx.x] = 0.f;
    s_end_e[threadIdx.x] = kZero;
  }
  Frames<SH, true> fr(p, b, n, lds);
  SumStep<SH> st;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st.m[r] = 1.f;
    st.e[r] = kZero;
  }
#pragma unroll
  for (int q = 0; q < R / 2; ++q) {
    const int i = (base >> 1) + q;
    st.col[q] = fr.column(i, L) * 8;
    st.closed[q] = i > 0 && i < L && tok[i] == tok[i - 1] ? kShut : 0;
  }
  const int blank = fr.blank_column() * 8;
  int edge = wave == 0 ? 0 : kZero;
  over_frames<SH, true>(
      fr, active,
      [&](int stage, int f, int t) {
        st.step(fr.at(stage, f), blank, 1.f, edge);
        edge = kZero;
        if ((t & (kRefresh - 1)) == kRefresh - 1) st.renormalize();
      },
      [&](bool write, int half) {
        if constexpr (W > 1) {
          if (write) {
            if (lane >= 64 - HL)
#pragma unroll
              for (int r = 0; r < R; ++r) {
                s_over_m[half][wave][(lane - (64 - HL)) * R + r] = st.m[r];
                s_over_e[half][wave][(lane - (64 - HL)) * R + r] = st.e[r];
              }
          } else if (wave > 0 && lane < HL) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
              st.m[r] = s_over_m[half][wave - 1][lane * R + r];
              st.e[r] = s_over_e[half][wave - 1][lane * R + r];
            }
          }
        }
      });
  __syncthreads();
  if (active && (wave == 0 || lane >= HL)) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      for (int i = 0; i < 2; ++i)
        if (base + r == 2 * L - i) {
          s_end_m[i] = st.m[r];
          s_end_e[i] = st.e[r];
        }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int hi = max(s_end_e[0], s_end_e[1]);
    const float sum = ldexpf(s_end_m[0], s_end_e[0] - hi) + ldexpf(s_end_m[1], s_end_e[1] - hi);
    p.total[b] = hi < kZero / 4 ? -INFINITY : (float)((double)hi * 0.693147180559945309 + (double)logf(sum));
  }
}

// workgroup b: the best path of sequence b; batch + b: the sum of all
template <int W, int R>
__global__ void __launch_bounds__(64 * W) align_kernel(AlignArgs p) {
  extern __shared__ char lds[];
  using SH = Shape<W, R>;
  const bool sum = (int)blockIdx.x >= p.batch;
  const int b = sum ? blockIdx.x - p.batch : blockIdx.x;
  const int L = min(max(p.token_lens[b], 0), p.most), n = min(max(p.frame_lens[b], 0), p.frames);
  if (sum) all_paths<SH>(p, b, L, n, lds);
  else best_path<SH>(p, b, L, n, lds);
}

template <int W, int R>
hipError_t launch_as(AlignArgs p, hipStream_t st) {
  p.direct = p.vocab <= p.most + 1;
  p.columns = p.direct ? p.vocab : p.most + 1;
  // frames per stage: as many as kStage loads per lane hold, a divisor of the refresh interval
  p.ahead = kRefresh;
  while (p.ahead > W && p.ahead / W * ((p.columns + 64) / 64) > kStage) p.ahead /= 2;
  const size_t lds = (size_t)2 * p.ahead * (p.columns + 1) * (p.total ? 8 : 4);
  auto* fn = align_kernel<W, R>;
  if (lds > 32 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3(p.total ? 2 * p.batch : p.batch), dim3(64 * W), lds, st, p);
  return hipGetLastError();
}

// The fewest states per lane that hold the sequences: a step's time grows with them (see the table in launch_align).
template <class F>
auto by_tokens(int most, F&& f) {
  const int states = 2 * most + 1;
  if (states <= Shape<1, 2>::kStates) return f(Shape<1, 2>{});
  if (states <= Shape<4, 2>::kStates) return f(Shape<4, 2>{});
  if (states <= Shape<4, 4>::kStates) return f(Shape<4, 4>{});
  if (states <= Shape<4, 8>::kStates) return f(Shape<4, 8>{});
  return f(Shape<4, 18>{});
}
static_assert(Shape<4, 18>::kStates >= 2 * TONE_ALIGN_MAX_TOKENS + 1, "the longest sequences fit");

hipError_t launch_align(const AlignArgs& p, hipStream_t st) {
  return by_tokens(p.most, [&](auto sh) { return launch_as<decltype(sh)::W, decltype(sh)::R>(p, st); });
}

int64_t align_workspace(int batch, int frames, int most) {
  return by_tokens(most, [&](auto sh) -> int64_t {
    using SH = decltype(sh);
    return (int64_t)batch * ((frames + SH::F - 1) / SH::F) * SH::W * 64 * 4;
  });
}

}  // namespace
}  // namespace tone

using namespace tone;

extern "C" {

int64_t tone_ctc_align_workspace(int batch, int frames, int tokens) {
  if (batch < 0 || frames < 0 || tokens < 0 || tokens > TONE_ALIGN_MAX_TOKENS) return -1;
  return align_workspace(batch, frames, tokens);
}

int tone_ctc_align(int device, const void* x, int type, int64_t stride, int64_t batch_stride, int64_t x_rows,
                   const int64_t* rows, int batch, int frames, int vocab, int blank, const int32_t* tokens, int max_tokens,
                   const int32_t* token_lens, const int32_t* frame_lens, float* score, float* total, int32_t* labels,
                   int32_t* spans, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "tone_ctc_align";
  if (batch < 0 || frames < 0 || x_rows < 0 || vocab <= 0 || vocab > (1 << 24))
    return refuse(what, "batch, frames, x_rows or vocab out of range");
  if (max_tokens < 0 || max_tokens > TONE_ALIGN_MAX_TOKENS) return refuse(what, "max_tokens must be in 0 .. TONE_ALIGN_MAX_TOKENS");
  if (!known_type(type)) return refuse(what, "unknown element type");
  if (blank < 0 || blank >= vocab) return refuse(what, "blank outside the vocabulary");
  if (batch == 0) return TONE_OK;
  if ((!x && frames && (!rows || x_rows)) || !token_lens || !frame_lens || !score || (frames && !labels) || (max_tokens && (!tokens || !spans)))
    return refuse(what, "null pointer");
  if (!aligned(x, type)) return refuse(what, "x not aligned to its element type");
  const int64_t need = tone_ctc_align_workspace(batch, frames, max_tokens);
  if (workspace_bytes < need || (need && !workspace)) return refuse(what, "workspace smaller than tone_ctc_align_workspace");
  AlignArgs p{x, type, stride, batch_stride, x_rows, rows, batch, frames, vocab, blank, tokens, max_tokens, token_lens, frame_lens,
              score, total, labels, spans, static_cast<uint32_t*>(workspace), 0, 0, 0};
  return launch_on(device, what, [&] { return launch_align(p, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
