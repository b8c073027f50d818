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
// LDS every 32 frames (half of that halves the overlap, but a refresh costs half a microsecond).  Waves of their own stage
// the frames' log probabilities in LDS some frames ahead, the columns being the vocabulary, or only the sequence's own labels
// where those are fewer.
//
// Which predecessor was taken is one bit (blank) or two (token) per state, F frames of a lane to a word of the workspace.
// Each state also carries where its path was 32 frames ago, so the path is first found at every 32nd frame, one look-up
// each, and then between them by all waves at once: a wave loads the words of its 32 frames and walks them with the state in
// scalar registers (v_readlane), so no load waits for the state it belongs to.
//
// The sum over paths runs in a workgroup of its own, beside the one that finds the best path.  Each state is a 64-bit mantissa
// and a 32-bit exponent of 2 (never a logarithm: no exp and log per state and frame, and no underflow, however unlikely a
// prefix is): three terms aligned to the largest exponent, added, times the label's probability.  That one is 1 + d times a
// power of 2 with d in 32 bits, which is off in proportion to the label's log probability and not to 1: rows that are almost
// sure of their label add up to a total close to 0, and it is right in proportion as well (in 32 bits throughout the same took
// 5 to 8 % less time, and a total of -1e-2 was off by 0.3 %, one of -1e-6 by all of it).
//
// What bounds it is the issue of one wave's instructions, one after the other at some 2.4 ns each: 91 ns per frame with two
// states per lane and one wave (187 frames and 43 tokens with the trace: 24.5 us), 97 with four waves (with the sum 102), 131
// with four states per lane, 171 with eight waves of those (48 phrases of 2000 frames and 700 tokens: 350 us, with their sums
// 370, 13 MB read).  From 256 workgroups on two of them share a CU: 128 hypotheses of 400 frames and 110 tokens with their sums
// take 48 us as one does, 192 take 61.
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
  uint32_t* words;                      // [batch][groups][W][64], groups of F frames
  uint16_t* came;                       // [batch][legs][states], legs of kLeg frames: the state at the frame before the leg
  int columns, direct;                  // columns staged per frame: the labels (direct), or 0 = blank, 1 + i = token i
  int ahead;                            // frames per stage
};

constexpr float kClosed = 6e4f;         // entries of this size and more (masks of lowest values) count as -inf
constexpr int kLeg = 32;                // frames between two refreshes of the waves' overlap, and two marks of the path
constexpr int kLoaders = 4;             // waves that stage the frames
constexpr int kBatch = 8;               // loads a loader lane has in flight
// Probability 0 is a mantissa of 0, which no later factor changes.  Its exponent has to stay below every other one, as the
// largest of a sum's exponents is what its terms are aligned to: a factor of 0 takes kShut off (adding saturates), and every
// 32 frames it is put to kZero.  Other exponents are held in [kLow, kHigh] there, what is below kLow becoming 0, and move by
// some 3 million (entries of 6e4) until the next time; kHigh + kShut lies far enough below kLow for that.
constexpr int kShut = -(1 << 30), kZero = -(1 << 30), kLow = -(1 << 28), kHigh = 1 << 29;

template <int W_, int R_>
struct Shape {
  static constexpr int W = W_, R = R_;
  static constexpr int HL = W > 1 ? 2 * kLeg / R : 0;   // lanes that repeat the wave below
  static constexpr int N = (64 - HL) * R;                    // states a wave adds
  static constexpr int kStates = (W - 1) * N + 64 * R;
  static constexpr int kBits = R / 2 * 3;
  static constexpr int F = R == 2 ? 8 : R == 4 ? 4 : 2;      // frames per word
  static_assert(F * kBits <= 32 && kLeg % F == 0 && 2 * kLeg % R == 0, "whole words and lanes");
  static_assert(W == 1 || N >= 2 * kLeg - 2, "a leg's path touches two waves at most");
  // which lane holds a wave's state i < 128 R
  __device__ static __forceinline__ int lane_of(int i) { return R == 2 ? i >> 1 : R == 4 ? i >> 2 : i >> 3; }
  static_assert(R == 2 || R == 4 || R == 8, "lane_of");
};

// a barrier for what the waves pass on in LDS: __syncthreads would also wait for the loads and the word stores under way
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// lane i: lane i - 1's value (wave_shr 1); lane 0 keeps `edge`'s
__device__ __forceinline__ int shift_in(int v, int edge) { return __builtin_amdgcn_update_dpp(edge, v, 0x138, 0xf, 0xf, false); }
__device__ __forceinline__ double shift_in(double v, double edge) {
  return __hiloint2double(shift_in(__double2hiint(v), __double2hiint(edge)), shift_in(__double2loint(v), __double2loint(edge)));
}

// a probability e^v as (1 + d) 2^e, 1 + d in [0.7, 1.42): v less n ln 2 in two terms (the reduction of Cody and Waite; the first
// is v itself where n is 0), d by the series of e^r - 1, whose first term left out is below 2^-25 of it.  d is off by two roundings
// at most, so the factor's logarithm by less than 2^-21 |v|, whatever v is.
struct Prob {
  float d;
  int e;
};
__device__ __forceinline__ Prob prob_of(float v) {
  if (v == -INFINITY) return {-1.f, kShut};
  const float n = rintf(v * 1.44269504f);
  const float r = fmaf(n, 1.90465430e-9f, fmaf(n, -0.693147182f, v));      // ln 2 = 0.693147182 - 1.90465430e-9
  float c = 1.f / 5040;
  c = fmaf(c, r, 1.f / 720);
  c = fmaf(c, r, 1.f / 120);
  c = fmaf(c, r, 1.f / 24);
  c = fmaf(c, r, 1.f / 6);
  c = fmaf(c, r, 0.5f);
  return {fmaf(r * r, c, r), (int)n};
}

// What is staged: [2][columns + 1][ahead + 2] entries of 8 bytes, a double (best path) or a Prob (sum); the last column is
// closed.  A column's frames lie together, so a lane reads two of them at once and the frame is an offset in the instruction;
// the two entries of padding spread the columns over the banks.
struct Frames {
  const AlignArgs p;
  const int b, n;
  const int32_t* tok;
  char* buf;

  __device__ Frames(const AlignArgs& p_, int b_, int n_, char* buf_)
      : p(p_), b(b_), n(n_), tok(p_.tokens + (int64_t)b_ * p_.most), buf(buf_) {}

  __device__ __forceinline__ int pitch() const { return (p.ahead + 2) * 8; }
  __device__ __forceinline__ char* stage(int i) const { return buf + (i & 1) * (p.columns + 1) * pitch(); }
  __device__ __forceinline__ int column(int i, int len) const {        // byte offset of token i of the sequence
    if (i >= len) return 0;                                            // a state behind the last: anything
    const int t = tok[i];
    return pitch() * (t < 0 || t >= p.vocab || t == p.blank ? p.columns : p.direct ? t : i + 1);
  }
  __device__ __forceinline__ int blank_column() const { return p.direct ? pitch() * p.blank : 0; }
};

// A loader wave: frames loader, loader + kLoaders, ... of each stage, 64 columns at a time.  The data of the stage after the
// next and the rows of the one after that are loaded a stage ahead of their use, so a stage waits for neither; only frames
// of many columns have more than kBatch loads, and those behind are loaded as they are written.
template <bool SUM>
__device__ __forceinline__ void load_frames(const Frames& fr, int loader, int lane) {
  const AlignArgs& p = fr.p;
  const int n = fr.n, ahead = p.ahead, per = max(1, ahead / kLoaders), shift = 31 - __builtin_clz(per), items = (p.columns / 64 + 1) * per;
  const int type = p.type, size = type == TONE_TYPE_FP32 ? 4 : 2, pitch = fr.pitch();
  const char* x = static_cast<const char*>(p.x) + (p.rows ? 0 : (int64_t)fr.b * p.batch_stride * size);
  const int64_t* rows = p.rows ? p.rows + (int64_t)fr.b * p.frames : nullptr;
  const int64_t stride = p.stride * size, x_rows = rows ? p.x_rows : INT64_MAX;
  int64_t row1 = -1, row2 = -1, row3 = -1;       // lane f: row of frame f, one, two and three stages on
  uint32_t raw_a[kBatch], raw_b[kBatch];
  bool have_a[kBatch], have_b[kBatch];
  auto frame = [&](int i) { return loader + kLoaders * (i & (per - 1)); };
  // byte offset of column c in a row; -1 where it is none
  auto offset = [&](int c) {
    if (c >= p.columns) return -1;
    const int label = p.direct ? c : c ? fr.tok[c - 1] : p.blank;
    return label >= 0 && label < p.vocab ? label * size : -1;
  };
  const int offset0 = offset(lane);
  // the frame's row is uniform: a scalar base, and what the lane adds (columns that are none load the row's first entry)
  auto load = [&](int64_t row, int i, int off, uint32_t& to) -> bool {
    const int f = frame(i);
    const int64_t r = ((int64_t)__builtin_amdgcn_readlane((int)(row >> 32), f) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)row, f);
    if (r < 0 || r >= x_rows) return false;
    const char* base = x + r * stride;
    const uint32_t o = max(off, 0);
    if (size == 4) to = *reinterpret_cast<const uint32_t*>(base + o);
    else to = *reinterpret_cast<const uint16_t*>(base + o);
    return true;
  };
  auto write = [&](int stage, int i, int off, uint32_t bits, bool ok) {
    const int c = (i >> shift) * 64 + lane;
    float v = __uint_as_float(type == TONE_TYPE_BF16 ? bits << 16 : bits);
    if (type == TONE_TYPE_FP16) v = __half2float(__ushort_as_half((uint16_t)bits));
    if (!(fabsf(v) < kClosed) || off < 0 || !ok) v = -INFINITY;
    if (c > p.columns) return;
    char* to = fr.stage(stage) + c * pitch + 8 * frame(i);
    if constexpr (SUM) *reinterpret_cast<Prob*>(to) = prob_of(v);
    else *reinterpret_cast<double*>(to) = v;
  };
  // one stage: loads of the one after the next issued, then the next one written from the loads issued a stage ago
  auto step = [&](int t0, int stage, uint32_t (&now)[kBatch], bool (&have)[kBatch], uint32_t (&later)[kBatch], bool (&have_later)[kBatch]) {
    row1 = row2;
    row2 = row3;
    row3 = -1;
    const int t = t0 + 3 * ahead + lane;
    if (lane < ahead && t < n) row3 = rows ? rows[t] : t;
    if (t0 + 2 * ahead >= 0) {
      const int m = min(n - (t0 + 2 * ahead), ahead);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        have_later[j] = false;
        if (j < items && frame(j) < m) have_later[j] = load(row2, j, j < per ? offset0 : offset((j >> shift) * 64 + lane), later[j]);
      }
    }
    if (t0 + ahead >= 0 && t0 + ahead < n) {
      const int m = min(n - (t0 + ahead), ahead);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (j < items && frame(j) < m) write(stage + 1, j, j < per ? offset0 : offset((j >> shift) * 64 + lane), now[j], have[j]);
      for (int i = kBatch; i < items; ++i)
        if (frame(i) < m) {
          const int off = offset((i >> shift) * 64 + lane);
          uint32_t bits = 0;
          const bool ok = load(row1, i, off, bits);
          write(stage + 1, i, off, bits, ok);
        }
    }
    if (t0 + ahead >= 0 && t0 + ahead < n) lds_barrier();      // as the stepping waves: before stage 0, and between stages
  };
  for (int t0 = -3 * ahead, stage = -3; t0 < n; t0 += 2 * ahead, stage += 2) {
    step(t0, stage, raw_a, have_a, raw_b, have_b);
    if (t0 + ahead < n) step(t0 + ahead, stage + 1, raw_b, have_b, raw_a, have_a);
  }
}

// The lane's states, and one frame: the highest first, since each needs the ones below it as they were.
template <class SH>
struct Best {
  static constexpr int Q = SH::R / 2;
  double a[SH::R];
  double below;                         // the state below the lane's first; lane 0: -inf
  int o[SH::R], below_o;                // the paths' states at the frame before the leg
  int col[Q];
  bool apart[Q];                        // token q may follow the token before it directly
  uint32_t word;

  struct Rows {                         // of two frames
    double2 blank, tok[Q];
  };
  struct Row {
    double blank, tok[Q];
    __device__ __forceinline__ Row(const Rows& r, int i) : blank(i ? r.blank.y : r.blank.x) {
#pragma unroll
      for (int q = 0; q < Q; ++q) tok[q] = i ? r.tok[q].y : r.tok[q].x;
    }
  };
  __device__ __forceinline__ void read(Rows& r, const char* frame, int blank) const {
    r.blank = *reinterpret_cast<const double2*>(frame + blank);
#pragma unroll
    for (int q = 0; q < Q; ++q) r.tok[q] = *reinterpret_cast<const double2*>(frame + col[q]);
  }
  __device__ __forceinline__ void clear(int base) {
#pragma unroll
    for (int i = 0; i < SH::R; ++i) a[i] = -INFINITY;
    below = -INFINITY;
    below_o = 0;
    word = 0;
    mark(base);
  }
  __device__ __forceinline__ void first(const Row& r, int base) {      // the first frame
    if (base == 0) {
      a[0] = r.blank;
      a[1] = r.tok[0];
    }
  }
  __device__ __forceinline__ void mark(int base) {
#pragma unroll
    for (int i = 0; i < SH::R; ++i) o[i] = base + i;
  }
  __device__ __forceinline__ void step(const Row& r) {
    below = shift_in(a[SH::R - 1], below);
    below_o = shift_in(o[SH::R - 1], below_o);
#pragma unroll
    for (int q = Q - 1; q >= 0; --q) {
      const double stay = a[2 * q + 1], one = a[2 * q], from = q ? a[q ? 2 * q - 1 : 0] : below;
      // not apart: a NaN, which no compare prefers and v_max_f64 passes over
      const double two = __hiloint2double(apart[q] ? __double2hiint(from) : 0x7ff80000, __double2loint(from));
      const int o_from = q ? o[q ? 2 * q - 1 : 0] : below_o;
      double m, token, blank;
      int o_token, o_blank;
      uint64_t c0, c1, c2;
      // one by hand: (a) v_max_f64 without the quieting of operands that fmax brings, (b) each compare's mask pushed into
      // the word by one add with carry, two instructions at least behind the compare as gfx950 demands of masks.  What a
      // DPP move reads next (o_token) is written three instructions before the end: two are demanded, and the compiler
      // does not look inside
      asm("v_cmp_gt_f64_e64 %[c1], %[one], %[stay]\n\t"
          "v_cmp_gt_f64_e64 %[c0], %[from], %[one]\n\t"
          "v_max_f64 %[m], %[stay], %[one]\n\t"
          "v_max_f64 %[blank], %[one], %[from]\n\t"
          "v_cmp_gt_f64_e64 %[c2], %[two], %[m]\n\t"
          "v_max_f64 %[token], %[m], %[two]\n\t"
          "v_cndmask_b32_e64 %[o_token], %[o_stay], %[o_one], %[c1]\n\t"
          "v_cndmask_b32_e64 %[o_blank], %[o_one], %[o_from], %[c0]\n\t"
          "v_cndmask_b32_e64 %[o_token], %[o_token], %[o_from], %[c2]\n\t"
          "v_addc_co_u32_e64 %[word], vcc, %[word], %[word], %[c1]\n\t"
          "v_addc_co_u32_e64 %[word], vcc, %[word], %[word], %[c2]\n\t"
          "v_addc_co_u32_e64 %[word], vcc, %[word], %[word], %[c0]"
          : [o_token] "=&v"(o_token), [o_blank] "=&v"(o_blank), [word] "+v"(word), [m] "=&v"(m), [blank] "=&v"(blank), [token] "=&v"(token), [c0] "=&s"(c0), [c1] "=&s"(c1), [c2] "=&s"(c2)
          : [o_stay] "v"(o[2 * q + 1]), [o_one] "v"(o[2 * q]), [o_from] "v"(o_from), [stay] "v"(stay), [one] "v"(one), [two] "v"(two), [from] "v"(from)
          : "vcc");
      a[2 * q + 1] = token + r.tok[q];
      a[2 * q] = blank + r.blank;
      o[2 * q + 1] = o_token;
      o[2 * q] = o_blank;
    }
  }
};

template <class SH>
struct Sum {
  static constexpr int Q = SH::R / 2;
  double m[SH::R], below_m;
  int e[SH::R], below_e;
  int col[Q];
  bool apart[Q];                        // token q may follow the token before it directly

  struct alignas(16) Two {
    Prob x, y;
  };
  struct Rows {
    Two blank, tok[Q];
  };
  struct Row {
    Prob blank, tok[Q];
    __device__ __forceinline__ Row(const Rows& r, int i) : blank(i ? r.blank.y : r.blank.x) {
#pragma unroll
      for (int q = 0; q < Q; ++q) tok[q] = i ? r.tok[q].y : r.tok[q].x;
    }
  };
  __device__ __forceinline__ void read(Rows& r, const char* frame, int blank) const {
    r.blank = *reinterpret_cast<const Two*>(frame + blank);
#pragma unroll
    for (int q = 0; q < Q; ++q) r.tok[q] = *reinterpret_cast<const Two*>(frame + col[q]);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < SH::R; ++i) {
      m[i] = 0.0;
      e[i] = kZero;
    }
    below_m = 0.0;
    below_e = kZero;
  }
  __device__ __forceinline__ void first(const Row& r, int base) {      // the first frame
    if (base == 0) {
      m[0] = 1.0 + r.blank.d;
      e[0] = r.blank.e;
      m[1] = 1.0 + r.tok[0].d;
      e[1] = r.tok[0].e;
    }
  }
  __device__ __forceinline__ void step(const Row& r) {
    below_m = shift_in(m[SH::R - 1], below_m);
    below_e = shift_in(e[SH::R - 1], below_e);
#pragma unroll
    for (int q = Q - 1; q >= 0; --q) {
      const double fm = q ? m[q ? 2 * q - 1 : 0] : below_m;
      const int fe = q ? e[q ? 2 * q - 1 : 0] : below_e;
      // from the two states below: what the blank takes, and the token where it may
      const int hi = max(e[2 * q], fe);
      const double sum = scaled(m[2 * q], e[2 * q], hi) + scaled(fm, fe, hi);
      const double up = apart[q] ? sum : m[2 * q];
      const int up_e = apart[q] ? hi : e[2 * q], top = max(e[2 * q + 1], up_e);
      const double all = scaled(m[2 * q + 1], e[2 * q + 1], top) + scaled(up, up_e, top);
      m[2 * q + 1] = fma(all, (double)r.tok[q].d, all);
      e[2 * q + 1] = __builtin_elementwise_add_sat(top, r.tok[q].e);
      m[2 * q] = fma(sum, (double)r.blank.d, sum);
      e[2 * q] = __builtin_elementwise_add_sat(hi, r.blank.e);
    }
  }
  __device__ static __forceinline__ double scaled(double m_, int e_, int hi) { return ldexp(m_, __builtin_elementwise_sub_sat(e_, hi)); }
  // a frame multiplies a mantissa by 0.7 to 4.3: 32 frames stay far inside fp64
  __device__ __forceinline__ void renormalize() {
#pragma unroll
    for (int r = 0; r < SH::R; ++r) {
      const int at = __builtin_elementwise_add_sat(e[r], __builtin_amdgcn_frexp_exp(m[r]));
      const bool none = m[r] == 0.0 || at < kLow;
      e[r] = none ? kZero : min(at, kHigh);
      m[r] = none ? 0.0 : __builtin_amdgcn_frexp_mant(m[r]);
    }
  }
};

// Takes `st` through the frames of a sequence (n > 0): word() after the last frame of every group of F frames the wave steps
// (skip(groups): it does not step these), leg(l) after the last frame of leg l, refresh(write, half) between two legs (W > 1).
// The loader waves fill the next stage meanwhile.  A wave steps only where a path can be: before frame s / 2 none has reached
// its first state s, and from the frame on from which its last state cannot reach the end any more its values are of no use
// (nor are those that would be drawn from them).
template <class SH, bool SUM, class State, class Word, class Skip, class Leg, class Refresh>
__device__ __forceinline__ void over_frames(const Frames& fr, State& st, int L, int wave, int lane, Word&& word, Skip&& skip, Leg&& leg,
                                            Refresh&& refresh) {
  constexpr int F = SH::F;
  const int n = fr.n, ahead = fr.p.ahead, blank = fr.blank_column();
  if (wave >= SH::W) {
    load_frames<SUM>(fr, wave - SH::W, lane);
    return;
  }
  const int low = wave * SH::N, high = low + 64 * SH::R - 1;
  lds_barrier();
  for (int t0 = 0, stage = 0; t0 < n; t0 += ahead, ++stage) {
    const int m = min(ahead, n - t0);
    if (low <= 2 * L && low <= 2 * (t0 + m) - 1 && (int64_t)high + 2 * (int64_t)(n - 1 - t0) >= 2 * L - 1) {
      const char* at = fr.stage(stage);
      typename State::Rows r, next;
      st.read(r, at, blank);
      for (int f = 0; f < m; f += F) {
        // the next two frames' entries under way (behind the sequence's or the stage's end: read and not used)
        if (t0 + f > 0 && f + F <= m) {
#pragma unroll
          for (int i = 0; i < F; i += 2) {
            at += 16;
            st.read(next, at, blank);
            st.step({r, 0});
            st.step({r, 1});
            r = next;
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < F; i += 2) {
            at += 16;
            st.read(next, at, blank);
            if (t0 + f + i == 0) st.first({r, 0}, low + lane * SH::R);
            else if (f + i < m) st.step({r, 0});
            if (f + i + 1 < m) st.step({r, 1});
            r = next;
          }
        }
        word();
      }
      if (((t0 + m) & (kLeg - 1)) == 0 || t0 + m == n) leg((t0 + m - 1) / kLeg);
    } else {
      skip((m + F - 1) / F);
    }
    if (t0 + m < n) {
      const bool now = SH::W > 1 && ((t0 + m) & (kLeg - 1)) == 0;
      const int half = ((t0 + m) / kLeg) & 1;
      if (now) refresh(true, half);
      lds_barrier();
      if (now) refresh(false, half);
    }
  }
}

// The path over the frames t0 .. t1 of one leg from its state `s` at t1, by one wave.  `at` is the state's place in the words:
// 64 R states of the wave below, then 64 R of the one that holds s (or that one alone, where it is wave 0).
template <class SH>
__device__ __forceinline__ void trace(const AlignArgs& p, int s, int t0, int t1, int n, const uint32_t* words, const int32_t* tok, int32_t* labels,
                                      int32_t* spans) {
  constexpr int W = SH::W, R = SH::R, F = SH::F, G = kLeg / F, V = W > 1 ? 2 : 1;
  constexpr int kOver = SH::HL * R;
  // steps back by the state's bits: even states (blank) bit 0; odd ones bit 2 over bit 1 (token: c1, c2): 2 if c2 else c1
  constexpr uint32_t kSteps = 0xa5a04444u;
  const int lane = threadIdx.x & 63;
  int w = 0, at = s;
  while (at >= 64 * R) {
    at -= SH::N;
    ++w;
  }
  if (w > 0) {
    at += 64 * R;
    --w;
  }
  const int g0 = t0 / F, last = t1 / F;
  uint32_t words_of[G][V];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v)
      words_of[i][v] = g0 + i <= last ? words[((int64_t)(g0 + i) * W + min(w + v, W - 1)) * 64 + lane] : 0;
  int path = 0;
#pragma unroll
  for (int i = G - 1; i >= 0; --i) {
    const int first = (g0 + i) * F;
    int drop = 0;                        // bits of the frames behind t in the word
    for (int t = min(t1, first + F - 1); t >= first; --t, drop += SH::kBits) {
      const int l = SH::lane_of(at), q = (at - l * R) >> 1;
      uint32_t word = __builtin_amdgcn_readlane(words_of[i][0], l & 63);
      if (V > 1 && at >= 64 * R) word = __builtin_amdgcn_readlane(words_of[i][V - 1], l & 63);
      path = lane == t - t0 ? s : path;
      const uint32_t bits = (word >> (drop + 3 * q)) & 7;
      const int how = (kSteps >> (2 * bits + 16 * (at & 1))) & 3;
      s -= how;
      at -= how;
      if (W > 1 && at >= 64 * R && at < 64 * R + kOver) at -= kOver;      // the wave below has it
    }
  }
  // s: the state at the frame before t0.  A token begins where the state before is another one, and ends there as well
  const int t = t0 + lane, prev = shift_in(path, t0 ? s : -1);
  if (t > t1) return;
  labels[t] = path & 1 ? tok[path >> 1] : p.blank;
  if (prev != path) {
    if (path & 1) spans[path & ~1] = t;
    if (prev >= 0 && (prev & 1)) spans[prev | 1] = t;
  }
  if (t == n - 1 && (path & 1)) spans[path | 1] = n;
}

// The stepping waves are 0 .. W - 1, the loaders W ...  A workgroup's waves are dealt to the CU's four SIMDs in turn, so of
// five the first and the last share one: the single stepping wave is the second.
template <class SH>
__device__ __forceinline__ int role() {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  return SH::W == 1 && wave < 2 ? 1 - wave : wave;
}

// what the waves pass on to the next one, by half, wave and state: a double, and behind all of them an int
template <class SH>
struct Over {
  static constexpr int kStates = SH::HL * SH::R, kAll = 2 * SH::W * kStates;
  static constexpr int kBytes = kAll ? kAll * 12 : 16;
  char* buf;
  __device__ __forceinline__ double& value(int half, int wave, int i) const { return reinterpret_cast<double*>(buf)[(half * SH::W + wave) * kStates + i]; }
  __device__ __forceinline__ int& exponent(int half, int wave, int i) const {
    return reinterpret_cast<int*>(buf + kAll * 8)[(half * SH::W + wave) * kStates + i];
  }
};

template <class SH>
__device__ void best_path(const AlignArgs& p, int b, int L, int n, char* lds, Over<SH> over) {
  constexpr int W = SH::W, R = SH::R, HL = SH::HL, kThreads = 64 * (W + kLoaders);
  constexpr int kLegs = 256;             // legs traced between two barriers
  __shared__ double s_end[2];
  __shared__ int s_state[kLegs];
  const int lane = threadIdx.x & 63, wave = role<SH>(), base = wave * SH::N + lane * R;
  uint32_t* words = p.words + (int64_t)b * ((p.frames + SH::F - 1) / SH::F) * W * 64;
  uint16_t* came = p.came + (int64_t)b * ((p.frames + kLeg - 1) / kLeg) * SH::kStates;
  int32_t* labels = p.labels + (int64_t)b * p.frames;
  int32_t* spans = p.spans + (int64_t)b * p.most * 2;
  const int32_t* tok = p.tokens + (int64_t)b * p.most;
  if (threadIdx.x < 2) s_end[threadIdx.x] = n == 0 && L == 0 && threadIdx.x == 0 ? 0.0 : -INFINITY;   // [0]: last blank, [1]: last token
  if (n > 0) {
    const Frames fr(p, b, n, lds);
    Best<SH> st;
#pragma unroll
    for (int q = 0; q < R / 2; ++q) {
      const int i = (base >> 1) + q;
      st.col[q] = wave < W ? fr.column(i, L) : 0;
      st.apart[q] = !(wave < W && i > 0 && i < L && tok[i] == tok[i - 1]);
    }
    uint32_t* out = words + wave * 64 + lane;
    st.clear(base);
    over_frames<SH, false>(
        fr, st, L, wave, lane,
        [&] {
          *out = st.word;
          out += W * 64;
          st.word = 0;
        },
        [&](int groups) { out += groups * (W * 64); },
        [&](int l) {
          if (wave == 0 || lane >= HL) {
            uint32_t* to = reinterpret_cast<uint32_t*>(came + (int64_t)l * SH::kStates + base);
#pragma unroll
            for (int q = 0; q < R / 2; ++q) to[q] = st.o[2 * q] | st.o[2 * q + 1] << 16;
          }
          st.mark(base);
        },
        [&](bool write, int half) {
          if constexpr (W > 1) {
            if (write) {
              if (lane >= 64 - HL)
#pragma unroll
                for (int r = 0; r < R; ++r) over.value(half, wave, (lane - (64 - HL)) * R + r) = st.a[r];
            } else if (wave > 0 && lane < HL) {
#pragma unroll
              for (int r = 0; r < R; ++r) st.a[r] = over.value(half, wave - 1, lane * R + r);
            }
          }
        });
    if (wave < W && (wave == 0 || lane >= HL)) {
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
  for (int t = (alive ? n : 0) + threadIdx.x; t < p.frames; t += kThreads) labels[t] = -1;
  for (int i = (alive ? 2 * L : 0) + threadIdx.x; i < 2 * p.most; i += kThreads) spans[i] = -1;
  if (threadIdx.x == 0) p.score[b] = (float)score;
  if (!alive || n == 0) return;
  int s = at_token > at_blank ? 2 * L - 1 : 2 * L;
  for (int leg = (n - 1) / kLeg; leg >= 0; leg -= kLegs) {              // s: the state at the end of `leg`
    const int low = max(0, leg - kLegs + 1);
    if (wave == 0) {
      for (int k = leg; k >= low; --k) {
        if (lane == 0) s_state[leg - k] = s;
        if (k > 0) s = __builtin_amdgcn_readfirstlane(came[(int64_t)k * SH::kStates + s]);
      }
    }
    __syncthreads();
    for (int k = leg - wave; k >= low; k -= W + kLoaders)
      trace<SH>(p, __builtin_amdgcn_readfirstlane(s_state[leg - k]), k * kLeg, min(n, (k + 1) * kLeg) - 1, n, words, tok, labels, spans);
    __syncthreads();
  }
}

template <class SH>
__device__ void all_paths(const AlignArgs& p, int b, int L, int n, char* lds, Over<SH> over) {
  constexpr int W = SH::W, R = SH::R, HL = SH::HL;
  __shared__ double s_end_m[2];
  __shared__ int s_end_e[2];
  const int lane = threadIdx.x & 63, wave = role<SH>(), base = wave * SH::N + lane * R;
  const int32_t* tok = p.tokens + (int64_t)b * p.most;
  if (n == 0) {
    if (threadIdx.x == 0) p.total[b] = L == 0 ? 0.f : -INFINITY;
    return;
  }
  if (threadIdx.x < 2) {
    s_end_m[threadIdx.x] = 0.0;
    s_end_e[threadIdx.x] = kZero;
  }
  const Frames fr(p, b, n, lds);
  Sum<SH> st;
#pragma unroll
  for (int q = 0; q < R / 2; ++q) {
    const int i = (base >> 1) + q;
    st.col[q] = wave < W ? fr.column(i, L) : 0;
    st.apart[q] = !(wave < W && i > 0 && i < L && tok[i] == tok[i - 1]);
  }
  st.clear();
  over_frames<SH, true>(
      fr, st, L, wave, lane,
      [] {}, [](int) {}, [&](int) { st.renormalize(); },
      [&](bool write, int half) {
        if constexpr (W > 1) {
          if (write) {
            if (lane >= 64 - HL)
#pragma unroll
              for (int r = 0; r < R; ++r) {
                over.value(half, wave, (lane - (64 - HL)) * R + r) = st.m[r];
                over.exponent(half, wave, (lane - (64 - HL)) * R + r) = st.e[r];
              }
          } else if (wave > 0 && lane < HL) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
              st.m[r] = over.value(half, wave - 1, lane * R + r);
              st.e[r] = over.exponent(half, wave - 1, lane * R + r);
            }
          }
        }
      });
  if (wave < W && (wave == 0 || lane >= HL)) {
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
    // mantissas are in [0.5, 1): a total close to 0 is the logarithm of a number close to 1, with no exponent to take off it
    int hi = max(s_end_e[0], s_end_e[1]);
    double sum = ldexp(s_end_m[0], s_end_e[0] - hi) + ldexp(s_end_m[1], s_end_e[1] - hi);
    if (sum < 0.70710678) {
      sum *= 2;
      --hi;
    } else if (sum > 1.41421356) {
      sum *= 0.5;
      ++hi;
    }
    p.total[b] = sum == 0.0 ? -INFINITY : (float)(hi * 0.693147180559945309 + log(sum));
  }
}

// workgroup b: the best path of sequence b; batch + b: the sum of all
template <int W, int R>
__global__ void __launch_bounds__(64 * (W + kLoaders)) align_kernel(AlignArgs p) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  using SH = Shape<W, R>;
  __shared__ __attribute__((aligned(16))) char s_over[Over<SH>::kBytes];
  const bool sum = (int)blockIdx.x >= p.batch;
  const int b = sum ? blockIdx.x - p.batch : blockIdx.x;
  const int L = min(max(p.token_lens[b], 0), p.most), n = min(max(p.frame_lens[b], 0), p.frames);
  if (sum) all_paths<SH>(p, b, L, n, lds, {s_over});
  else best_path<SH>(p, b, L, n, lds, {s_over});
}

template <int W, int R>
hipError_t launch_as(AlignArgs p, hipStream_t st) {
  p.direct = p.vocab <= p.most + 1;
  p.columns = p.direct ? p.vocab : p.most + 1;
  // frames per stage: a leg, or a divisor of it that leaves room for two stages beside the rest of the LDS (never fewer than a
  // word has)
  p.ahead = kLeg;
  constexpr int kLds = 128 * 1024;
  while (p.ahead > 2 && 16 * (p.ahead + 2) * (p.columns + 1) > kLds) p.ahead /= 2;
  static_assert(16 * (2 + 2) * (TONE_ALIGN_MAX_TOKENS + 2) <= kLds, "two frames of the longest sequences fit");
  const size_t lds = (size_t)16 * (p.ahead + 2) * (p.columns + 1);
  auto* fn = align_kernel<W, R>;
  if (lds > 32 * 1024) {                 // the same limit whoever calls: calls on several threads do not undo each other's
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3(p.total ? 2 * p.batch : p.batch), dim3(64 * (W + kLoaders)), lds, st, p);
  return hipGetLastError();
}

// The fewest states per lane and waves that hold the sequences.  One sequence of 2000 frames, without and with its sum: 43
// tokens 189 / 189 us, 150 (four waves) 201 / 209, 400 (four states per lane) 269 / 269, 700 (eight waves) 342 / 367, 900 (twelve
// waves) 376 / 416, 1300 (eight waves of eight states) 543 / 581; without, 700 tokens on four waves of eight states take 532, 900
// on eight of eight 587.
template <class Fn>
auto by_tokens(int most, Fn&& fn) {
  const int states = 2 * most + 1;
  if (states <= Shape<1, 2>::kStates) return fn(Shape<1, 2>{});
  if (states <= Shape<4, 2>::kStates) return fn(Shape<4, 2>{});
  if (states <= Shape<4, 4>::kStates) return fn(Shape<4, 4>{});
  if (states <= Shape<8, 4>::kStates) return fn(Shape<8, 4>{});
  if (states <= Shape<12, 4>::kStates) return fn(Shape<12, 4>{});
  return fn(Shape<8, 8>{});
}
static_assert(Shape<8, 8>::kStates >= 2 * TONE_ALIGN_MAX_TOKENS + 1, "the longest sequences fit");

hipError_t launch_align(const AlignArgs& p, hipStream_t st) {
  return by_tokens(p.most, [&](auto sh) { return launch_as<decltype(sh)::W, decltype(sh)::R>(p, st); });
}

// bytes of the words, and of the states at the legs' beginnings behind them
struct Workspace {
  int64_t words, came;
};
Workspace align_workspace(int batch, int frames, int most) {
  return by_tokens(most, [&](auto sh) -> Workspace {
    using SH = decltype(sh);
    return {(int64_t)batch * ((frames + SH::F - 1) / SH::F) * SH::W * 64 * 4, (int64_t)batch * ((frames + kLeg - 1) / kLeg) * SH::kStates * 2};
  });
}

}  // namespace
}  // namespace tone

using namespace tone;

extern "C" {

int64_t tone_ctc_align_workspace(int batch, int frames, int tokens) {
  if (batch < 0 || frames < 0 || frames > kMaxFrames || tokens < 0 || tokens > TONE_ALIGN_MAX_TOKENS) return -1;
  const Workspace w = align_workspace(batch, frames, tokens);
  return w.words + w.came;
}

int tone_ctc_align(int device, const void* x, int type, int64_t stride, int64_t batch_stride, int64_t x_rows,
                   const int64_t* rows, int batch, int frames, int vocab, int blank, const int32_t* tokens, int max_tokens,
                   const int32_t* token_lens, const int32_t* frame_lens, float* score, float* total, int32_t* labels,
                   int32_t* spans, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "tone_ctc_align";
  if (batch < 0 || frames < 0 || x_rows < 0 || vocab <= 0 || vocab > (1 << 24))
    return refuse(what, "batch, frames, x_rows or vocab out of range");
  if (frames > kMaxFrames || batch > kMaxThreads / (2 * 64 * (12 + kLoaders))) return refuse(what, "batch or frames too large for one launch");
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
              score, total, labels, spans, static_cast<uint32_t*>(workspace),
              reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + align_workspace(batch, frames, max_tokens).words), 0, 0, 0};
  return launch_on(device, what, [&] { return launch_align(p, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
