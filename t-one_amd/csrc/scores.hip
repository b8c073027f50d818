// What each row of (log) probabilities says: for x over V entries, with m = max x and s = sum e^(x - m),
//   log probability of a given token t   x_t - m - ln s
//   entropy                              ln s - (sum e^(x - m) (x - m)) / s
//   rank of t                            #{x_v > x_t} + #{v < t, x_v = x_t}
//   top k                                by value, equal values by the lowest index, as log probabilities
// Statistics are held in 32 bits whatever the input's type.
#include "scoring.h"

#include <algorithm>

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

// larger value = larger key; equal values: the lower index has the larger key.  -0 and +0 are one value.
__device__ __forceinline__ uint64_t order_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((uint64_t)o << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// one wave per row
template <typename T>
__global__ void __launch_bounds__(256) scores_kernel(ScoreArgs p) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= p.n) return;
  const int64_t row = p.rows ? p.rows[n] : n;
  const bool here = row >= 0 && row < p.x_rows;
  if (!here) {
    if (lane == 0) {
      if (p.logprob) p.logprob[n] = 0.f;
      if (p.rank) p.rank[n] = -1;
      p.entropy[n] = 0.f;
    }
    if (lane < p.k) {
      p.top_lp[n * p.k + lane] = -INFINITY;
      p.top_ids[n * p.k + lane] = -1;
    }
    return;
  }
  const T* x = static_cast<const T*>(p.x) + row * p.stride;
  const int t = p.tokens ? p.tokens[n] : -1;
  const bool given = t >= 0 && t < p.vocab;
  const float xt = given ? load_elem(x + t) : 0.f;
  float m = -INFINITY;
  for (int v = lane; v < p.vocab; v += 64) m = fmaxf(m, load_elem(x + v));
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  float s = 0.f, u = 0.f;
  int above = 0;
  for (int v = lane; v < p.vocab; v += 64) {
    const float xv = load_elem(x + v);
    const float z = xv - m, e = expf(z);
    if (xv > -INFINITY || !(xv == xv)) {
      s += e;
      u += e > 0.f ? e * z : (z == z ? 0.f : z);
    }
    above += xv > xt || (xv == xt && v < t);
  }
  for (int o = 32; o; o >>= 1) {
    s += __shfl_xor(s, o);
    u += __shfl_xor(u, o);
    above += __shfl_xor(above, o);
  }
  const bool left = !(s == 0.f);
  const float ls = logf(s);
  if (lane == 0) {
    if (p.logprob) p.logprob[n] = given ? (left ? xt - m - ls : -INFINITY) : 0.f;
    if (p.rank) p.rank[n] = given ? above : -1;
    p.entropy[n] = left ? ls - u / s : 0.f;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.k; ++i) {
    uint64_t best = 0;
    for (int v = lane; v < p.vocab; v += 64) {
      const uint64_t key = order_key(load_elem(x + v), v);
      if (key < last && key > best) best = key;
    }
    for (int o = 32; o; o >>= 1) {
      const uint64_t other = __shfl_xor((unsigned long long)best, o);
      if (other > best) best = other;
    }
    last = best;
    if (lane == 0) {
      p.top_lp[n * p.k + i] = left ? key_value(best) - m - ls : -INFINITY;
      p.top_ids[n * p.k + i] = (int32_t)~(uint32_t)best;
    }
  }
}

hipError_t launch_scores(const ScoreArgs& p, int type, hipStream_t st) {
  const dim3 grid((unsigned)((p.n + 3) / 4));
  switch (type) {
    case TONE_TYPE_FP32: hipLaunchKernelGGL(scores_kernel<float>, grid, dim3(256), 0, st, p); break;
    case TONE_TYPE_FP16: hipLaunchKernelGGL(scores_kernel<__half>, grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL(scores_kernel<Bf16>, grid, dim3(256), 0, st, p);
  }
  return hipGetLastError();
}

}  // namespace
}  // namespace tone

using namespace tone;

extern "C" {

int64_t tone_token_scores_workspace(int64_t n, int vocab, int k) { return n < 0 || vocab <= 0 || k < 0 ? -1 : 0; }

int tone_token_scores(int device, const void* x, int type, int64_t stride, int64_t x_rows, const int64_t* rows, int64_t n,
                      int vocab, const int32_t* tokens, int k, float* logprob, float* entropy, int32_t* rank,
                      float* top_logprob, int32_t* top_ids, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "tone_token_scores";
  if (n < 0 || x_rows < 0 || vocab <= 0 || vocab > (1 << 24)) return refuse(what, "n, x_rows or vocab out of range");
  if (!known_type(type)) return refuse(what, "unknown element type");
  if (k < 0 || k > TONE_SCORES_MAX_K || k > vocab) return refuse(what, "k must be in 0 .. min(vocab, TONE_SCORES_MAX_K)");
  if (n == 0) return TONE_OK;
  if ((!x && x_rows) || !entropy || (k && (!top_logprob || !top_ids))) return refuse(what, "null pointer");
  if (tokens && (!logprob || !rank)) return refuse(what, "tokens without logprob or rank");
  if (!rows && x_rows < n) return refuse(what, "fewer rows in x than outputs");
  if (stride < vocab && x_rows > 1) return refuse(what, "row stride < vocab");
  if ((n + 3) / 4 > INT32_MAX) return refuse(what, "too many rows for one launch");
  const int64_t need = tone_token_scores_workspace(n, vocab, k);
  if (workspace_bytes < need || (need && !workspace)) return refuse(what, "workspace smaller than tone_token_scores_workspace");
  ScoreArgs p{x, stride, x_rows, rows, n, vocab, k, tokens, tokens ? logprob : nullptr, entropy, tokens ? rank : nullptr,
              top_logprob, top_ids};
  return launch_on(device, what, [&] { return launch_scores(p, type, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
