// CTC alignment of given token sequences.  A sequence of L tokens is the chain of 2L + 1 states blank, token 0, blank, ...,
// token L - 1, blank; a path holds one state per frame, starts in state 0 or 1, stays, moves on by one, or by two over the
// blank between two different tokens, and ends in one of the last two.  With e_t(s) the frame's log probability of the
// state's label
//   best_t(s)  = max(best_{t-1}(s), best_{t-1}(s - 1), best_{t-1}(s - 2) where allowed) + e_t(s)
//   total_t(s) = the same with log-sum-exp
// The first of equals is taken in that order, and the last blank before the last token at the end.  The sums are held in
// 64 bits: a minute of frames adds up 2000 terms, the paths' difference may be one rounding of a term, and the sequence
// of additions is the definition's, so the path is reproducible bit for bit.
#include "scoring.h"

#include <algorithm>

namespace tone {
namespace {

struct AlignArgs {
  const void* x;                        // frame (b, t) at b * batch_stride + t * stride, or rows[b][t] * stride
  int64_t stride, batch_stride, x_rows;
  const int64_t* rows;
  int batch, frames, vocab, blank;
  const int32_t* tokens;                // [batch][most]
  int most;
  const int32_t *token_lens, *frame_lens;
  float *score, *total;                 // total: or nullptr
  int32_t *labels, *spans;              // [batch][frames], [batch][most][2]
  uint8_t* came;
};

constexpr int kThreads = 256;

__device__ __forceinline__ double lse3(double a, double b, double c) {
  const double h = fmax(fmax(a, b), c);
  if (!(h > -INFINITY)) return h;
  return h + (double)logf(expf((float)(a - h)) + expf((float)(b - h)) + expf((float)(c - h)));
}

template <typename T, bool TOTAL>
__global__ void __launch_bounds__(kThreads) align_kernel(AlignArgs p) {
  extern __shared__ double lat[];       // [2][S + 2] best, [2][S + 2] total: two unreachable states in front
  const int b = blockIdx.x, tid = threadIdx.x;
  const int S = 2 * p.most + 1, ld = S + 2;
  const int L = min(max(p.token_lens[b], 0), p.most), F = min(max(p.frame_lens[b], 0), p.frames), SL = 2 * L + 1;
  const int32_t* tok = p.tokens + (int64_t)b * p.most;
  uint8_t* came = p.came + (int64_t)b * p.frames * S;
  double *best = lat, *sum = lat + 2 * ld;
  for (int i = tid; i < 2 * ld; i += kThreads) {
    best[i] = -INFINITY;
    if (TOTAL) sum[i] = -INFINITY;
  }
  __syncthreads();
  for (int t = 0; t < F; ++t) {
    const double* from = best + (t & 1) * ld;
    double* to = best + (~t & 1) * ld;
    const double* sfrom = sum + (t & 1) * ld;
    double* sto = sum + (~t & 1) * ld;
    const int64_t row = p.rows ? p.rows[(int64_t)b * p.frames + t] : 0;
    const bool here = !p.rows || (row >= 0 && row < p.x_rows);
    const T* x = static_cast<const T*>(p.x) + (p.rows ? row * p.stride : b * p.batch_stride + t * p.stride);
    for (int s = tid; s < SL; s += kThreads) {
      const int label = s & 1 ? tok[s >> 1] : p.blank;
      const bool fine = here && label >= 0 && label < p.vocab && (!(s & 1) || label != p.blank);
      float e = fine ? load_elem(x + label) : -INFINITY;
      if (!(fabsf(e) < INFINITY)) e = -INFINITY;
      const bool skip = (s & 1) && s > 1 && label != tok[(s >> 1) - 1];
      double stay = from[s + 2], one = from[s + 1], two = skip ? from[s] : -INFINITY;
      if (t == 0) {
        stay = s < 2 ? 0.0 : -INFINITY;
        one = two = -INFINITY;
      }
      double m = stay;
      int how = 0;
      if (one > m) { m = one; how = 1; }
      if (two > m) { m = two; how = 2; }
      to[s + 2] = m + e;
      came[(int64_t)t * S + s] = how;
      if (TOTAL) {
        double a = sfrom[s + 2], c1 = sfrom[s + 1], c2 = skip ? sfrom[s] : -INFINITY;
        if (t == 0) {
          a = s < 2 ? 0.0 : -INFINITY;
          c1 = c2 = -INFINITY;
        }
        sto[s + 2] = lse3(a, c1, c2) + e;
      }
    }
    __syncthreads();
  }
  int32_t* labels = p.labels + (int64_t)b * p.frames;
  int32_t* spans = p.spans + (int64_t)b * p.most * 2;
  const double* fin = best + (F & 1) * ld;
  const double* sfin = sum + (F & 1) * ld;
  double at_blank = fin[2 * L + 2], at_token = L ? fin[2 * L + 1] : -INFINITY;
  if (F == 0) at_blank = L ? -INFINITY : 0.0;
  const double score = fmax(at_blank, at_token);
  const bool alive = score > -INFINITY;
  for (int t = tid; t < p.frames; t += kThreads) labels[t] = -1;
  for (int i = tid; i < 2 * p.most; i += kThreads) spans[i] = -1;
  __syncthreads();
  if (tid == 0) {
    p.score[b] = (float)score;
    if (TOTAL) p.total[b] = F ? (float)lse3(sfin[2 * L + 2], L ? sfin[2 * L + 1] : -INFINITY, -INFINITY) : (float)score;
    if (alive) {
      int s = at_token > at_blank ? 2 * L - 1 : 2 * L;
      for (int t = F - 1; t >= 0; --t) {
        labels[t] = s & 1 ? tok[s >> 1] : p.blank;
        if (s & 1) {
          spans[s & ~1] = t;
          if (spans[s | 1] < 0) spans[s | 1] = t + 1;
        }
        s = max(0, s - came[(int64_t)t * S + s]);
      }
    }
  }
}

template <typename T>
hipError_t launch_as(const AlignArgs& p, hipStream_t st) {
  const size_t lds = (size_t)(p.total ? 4 : 2) * (2 * p.most + 3) * sizeof(double);
  auto* fn = p.total ? align_kernel<T, true> : align_kernel<T, false>;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fn, dim3(p.batch), dim3(kThreads), lds, st, p);
  return hipGetLastError();
}

hipError_t launch_align(const AlignArgs& p, int type, hipStream_t st) {
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

int64_t tone_ctc_align_workspace(int batch, int frames, int tokens) {
  if (batch < 0 || frames < 0 || tokens < 0 || tokens > TONE_ALIGN_MAX_TOKENS) return -1;
  return (int64_t)batch * frames * (2 * tokens + 1);
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
  AlignArgs p{x, stride, batch_stride, x_rows, rows, batch, frames, vocab, blank, tokens, max_tokens, token_lens, frame_lens,
              score, total, labels, spans, static_cast<uint8_t*>(workspace)};
  return launch_on(device, what, [&] { return launch_align(p, type, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
