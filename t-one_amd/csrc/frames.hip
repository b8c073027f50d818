// Pages of frames: a pool of rows (one per acoustic frame) shared by many streams in pages of P rows, the page tables and
// slot maps built on the device from the streams' frame counts, and the copy of a step's rows through such a map.
//
// A stream holds the frames [first, length), so the pages [first / P, ceil(length / P)) (none when first == length); its
// table row lists them from entry 0.  A request moves it to [max(first, keep), length + add): the pages of the old range
// that are not in the new one go back to the free queue, the pages of the new one that are not in the old one come from
// it.  Which entries of the queue a request takes or fills is the prefix sum, in batch order, of the pages the requests
// before it take or release, so the result does not depend on how the work is scheduled.  The queue is FIFO: [head, tail)
// modulo n_pages are the free pages.  Pages are only taken from what was free before the call, so the entries read
// ([head, head + taken)) and the entries written ([tail, tail + released)) never meet: free + released <= n_pages.
#include "scoring.h"

#include <algorithm>

namespace tone {
namespace {

struct PlanArgs {
  int32_t* table;                       // [n_rows][width], rows `stride` entries apart
  int64_t stride;
  int n_rows, width;
  int32_t* queue;                       // [n_pages]
  int n_pages, page;
  const int64_t* cursors_in;            // head, tail of the queue
  int64_t* cursors_out;
  const int32_t *rows_in, *rows_out, *first, *length, *keep, *add;   // [batch]
  int batch;
  int64_t* slots;                       // [batch][max_add]
  int max_add;
  int32_t* status;
};

struct SlotArgs {
  const int32_t* table;
  int64_t stride;
  int n_rows, width, n_pages, page;
  const int32_t *rows, *first, *begin, *count;   // [batch]
  int batch;
  int64_t* slots;                       // [batch][max_count]
  int max_count;
};

struct PutArgs {
  const void* src;
  int src_type;
  int64_t src_stride;
  const int64_t* slots;
  int64_t n;
  int vocab;
  void* pool;
  int pool_type;
  int64_t pool_stride, pool_rows;
};

constexpr int kPlanThreads = 256;
constexpr int kPlanRows = 32;          // requests a workgroup writes, at most

struct Request {
  int64_t kept, end;                   // the frames held after the call
  int64_t lo0, hi0, lo1, hi1;          // pages held before / after
  int64_t from;                        // first page taken
  int take, drop;
  bool bad, wide;
};

__device__ __forceinline__ Request read_request(const PlanArgs& p, int b) {
  Request r;
  const int64_t first = p.first[b], length = p.length[b], keep = p.keep[b], add = p.add[b], P = p.page;
  const int ri = p.rows_in[b], ro = p.rows_out[b];
  r.kept = first > keep ? first : keep;
  r.end = length + add;
  r.bad = first < 0 || first > length || add < 0 || add > p.max_add || keep < 0 || keep > r.end || ri < 0 || ri >= p.n_rows ||
          ro < 0 || ro >= p.n_rows || ri == ro;
  if (r.bad) {
    r.lo0 = r.hi0 = r.lo1 = r.hi1 = r.from = 0;
    r.take = r.drop = 0;
    r.wide = false;
    return r;
  }
  const bool had = first < length, has = r.kept < r.end;
  // frame numbers are 31 bits, the end 32: unsigned 32-bit divisions
  const uint32_t u = (uint32_t)P;
  r.lo0 = (uint32_t)first / u;
  r.hi0 = had ? ((uint32_t)length - 1u) / u + 1 : r.lo0;
  r.lo1 = (uint32_t)r.kept / u;
  r.hi1 = has ? ((uint32_t)r.end - 1u) / u + 1 : r.lo1;
  r.from = had && r.hi0 > r.lo1 ? r.hi0 : r.lo1;
  r.take = has ? (int)(r.hi1 - r.from) : 0;
  r.drop = had ? (int)((has && r.lo1 < r.hi0 ? r.lo1 : r.hi0) - r.lo0) : 0;
  r.wide = r.hi1 - r.lo1 > p.width || r.hi0 - r.lo0 > p.width;
  return r;
}

// One launch: every workgroup adds up the pages of all requests (16 bytes each, out of L2) to place its own ones, instead of
// a scan kernel in front of a writing kernel.  blockIdx.x: up to kPlanRows requests; blockIdx.y: a share of their slots.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PlanArgs p, int rows_per) {
  __shared__ int64_t part[kPlanThreads / 64][4];
  __shared__ int s_take[kPlanRows], s_drop[kPlanRows];
  __shared__ int s_flags;
  const int tid = threadIdx.x, r0 = blockIdx.x * rows_per, r1 = min(p.batch, r0 + rows_per);
  if (tid == 0) s_flags = 0;
  __syncthreads();
  int64_t take = 0, take0 = 0, drop = 0, drop0 = 0;      // of all requests / of those before r0
  int flags = 0;
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const Request r = read_request(p, b);
    flags |= (r.wide ? TONE_FRAMES_ROW_FULL : 0) | (r.bad ? TONE_FRAMES_BAD_REQUEST : 0);
    take += r.take;
    drop += r.drop;
    if (b < r0) {
      take0 += r.take;
      drop0 += r.drop;
    } else if (b < r1) {
      s_take[b - r0] = r.take;
      s_drop[b - r0] = r.drop;
    }
  }
  int64_t v[4] = {take, take0, drop, drop0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int o = 32; o; o >>= 1) v[i] += __shfl_xor(v[i], o);
    if ((tid & 63) == 0) part[tid >> 6][i] = v[i];
  }
  if (flags) atomicOr(&s_flags, flags);
  __syncthreads();
  flags = s_flags;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) v[i] += part[w][i];
  }
  const int64_t head = p.cursors_in[0], tail = p.cursors_in[1];
  // free + released <= n_pages holds for every state these calls produce; anything else is not a queue of this pool
  if (head < 0 || tail < head || tail - head + v[2] > p.n_pages) flags |= TONE_FRAMES_BAD_QUEUE;
  else if (v[0] > tail - head) flags |= TONE_FRAMES_NO_PAGES;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    p.cursors_out[0] = head + (flags ? 0 : v[0]);
    p.cursors_out[1] = tail + (flags ? 0 : v[2]);
    p.status[0] = flags;
  }
  const int64_t h0 = flags ? 0 : head % p.n_pages, q0 = flags ? 0 : tail % p.n_pages;
  int64_t at_take = h0 + v[1], at_drop = q0 + v[3];
  const int seg = (p.max_add + gridDim.y - 1) / gridDim.y, s0 = blockIdx.y * seg, s1 = min(p.max_add, s0 + seg);
  for (int b = r0; b < r1; ++b) {
    const Request r = read_request(p, b);
    int64_t* slots = p.slots + (int64_t)b * p.max_add;
    if (flags) {
      for (int j = s0 + tid; j < s1; j += kPlanThreads) slots[j] = -1;
      const int ri = p.rows_in[b], ro = p.rows_out[b];
      if (blockIdx.y == 0 && ri >= 0 && ri < p.n_rows && ro >= 0 && ro < p.n_rows)
        for (int j = tid; j < p.width; j += kPlanThreads) p.table[ro * p.stride + j] = p.table[ri * p.stride + j];
      continue;
    }
    const int32_t* before = p.table + p.rows_in[b] * p.stride;
    // page of logical page lp: kept from the old row, or the next entry of the queue
    auto page_of = [&](int64_t lp) -> int32_t {
      if (lp < r.hi0 && r.hi0 > r.lo0) return before[lp - r.lo0];
      int64_t i = at_take + (lp - r.from);
      if (i >= p.n_pages) i -= p.n_pages;      // at_take < 2 n_pages: taken <= free <= n_pages
      return p.queue[i];
    };
    if (blockIdx.y == 0) {
      int32_t* after = p.table + p.rows_out[b] * p.stride;
      for (int j = tid; j < p.width; j += kPlanThreads) after[j] = r.lo1 + j < r.hi1 ? page_of(r.lo1 + j) : -1;
      for (int j = tid; j < r.drop; j += kPlanThreads) {
        int64_t i = at_drop + j;
        if (i >= p.n_pages) i -= p.n_pages;
        p.queue[i] = before[j];
      }
    }
    const int64_t length = p.length[b];
    const int add = p.add[b];
    const uint32_t base = (uint32_t)(r.lo1 * p.page), u = (uint32_t)p.page;
    for (int j = s0 + tid; j < s1; j += kPlanThreads) {
      const int64_t f = length + j;
      int64_t slot = -1;
      if (j < add && f >= r.kept) {
        const uint32_t off = (uint32_t)f - base, q = off / u;
        const int32_t pg = page_of(r.lo1 + q);
        if (pg >= 0 && pg < p.n_pages) slot = (int64_t)pg * u + (off - q * u);
      }
      slots[j] = slot;
    }
    at_take += s_take[b - r0];
    at_drop += s_drop[b - r0];
  }
}

__global__ void __launch_bounds__(256) slots_kernel(SlotArgs p, int segs) {
  const int b = blockIdx.x / segs;
  const int j = (blockIdx.x - b * segs) * 256 + threadIdx.x;
  if (j >= p.max_count) return;
  const int row = p.rows[b], first = p.first[b], count = p.count[b];
  const int64_t f = (int64_t)p.begin[b] + j;
  int64_t slot = -1;
  if (row >= 0 && row < p.n_rows && first >= 0 && j < count && f >= first && f <= 0x7fffffff) {
    const uint32_t u = (uint32_t)p.page, q = (uint32_t)f / u, at = q - (uint32_t)first / u;
    if (at < (uint32_t)p.width) {
      const int32_t pg = p.table[row * p.stride + at];
      if (pg >= 0 && pg < p.n_pages) slot = (int64_t)pg * u + ((uint32_t)f - q * u);
    }
  }
  p.slots[(int64_t)b * p.max_count + j] = slot;
}

// rows [16 x blockIdx.x, + 16) of src, one element per thread and step
template <typename S, typename D>
__global__ void __launch_bounds__(256) put_kernel(const S* __restrict__ src, int64_t src_stride, const int64_t* __restrict__ slots,
                                                  int64_t n, int vocab, D* __restrict__ pool, int64_t pool_stride, int64_t pool_rows) {
  const int64_t r0 = (int64_t)blockIdx.x * 16;
  const int rows = (int)min((int64_t)16, n - r0);
  for (int e = threadIdx.x; e < rows * vocab; e += 256) {
    const int r = e / vocab, c = e - r * vocab;
    const int64_t s = slots[r0 + r];
    if (s >= 0 && s < pool_rows) store_elem(pool + s * pool_stride + c, load_elem(src + (r0 + r) * src_stride + c));
  }
}

template <typename S>
hipError_t put_from(const PutArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.n + 15) / 16));
  const S* src = static_cast<const S*>(a.src);
  switch (a.pool_type) {
    case TONE_TYPE_FP32:
      hipLaunchKernelGGL((put_kernel<S, float>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, a.vocab,
                         static_cast<float*>(a.pool), a.pool_stride, a.pool_rows);
      break;
    case TONE_TYPE_FP16:
      hipLaunchKernelGGL((put_kernel<S, __half>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, a.vocab,
                         static_cast<__half*>(a.pool), a.pool_stride, a.pool_rows);
      break;
    default:
      hipLaunchKernelGGL((put_kernel<S, Bf16>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, a.vocab,
                         static_cast<Bf16*>(a.pool), a.pool_stride, a.pool_rows);
  }
  return hipGetLastError();
}

hipError_t launch_plan(const PlanArgs& p, hipStream_t st) {
  // about one workgroup per CU over the requests; long slot rows are shared by several
  const int rows_per = std::min(kPlanRows, std::max(1, (p.batch + 255) / 256));
  const int gx = std::max(1, (p.batch + rows_per - 1) / rows_per);   // an empty batch still writes the cursors and the status
  const int gy = std::max(1, std::min({64, 1024 / std::max(1, gx), (p.max_add + 1023) / 1024}));
  hipLaunchKernelGGL(plan_kernel, dim3(gx, gy), dim3(kPlanThreads), 0, st, p, rows_per);
  return hipGetLastError();
}

hipError_t launch_slots(const SlotArgs& p, hipStream_t st) {
  const int segs = (p.max_count + 255) / 256;
  hipLaunchKernelGGL(slots_kernel, dim3((unsigned)segs * (unsigned)p.batch), dim3(256), 0, st, p, segs);
  return hipGetLastError();
}

hipError_t launch_put(const PutArgs& a, hipStream_t st) {
  switch (a.src_type) {
    case TONE_TYPE_FP32: return put_from<float>(a, st);
    case TONE_TYPE_FP16: return put_from<__half>(a, st);
    default: return put_from<Bf16>(a, st);
  }
}

}  // namespace
}  // namespace tone

using namespace tone;

extern "C" {

int tone_frames_plan(int device, int32_t* table, int64_t table_stride, int n_rows, int width, int32_t* queue, int n_pages,
                     int page_size, const int64_t* cursors_in, int64_t* cursors_out, const int32_t* rows_in,
                     const int32_t* rows_out, const int32_t* first, const int32_t* length, const int32_t* keep,
                     const int32_t* add, int batch, int64_t* slots, int max_add, int32_t* status, void* stream) {
  const char* what = "tone_frames_plan";
  if (batch < 0 || max_add < 0) return refuse(what, "negative batch or max_add");
  if (!table || !queue || !cursors_in || !cursors_out || !status) return refuse(what, "null table, queue, cursors or status");
  if (batch && (!rows_in || !rows_out || !first || !length || !keep || !add || (max_add && !slots)))
    return refuse(what, "null request array or slots");
  if (cursors_in == cursors_out) return refuse(what, "cursors_out must differ from cursors_in");
  if (n_rows <= 0 || width <= 0 || n_pages <= 0 || page_size <= 0 || table_stride < width)
    return refuse(what, "rows, width, pages and page size must be positive, table_stride >= width");
  if ((int64_t)width * page_size > INT32_MAX) return refuse(what, "width x page_size exceeds 2^31 - 1 frames");
  PlanArgs p{table, table_stride, n_rows, width, queue, n_pages, page_size, cursors_in, cursors_out, rows_in, rows_out,
             first, length, keep, add, batch, slots, max_add, status};
  return launch_on(device, what, [&] { return launch_plan(p, static_cast<hipStream_t>(stream)); });
}

int tone_frames_slots(int device, const int32_t* table, int64_t table_stride, int n_rows, int width, int n_pages, int page_size,
                      const int32_t* rows, const int32_t* first, const int32_t* begin, const int32_t* count, int batch,
                      int64_t* slots, int max_count, void* stream) {
  const char* what = "tone_frames_slots";
  if (batch < 0 || max_count < 0) return refuse(what, "negative batch or max_count");
  if (batch == 0 || max_count == 0) return TONE_OK;
  if (!table || !rows || !first || !begin || !count || !slots) return refuse(what, "null pointer");
  if (n_rows <= 0 || width <= 0 || n_pages <= 0 || page_size <= 0 || table_stride < width)
    return refuse(what, "rows, width, pages and page size must be positive, table_stride >= width");
  if (((int64_t)max_count + 255) / 256 * batch > INT32_MAX) return refuse(what, "batch x max_count too large for one launch");
  SlotArgs p{table, table_stride, n_rows, width, n_pages, page_size, rows, first, begin, count, batch, slots, max_count};
  return launch_on(device, what, [&] { return launch_slots(p, static_cast<hipStream_t>(stream)); });
}

int tone_frames_put(int device, const void* src, int src_type, int64_t src_stride, const int64_t* slots, int64_t n, int vocab,
                    void* pool, int pool_type, int64_t pool_stride, int64_t pool_rows, void* stream) {
  const char* what = "tone_frames_put";
  if (n < 0 || vocab <= 0 || vocab > (1 << 24) || pool_rows < 0) return refuse(what, "n, vocab or pool_rows out of range");
  if (!known_type(src_type) || !known_type(pool_type)) return refuse(what, "unknown element type");
  if (n == 0) return TONE_OK;
  if (!src || !slots || (!pool && pool_rows)) return refuse(what, "null pointer");
  if (src_stride < vocab || pool_stride < vocab) return refuse(what, "row stride < vocab");
  if (!aligned(src, src_type) || !aligned(pool, pool_type)) return refuse(what, "src or pool not aligned to its element type");
  if ((n + 15) / 16 > INT32_MAX) return refuse(what, "too many rows for one launch");
  PutArgs p{src, src_type, src_stride, slots, n, vocab, pool, pool_type, pool_stride, pool_rows};
  return launch_on(device, what, [&] { return launch_put(p, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
