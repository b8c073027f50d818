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
#include <type_traits>

namespace tone {
namespace {

// n / d for 0 <= n < 2^31 by one multiplication (Granlund and Montgomery, division by invariant integers): m = ceil(2^(31 + l)
// / d), 2^l >= d (m < 2^32; exact over that range)
struct Divisor {
  uint32_t d, m;
  int s;
  explicit Divisor(uint32_t d_) : d(d_), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + d - 1) / d);
    s += 31 - 32;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return d == 1 ? n : __umulhi(n, m) >> s;
  }
};

struct PlanArgs {
  int32_t* table;                       // [n_rows][width], rows `stride` entries apart
  int64_t stride;
  int n_rows, width;
  int32_t* queue;                       // [n_pages]
  int n_pages, page;
  Divisor by_page, by_pages;            // frames to pages; queue positions to rounds of the queue
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
  Divisor by_page;
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

struct Request {
  int first, length, kept, end;         // frames held before: [first, length), after: [kept, end)
  int lo0, hi0, lo1, hi1;               // pages held before / after
  int from;                             // first page taken
  int take, drop;
  bool bad, wide;
};

__device__ __forceinline__ Request read_request(const PlanArgs& p, int b) {
  Request r;
  const int first = p.first[b], length = p.length[b], keep = p.keep[b], add = p.add[b], ri = p.rows_in[b], ro = p.rows_out[b];
  const int64_t end = (int64_t)length + add;
  r.first = first;
  r.length = length;
  r.kept = max(first, keep);
  r.end = (int)end;
  r.bad = first < 0 || first > length || add < 0 || add > p.max_add || keep < 0 || end > INT32_MAX || keep > end || ri < 0 ||
          ri >= p.n_rows || ro < 0 || ro >= p.n_rows || ri == ro;
  if (r.bad) {
    r.lo0 = r.hi0 = r.lo1 = r.hi1 = r.from = 0;
    r.take = r.drop = 0;
    r.wide = false;
    return r;
  }
  const bool had = first < length, has = r.kept < r.end;
  r.lo0 = p.by_page(first);
  r.hi0 = had ? p.by_page(length - 1) + 1 : r.lo0;
  r.lo1 = p.by_page(r.kept);
  r.hi1 = has ? p.by_page(r.end - 1) + 1 : r.lo1;
  r.from = had ? max(r.hi0, r.lo1) : r.lo1;
  r.take = has ? r.hi1 - r.from : 0;
  r.drop = had ? (has ? min(r.lo1, r.hi0) : r.hi0) - r.lo0 : 0;
  r.wide = r.hi1 - r.lo1 > p.width || r.hi0 - r.lo0 > p.width;
  return r;
}

// One launch: every workgroup adds up the pages of all requests (24 bytes each, out of L2) to place its own ones, instead of a
// scan kernel in front of a writing kernel.  blockIdx.x: WAVES / per requests of `per` waves each, so that a request's chain
// of dependent loads (its row, its pages, its slots) is walked by all of them at once; blockIdx.y: a share of the slots.
// All requests are read by every workgroup: 65,536 take 0.86 ms and 262,144 20 ms, so TONE_FRAMES_MAX_BATCH is the end.
// What bounds fewer is that chain: everything that does not depend on the sums is loaded in front of them.  4096 streams that
// append 10 frames each (1.2 MB) take 12.0 us, 96 recordings of up to 18,000 frames (14 MB of slots) 10.6, one stream 4.6.
template <int WAVES>
__global__ void __launch_bounds__(64 * WAVES) plan_kernel(PlanArgs p, int per) {
  __shared__ int64_t part[WAVES][4];
  __shared__ int s_take[WAVES], s_drop[WAVES];
  __shared__ int s_flags;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), rows = WAVES / per, r0 = blockIdx.x * rows, r1 = min(p.batch, r0 + rows);
  const int mine = wave / per, own = r0 + mine, at = (wave - mine * per) * 64 + (tid & 63), step = 64 * per;
  const int64_t head = p.cursors_in[0], tail = p.cursors_in[1];
  Request r;
  int ri = -1, ro = -1;
  if (own < r1) {
    r = read_request(p, own);
    ri = p.rows_in[own];
    ro = p.rows_out[own];
  }
  if (tid == 0) s_flags = 0;
  __syncthreads();
  int64_t v[4] = {0, 0, 0, 0};          // taken by all / by those before r0; released likewise
  int flags = 0;
#pragma unroll 4
  for (int b = tid; b < p.batch; b += 64 * WAVES) {
    const Request q = read_request(p, b);
    flags |= (q.wide ? TONE_FRAMES_ROW_FULL : 0) | (q.bad ? TONE_FRAMES_BAD_REQUEST : 0);
    v[0] += q.take;
    v[2] += q.drop;
    v[1] += b < r0 ? q.take : 0;
    v[3] += b < r0 ? q.drop : 0;
  }
  if (own < r1 && at == 0) {
    s_take[mine] = r.take;
    s_drop[mine] = r.drop;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    for (int o = 32; o; o >>= 1) v[i] += __shfl_xor(v[i], o);
    if ((tid & 63) == 0) part[wave][i] = v[i];
  }
  if (flags) atomicOr(&s_flags, flags);
  __syncthreads();
  flags = s_flags;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v[i] += part[w][i];
  }
  // free + released <= n_pages holds for every state these calls produce; anything else is not a queue of this pool
  // (tail - head by itself first: cursors near 2^63 would pass the sum's end)
  if (head < 0 || tail < head || tail - head > p.n_pages || tail - head + v[2] > p.n_pages) flags |= TONE_FRAMES_BAD_QUEUE;
  else if (v[0] > tail - head) flags |= TONE_FRAMES_NO_PAGES;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) {
    p.cursors_out[0] = head + (flags ? 0 : v[0]);
    p.cursors_out[1] = tail + (flags ? 0 : v[2]);
    p.status[0] = flags;
  }
  if (own >= r1) return;
  const int seg = (p.max_add + gridDim.y - 1) / gridDim.y, s0 = min(p.max_add, (int)blockIdx.y * seg), s1 = min(p.max_add, s0 + seg);
  int64_t* slots = p.slots + (int64_t)own * p.max_add;
  if (flags) {
    for (int j = s0 + at; j < s1; j += step) slots[j] = -1;
    if (blockIdx.y == 0 && ri >= 0 && ri < p.n_rows && ro >= 0 && ro < p.n_rows && ri != ro)
      for (int j = at; j < p.width; j += step) p.table[ro * p.stride + j] = p.table[ri * p.stride + j];
    return;
  }
  // positions in the queue, modulo n_pages once: both are below 2 n_pages, as taken <= free and free + released <= n_pages
  // (a 64-bit remainder takes a microsecond; cursors stay below 2^31 for years of 4096 streams)
  int64_t take = head <= INT32_MAX ? (int)head - p.by_pages((uint32_t)head) * p.n_pages : head % p.n_pages;
  int64_t drop = take + (tail - head);
  if (drop >= p.n_pages) drop -= p.n_pages;
  take += v[1];
  drop += v[3];
  for (int i = 0; i < mine; ++i) {
    take += s_take[i];
    drop += s_drop[i];
  }
  const int32_t* before = p.table + ri * p.stride;
  // page of logical page lp: kept from the old row, or the next entry of the queue
  auto page_of = [&](int lp) -> int32_t {
    if (lp < r.hi0 && r.hi0 > r.lo0) return before[lp - r.lo0];
    int64_t i = take + (lp - r.from);
    if (i >= p.n_pages) i -= p.n_pages;
    return p.queue[i];
  };
  if (blockIdx.y == 0) {
    int32_t* after = p.table + ro * p.stride;
    for (int j = at; j < p.width; j += step) after[j] = r.lo1 + j < r.hi1 ? page_of(r.lo1 + j) : -1;
    for (int j = at; j < r.drop; j += step) {
      int64_t i = drop + j;
      if (i >= p.n_pages) i -= p.n_pages;
      p.queue[i] = before[j];
    }
  }
  const int new_end = min(s1, r.end - r.length);
  for (int j = s0 + at; j < s1; j += step) {
    int64_t slot = -1;
    const int f = r.length + j;
    if (j < new_end && f >= r.kept) {
      const int q = p.by_page(f);
      const int32_t pg = page_of(q);
      if (pg >= 0 && pg < p.n_pages) slot = (int64_t)pg * p.page + (f - q * p.page);
    }
    slots[j] = slot;
  }
}

// A thread per slot: its request, then its page.  187 frames take 1.9 us, a launch's time.
__global__ void __launch_bounds__(256) slots_kernel(SlotArgs p, int segs) {
  const int b = blockIdx.x / segs;
  const int j = (blockIdx.x - b * segs) * 256 + threadIdx.x;
  if (j >= p.max_count) return;
  const int row = p.rows[b], first = p.first[b], count = p.count[b];
  const int64_t f = (int64_t)p.begin[b] + j;
  int64_t slot = -1;
  if (row >= 0 && row < p.n_rows && first >= 0 && j < count && f >= first && f <= INT32_MAX) {
    const int q = p.by_page((uint32_t)f), at = q - (int)p.by_page(first);
    if (at < p.width) {
      const int32_t pg = p.table[row * p.stride + at];
      if (pg >= 0 && pg < p.n_pages) slot = (int64_t)pg * p.page + ((int)f - q * p.page);
    }
  }
  p.slots[(int64_t)b * p.max_count + j] = slot;
}

constexpr int kPutEach = 8;                          // entries a thread has in flight
constexpr int kPutChunk = 256 * kPutEach;

// Entries kPutChunk * blockIdx.x ... of the rows laid end to end: consecutive lanes copy consecutive entries of a row, all of
// a thread's loads are issued before its first store, and the rows' slots come from LDS.  Memory bounds it: 1.73 M rows of 35
// fp32 entries into an fp16 pool (377 MB) take 95 us, 4.0 TB/s where a copy reaches 4.5; 40,960 rows fp32 to fp32 4.5 us.
template <typename S, typename D>
__global__ void __launch_bounds__(256) put_kernel(const S* __restrict__ src, int64_t src_stride, const int64_t* __restrict__ slots,
                                                  int64_t n, Divisor by_vocab, D* __restrict__ pool, int64_t pool_stride, int64_t pool_rows) {
  __shared__ int64_t s_slot[kPutChunk + 1];
  const int vocab = by_vocab.d;
  const int64_t e0 = (int64_t)blockIdx.x * kPutChunk, row0 = e0 / vocab;
  const int c0 = (int)(e0 - row0 * vocab), entries = (int)min((int64_t)kPutChunk, n * vocab - e0);
  const int rows = by_vocab(c0 + entries - 1) + 1;   // at most kPutChunk + 1 (vocab 1: kPutChunk)
  for (int r = threadIdx.x; r < rows; r += 256) s_slot[r] = slots[row0 + r];
  float v[kPutEach];
#pragma unroll
  for (int i = 0; i < kPutEach; ++i) {
    const int e = i * 256 + threadIdx.x;
    if (e < entries) {
      const int r = by_vocab(c0 + e);
      v[i] = load_elem(src + (row0 + r) * src_stride + (c0 + e - r * vocab));
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPutEach; ++i) {
    const int e = i * 256 + threadIdx.x;
    if (e < entries) {
      const int r = by_vocab(c0 + e);
      const int64_t s = s_slot[r];
      if (s >= 0 && s < pool_rows) store_elem(pool + s * pool_stride + (c0 + e - r * vocab), v[i]);
    }
  }
}

template <typename S>
hipError_t put_from(const PutArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((a.n * a.vocab + kPutChunk - 1) / kPutChunk));
  const S* src = static_cast<const S*>(a.src);
  const Divisor by(a.vocab);
  switch (a.pool_type) {
    case TONE_TYPE_FP32:
      hipLaunchKernelGGL((put_kernel<S, float>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, by, static_cast<float*>(a.pool),
                         a.pool_stride, a.pool_rows);
      break;
    case TONE_TYPE_FP16:
      hipLaunchKernelGGL((put_kernel<S, __half>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, by, static_cast<__half*>(a.pool),
                         a.pool_stride, a.pool_rows);
      break;
    default:
      hipLaunchKernelGGL((put_kernel<S, Bf16>), grid, dim3(256), 0, st, src, a.src_stride, a.slots, a.n, by, static_cast<Bf16*>(a.pool),
                         a.pool_stride, a.pool_rows);
  }
  return hipGetLastError();
}

hipError_t launch_plan(const PlanArgs& p, hipStream_t st) {
  // Every workgroup passes over all requests, so the more there are, the more waves share a pass and the fewer waves a request
  // gets; long slot rows are cut in pieces.  us with 4 / 8 / 16 waves per workgroup, 10 frames each: 96 requests 5.5 / 5.7 /
  // 7.3, 512 6.5 / 6.5 / 8.6, 1024 7.8 / 7.4 / 9.9, 2048 10.8 / 8.8 / 11.0, 4096 19.0 / 13.6 / 12.6; 96 of 18,000: 10.6 / 12.4.
  const auto go = [&](auto waves) {
    constexpr int W = decltype(waves)::value;
    int per = 1;
    while (per < W && (int64_t)p.batch * per < W * 256) per *= 2;
    const int rows = W / per, gx = std::max(1, (p.batch + rows - 1) / rows);   // an empty batch still writes the cursors and the status
    const int gy = std::max(1, std::min(2048 / gx, (p.max_add + 64 * per * 4 - 1) / (64 * per * 4)));
    hipLaunchKernelGGL(plan_kernel<W>, dim3(gx, gy), dim3(64 * W), 0, st, p, per);
  };
  if (p.batch <= 512) go(std::integral_constant<int, 4>{});
  else if (p.batch <= 2048) go(std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 16>{});
  return hipGetLastError();
}

hipError_t launch_slots(const SlotArgs& p, hipStream_t st) {
  const int segs = (p.max_count + 255) / 256;
  hipLaunchKernelGGL(slots_kernel, dim3((unsigned)segs * (unsigned)p.batch), dim3(256), 0, st, p, segs);
  return hipGetLastError();
}

// Whether the rows of src and the pool share memory.  Rows are copied in no order, so a row that is read and written would be
// torn; columns side by side in rows of one length are apart.
bool meet(const void* src, int src_type, int64_t src_stride, int64_t n, const void* pool, int pool_type, int64_t pool_stride,
          int64_t pool_rows, int vocab) {
  if (pool_rows == 0) return false;
  using Wide = __int128;                 // strides are the caller's: no product below can overflow
  const auto size = [](int type) { return type == TONE_TYPE_FP32 ? 4 : 2; };
  const Wide row = (Wide)vocab * size(src_type), pool_row = (Wide)vocab * size(pool_type);
  Wide pitch = (Wide)src_stride * size(src_type);
  const Wide pool_pitch = (Wide)pool_stride * size(pool_type);
  const Wide at = (Wide) reinterpret_cast<uintptr_t>(src) - (Wide) reinterpret_cast<uintptr_t>(pool);
  if (at >= (pool_rows - 1) * pool_pitch + pool_row || at + (n - 1) * pitch + row <= 0) return false;
  if (n == 1) pitch = pool_pitch;
  else if (pool_rows > 1 && pitch != pool_pitch) return true;
  const Wide in = (at % pitch + pitch) % pitch;
  return !(in >= pool_row && in + row <= pitch);
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
  if (max_add > kMaxFrames || batch > TONE_FRAMES_MAX_BATCH) return refuse(what, "batch or max_add too large for one launch");
  if (!table || !queue || !cursors_in || !cursors_out || !status) return refuse(what, "null table, queue, cursors or status");
  if (batch && (!rows_in || !rows_out || !first || !length || !keep || !add || (max_add && !slots)))
    return refuse(what, "null request array or slots");
  if (cursors_in < cursors_out + 2 && cursors_out < cursors_in + 2) return refuse(what, "cursors_out overlaps cursors_in");
  if (n_rows <= 0 || width <= 0 || n_pages <= 0 || page_size <= 0 || table_stride < width)
    return refuse(what, "rows, width, pages and page size must be positive, table_stride >= width");
  if ((int64_t)width * page_size > INT32_MAX) return refuse(what, "width x page_size exceeds 2^31 - 1 frames");
  PlanArgs p{table, table_stride, n_rows, width, queue, n_pages, page_size, Divisor(page_size), Divisor(n_pages), cursors_in, cursors_out, rows_in, rows_out,
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
  if (max_count > kMaxFrames || ((int64_t)max_count + 255) / 256 * batch > kMaxThreads / 256) return refuse(what, "batch x max_count too large for one launch");
  SlotArgs p{table, table_stride, n_rows, width, n_pages, page_size, Divisor(page_size), rows, first, begin, count, batch, slots, max_count};
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
  if (n > (kMaxThreads / 256 - 1) * kPutChunk / vocab) return refuse(what, "too many rows for one launch");
  if (meet(src, src_type, src_stride, n, pool, pool_type, pool_stride, pool_rows, vocab)) return refuse(what, "src overlaps the pool");
  PutArgs p{src, src_type, src_stride, slots, n, vocab, pool, pool_type, pool_stride, pool_rows};
  return launch_on(device, what, [&] { return launch_put(p, static_cast<hipStream_t>(stream)); });
}

}  // extern "C"
