// dash_pool.cu -- pages of a block-paged cache: copied, shared (forked), freed
// and compacted, and the accepted tokens of a draft moved to the front.
//
// Moving data: one launch for up to kMaxTensors tensors (all layers), whose
// descriptors travel in the kernel's arguments; bound by memory traffic (every
// byte read once and written once).  Page tables: one CTA walks the requests
// in order, so what pages a request gets depends on nothing but the state and
// the requests; counts are integers and every page's fate is decided by its
// final count, not by the order of the atomics that made it.
//
// Measured (CUDA graph): compaction of 1.1 GB of traffic in 12 layers 195 us (5.7 TB/s; a plain
// copy 6.5), 64 forks with 243 MB of copied pages and their freeing 46 us, 2 forks
// 12.4 us and a commit of 8 sequences 8.4 us (bound by launches and dependent loads).
// The copy's CTAs take their places while the tables are still worked on
// (programmatic dependent launch: fork 14.4 -> 12.4 us).
#include "dash_common.cuh"
#include "dash_internal.h"

namespace dash {
namespace {

constexpr int kMaxTensors = 64;

struct TensorDesc {
  uint8_t* base;
  int64_t page_stride, tok_stride;
  int32_t tok_bytes, page_toks;
  int32_t log_vec;      // log2 of the bytes moved per access
  int32_t first;        // first work item of this tensor (per pair)
};

struct TensorSet {
  TensorDesc t[kMaxTensors];
  int n;
  int items;            // work items per pair, all tensors
};

template <typename V>
__device__ __forceinline__ V ld(const uint8_t* p) { return *reinterpret_cast<const V*>(p); }
template <typename V>
__device__ __forceinline__ void st(uint8_t* p, V v) { *reinterpret_cast<V*>(p) = v; }

constexpr int kCopyThreads = 256;
constexpr int kCopyBatch = 4;          // accesses in flight per thread

// the part [first, first + kCopyThreads * kCopyBatch) of a page's accesses
template <typename V>
__device__ __forceinline__ void copy_item(const TensorDesc& t, int64_t src, int64_t dst, int item) {
  const int per_tok = t.tok_bytes / (int)sizeof(V);
  const int total = per_tok * t.page_toks;
  const uint8_t* s = t.base + src * t.page_stride;
  uint8_t* d = t.base + dst * t.page_stride;
  V x[kCopyBatch];
  int64_t off[kCopyBatch];
#pragma unroll
  for (int k = 0; k < kCopyBatch; ++k) {
    const int e = (item * kCopyBatch + k) * kCopyThreads + threadIdx.x;
    off[k] = -1;
    if (e < total) {
      off[k] = t.page_toks == 1 ? (int64_t)e * (int)sizeof(V)
                                : (int64_t)(e / per_tok) * t.tok_stride + (int64_t)(e % per_tok) * (int)sizeof(V);
      x[k] = ld<V>(s + off[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kCopyBatch; ++k)
    if (off[k] >= 0) st<V>(d + off[k], x[k]);
}

__device__ __forceinline__ int find_tensor(const TensorSet& ts, int item) {
  int lo = 0, hi = ts.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ts.t[mid].first <= item) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Inclusive sum over the CTA (blockDim.x a multiple of 32, <= 1024); every
// thread gets its own prefix and the total.
__device__ int block_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = lane < nw ? s_warp[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = s_warp[nw - 1];
  const int r = v + (warp ? s_warp[warp - 1] : 0);
  __syncthreads();
  return r;
}

constexpr int kPoolThreads = 1024;

}  // namespace

// ---------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------
// A block table whose pages get new ids while their data moves (compaction).
struct TableMap {
  const int32_t* from;
  int32_t* to;
  const int32_t* new_id;
  int64_t from_stride, to_stride;
  int32_t rows, width;
};
constexpr int kMapBlocks = 32;

__global__ void __launch_bounds__(kCopyThreads) pages_copy_kernel(const __grid_constant__ TensorSet ts,
                                                                  const int32_t* src, const int32_t* dst, int n,
                                                                  const int32_t* count, int64_t num_pages,
                                                                  const __grid_constant__ TableMap tm) {
  // starts while the kernel that writes the pairs runs
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the table's entries, in the first CTAs, beside the copies
  if (tm.rows && blockIdx.x < kMapBlocks) {
    const int64_t entries = (int64_t)tm.rows * tm.width;
#pragma unroll 4
    for (int64_t e = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; e < entries;
         e += (int64_t)kMapBlocks * kCopyThreads) {
      const int row = (int)(e / tm.width), col = (int)(e - (int64_t)row * tm.width);
      const int page = tm.from[row * tm.from_stride + col];
      tm.to[row * tm.to_stride + col] = page >= 0 && page < num_pages ? tm.new_id[page] : page;
    }
  }
  const int live = count ? min(n, *count) : n;
  const int64_t units = (int64_t)live * ts.items;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int pair = (int)(u / ts.items), it = (int)(u - (int64_t)pair * ts.items);
    const int64_t s = src[pair], d = dst[pair];
    if (s < 0 || d < 0 || s == d || s >= num_pages || d >= num_pages) continue;
    const TensorDesc& t = ts.t[find_tensor(ts, it)];
    const int item = it - t.first;
    switch (t.log_vec) {
      case 4: copy_item<uint4>(t, s, d, item); break;
      case 3: copy_item<uint2>(t, s, d, item); break;
      case 2: copy_item<uint32_t>(t, s, d, item); break;
      case 1: copy_item<uint16_t>(t, s, d, item); break;
      default: copy_item<uint8_t>(t, s, d, item);
    }
  }
}

// The pairs that may run at the same time: no destination is another pair's
// source or destination.  Of two pairs a -> b, b -> c both are left out: the second
// reads what the first was to write, and which of them was meant to come first is
// not known.  One CTA; three bit sets over the pages (destination
// once, destination more than once, source) in shared memory.
__global__ void __launch_bounds__(kPoolThreads) pages_check_kernel(const int32_t* src, const int32_t* dst, int n,
                                                                   const int32_t* count, int num_pages, int32_t* list,
                                                                   DeviceError* err) {
  extern __shared__ uint32_t s_bits[];
  asm volatile("griddepcontrol.launch_dependents;");          // the copy's CTAs may take their places
  const int words = (num_pages + 31) / 32;
  uint32_t *once = s_bits, *more = s_bits + words, *from = s_bits + 2 * words;
  const int live = count ? min(n, *count) : n;
  for (int w = threadIdx.x; w < 3 * words; w += kPoolThreads) s_bits[w] = 0u;
  __syncthreads();
  auto valid = [&](int s, int d) { return s >= 0 && d >= 0 && s != d && s < num_pages && d < num_pages; };
  for (int i = threadIdx.x; i < live; i += kPoolThreads) {
    const int s = src[i], d = dst[i];
    if (!valid(s, d)) continue;
    const uint32_t bit = 1u << (d & 31);
    if (atomicOr(once + (d >> 5), bit) & bit) atomicOr(more + (d >> 5), bit);
    atomicOr(from + (s >> 5), 1u << (s & 31));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPoolThreads) {
    int s = i < live ? src[i] : -1, d = i < live ? dst[i] : -1;
    bool ok = i < live && valid(s, d);
    if (i < live && (s >= num_pages || d >= num_pages)) record_error(err, DASH_DEV_BAD_ROW, 90, max(s, d));
    if (ok) {
      const bool clash = ((more[d >> 5] | from[d >> 5]) >> (d & 31)) & 1u || ((once[s >> 5] >> (s & 31)) & 1u);
      if (clash) record_error(err, DASH_DEV_BAD_ROW, 91, d);
      ok = !clash;
    }
    list[i] = ok ? s : -1;
    list[n + i] = ok ? d : -1;
  }
}

// ---------------------------------------------------------------------------
// accepted tokens to the front
// ---------------------------------------------------------------------------
constexpr int kCommitThreads = 128;
constexpr int kCommitNodes = 256;
constexpr int kCommitBatch = 8;

// A thread owns one access column of a sequence's tokens in one tensor and
// moves its tokens in order, kCommitBatch loads before their stores.  path
// rises strictly, so path[i] >= i and a source is never the target of an
// earlier move; threads never touch each other's bytes.
template <typename V>
__device__ void commit_column(const TensorDesc& t, const int64_t* s_src, const int64_t* s_dst, int n, int bs, int col) {
  const int64_t c = (int64_t)col * (int)sizeof(V);
  for (int i0 = 0; i0 < n; i0 += kCommitBatch) {
    V x[kCommitBatch];
#pragma unroll
    for (int k = 0; k < kCommitBatch; ++k) {
      const int64_t sl = i0 + k < n ? s_src[i0 + k] : -1;
      if (sl >= 0) x[k] = ld<V>(t.base + (sl / bs) * t.page_stride + (sl % bs) * t.tok_stride + c);
    }
#pragma unroll
    for (int k = 0; k < kCommitBatch; ++k) {
      const int64_t dl = i0 + k < n ? s_dst[i0 + k] : -1;
      if (dl >= 0) st<V>(t.base + (dl / bs) * t.page_stride + (dl % bs) * t.tok_stride + c, x[k]);
    }
  }
}

__global__ void __launch_bounds__(kCommitThreads) draft_commit_kernel(const __grid_constant__ TensorSet ts,
                                                                      const DashCommitArgs a) {
  __shared__ int64_t s_src[kCommitNodes], s_dst[kCommitNodes];
  __shared__ int s_n;
  const int s = blockIdx.y, bs = a.block_size;
  const int acc = min(a.n_accept[s], a.max_nodes - 1);
  if (acc <= 0) return;
  if (threadIdx.x == 0) s_n = acc;
  __syncthreads();
  const int ctx = a.ctx_len[s];
  const int32_t* path = a.path + (int64_t)s * a.path_stride;
  const int32_t* bt = a.block_table + (int64_t)s * a.bt_stride;
  for (int i = threadIdx.x + 1; i <= acc; i += kCommitThreads) {
    const int p = path[i], q = i > 1 ? path[i - 1] : 0;
    if (p <= q || p >= a.max_nodes || ctx < 0 || ctx > INT32_MAX - kCommitNodes) {
      if (blockIdx.x == 0) record_error(a.device_error, DASH_DEV_BAD_TREE, 92, p);
      atomicMin(&s_n, i - 1);
      continue;
    }
    // p == i: the token is where it belongs already
    const int bf = (ctx + p) / bs, bd = (ctx + i) / bs;
    const int64_t pf = bf < a.bt_width ? (int64_t)bt[bf] : -1, pd = bd < a.bt_width ? (int64_t)bt[bd] : -1;
    bool ok = pf >= 0 && pd >= 0 && pf < a.num_pages && pd < a.num_pages;
    if (!ok && blockIdx.x == 0)
      record_error(a.device_error, DASH_DEV_BAD_PAGE, 93, pf < 0 || pf >= a.num_pages ? pf : pd);
    ok = ok && p != i;
    s_src[i - 1] = ok ? pf * bs + (ctx + p) % bs : -1;
    s_dst[i - 1] = ok ? pd * bs + (ctx + i) % bs : -1;
  }
  __syncthreads();
  const int n = s_n;
  // column of the whole set of tensors -> (tensor, column)
  const int item = blockIdx.x * kCommitThreads + threadIdx.x;
  if (item >= ts.items) return;
  const TensorDesc& t = ts.t[find_tensor(ts, item)];
  const int col = item - t.first;
  switch (t.log_vec) {
    case 4: commit_column<uint4>(t, s_src, s_dst, n, bs, col); break;
    case 3: commit_column<uint2>(t, s_src, s_dst, n, bs, col); break;
    case 2: commit_column<uint32_t>(t, s_src, s_dst, n, bs, col); break;
    case 1: commit_column<uint16_t>(t, s_src, s_dst, n, bs, col); break;
    default: commit_column<uint8_t>(t, s_src, s_dst, n, bs, col);
  }
}

// ---------------------------------------------------------------------------
// page tables
// ---------------------------------------------------------------------------
// first[row] = lowest request naming the row (shared memory, max_rows ints)
__device__ void first_requests(int* first, const int32_t* rows, int n, int max_rows) {
  for (int r = threadIdx.x; r < max_rows; r += kPoolThreads) first[r] = INT32_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPoolThreads)
    if (rows[i] >= 0 && rows[i] < max_rows) atomicMin(first + rows[i], i);
  __syncthreads();
}

// a row's blocks, inside the table's row
__device__ __forceinline__ int held_blocks(const DashPagePool& p, int row) {
  return min(max(p.n_blocks[row], 0), p.bt_width);
}

// page popped as the k-th of this call, or -1 when the stack does not hold it
__device__ __forceinline__ int pop_page(const DashPagePool& p, int n_free, int k) {
  const int at = n_free - 1 - k;
  if (at < 0) return -1;
  const int page = p.free_list[at];
  return page >= 0 && page < p.num_pages ? page : -1;
}

__global__ void __launch_bounds__(kPoolThreads) pages_reserve_kernel(const DashPagesArgs a) {
  extern __shared__ int s_first[];
  __shared__ int s_warp[32];
  __shared__ int4 s_req[kPoolThreads];
  const DashPagePool& p = a.pool;
  first_requests(s_first, a.rows, a.n, p.max_rows);
  const int n_free = min(max(*p.n_free, 0), p.num_pages);
  int taken = 0;                                   // pages asked for by the requests before this slice
  int used = 0;                                    // pages given out
  for (int i0 = 0; i0 < a.n; i0 += kPoolThreads) {
    const int i = i0 + threadIdx.x;
    int row = -1, have = 0, add = 0;
    if (i < a.n) {
      row = a.rows[i];
      const int len = a.lens[i];
      const bool fits = row >= 0 && row < p.max_rows && s_first[row] == i && len >= 0 &&
                        (len + (int64_t)p.block_size - 1) / p.block_size <= p.bt_width;
      if (!fits) {
        record_error(a.device_error, DASH_DEV_BAD_ROW, 94, row);
        row = -1;
      } else {
        have = held_blocks(p, row);
        // (more than all pages is one too many, so that the sums stay small)
        add = min(max(0, (int)((len + (int64_t)p.block_size - 1) / p.block_size) - have), p.num_pages + 1);
      }
    }
    int total;
    const int end = taken + block_scan(add, s_warp, total);
    const bool got = add > 0 && end <= n_free;
    if (add > 0 && !got) record_error(a.device_error, DASH_DEV_NO_PAGE, 95, row);
    if (got) p.n_blocks[row] = have + add;
    s_req[threadIdx.x] = make_int4(got ? row : -1, have, add, end - add);
    int given;
    block_scan(got ? add : 0, s_warp, given);      // also orders s_req
    used += given;
    taken = min(taken + total, p.num_pages + 1);
    // a warp per request writes its pages
    for (int u = threadIdx.x >> 5; u < min(kPoolThreads, a.n - i0); u += kPoolThreads / 32) {
      const int4 rq = s_req[u];
      if (rq.x < 0) continue;
      for (int k = threadIdx.x & 31; k < rq.z; k += 32) {
        const int page = pop_page(p, n_free, rq.w + k);
        p.block_table[(int64_t)rq.x * p.bt_stride + rq.y + k] = page;
        if (page >= 0) p.ref[page] = 1;
        p.free_list[n_free - 1 - (rq.w + k)] = -1;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.n_free = n_free - used;
}

__global__ void __launch_bounds__(kPoolThreads) pages_fork_kernel(const DashPagesArgs a) {
  extern __shared__ int s_first[];
  __shared__ int s_warp[32];
  __shared__ int4 s_req[kPoolThreads];
  asm volatile("griddepcontrol.launch_dependents;");          // the copy's CTAs may take their places
  const DashPagePool& p = a.pool;
  const int bs = p.block_size;
  first_requests(s_first, a.rows, a.n, p.max_rows);
  const int n_free = min(max(*p.n_free, 0), p.num_pages);
  int taken = 0, used = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPoolThreads) {
    const int i = i0 + threadIdx.x;
    int dst = -1, src = -1, full = 0, part = 0;
    if (i < a.n) {
      dst = a.rows[i];
      src = a.src[i];
      const int len = a.lens[i];
      // a src that is a dst of this call too is refused, so no request
      // depends on another's row
      const bool ok = dst >= 0 && dst < p.max_rows && s_first[dst] == i && src >= 0 && src < p.max_rows &&
                      len >= 0 && s_first[src] == INT32_MAX && p.n_blocks[dst] == 0 &&
                      (len + (int64_t)bs - 1) / bs <= held_blocks(p, src);
      if (!ok) {
        record_error(a.device_error, DASH_DEV_BAD_ROW, 96, dst);
        dst = -1;
      } else {
        full = len / bs;
        part = len % bs ? 1 : 0;
      }
    }
    int total;
    const int end = taken + block_scan(part, s_warp, total);
    const bool got = dst >= 0 && (!part || end <= n_free);
    if (dst >= 0 && !got) record_error(a.device_error, DASH_DEV_NO_PAGE, 97, dst);
    int from = -1, to = -1;
    if (got) {
      if (part) {
        from = p.block_table[(int64_t)src * p.bt_stride + full];
        to = pop_page(p, n_free, end - 1);
        p.block_table[(int64_t)dst * p.bt_stride + full] = to;
        if (to >= 0) p.ref[to] = 1;
        p.free_list[n_free - end] = -1;
      }
      p.n_blocks[dst] = full + part;
    }
    s_req[threadIdx.x] = make_int4(got ? dst : -1, src, full, 0);
    if (i < a.n) {
      a.copy_src[i] = from;
      a.copy_dst[i] = to;
    }
    int given;
    block_scan(got ? part : 0, s_warp, given);     // also orders s_req
    used += given;
    taken += total;
    // a warp per request shares the full pages
    for (int u = threadIdx.x >> 5; u < min(kPoolThreads, a.n - i0); u += kPoolThreads / 32) {
      const int4 rq = s_req[u];
      if (rq.x < 0) continue;
      for (int b = threadIdx.x & 31; b < rq.z; b += 32) {
        const int page = p.block_table[(int64_t)rq.y * p.bt_stride + b];
        p.block_table[(int64_t)rq.x * p.bt_stride + b] = page;
        if (page >= 0 && page < p.num_pages) atomicAdd(p.ref + page, 1);
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *p.n_free = n_free - used;
}

// set bits of the words before word w, w < words, in place of the words' counts
__device__ void scan_words(const uint32_t* bits, int* before, int words, int* s_warp) {
  int base = 0;
  for (int w0 = 0; w0 < words; w0 += kPoolThreads) {
    const int w = w0 + threadIdx.x;
    const int c = w < words ? __popc(bits[w]) : 0;
    int total;
    const int end = block_scan(c, s_warp, total);
    if (w < words) before[w] = base + end - c;
    base += total;
  }
  if (threadIdx.x == 0) before[words] = base;
  __syncthreads();
}

__global__ void __launch_bounds__(kPoolThreads) pages_free_kernel(const DashPagesArgs a) {
  extern __shared__ int s_first[];                 // [max_rows], then the freed pages' bits and prefix sums
  __shared__ int s_warp[32];
  const DashPagePool& p = a.pool;
  const int words = (p.num_pages + 31) / 32;
  uint32_t* freed = reinterpret_cast<uint32_t*>(s_first + p.max_rows);
  int* before = s_first + p.max_rows + words;
  for (int w = threadIdx.x; w < words; w += kPoolThreads) freed[w] = 0u;
  first_requests(s_first, a.rows, a.n, p.max_rows);
  const int n_free = min(max(*p.n_free, 0), p.num_pages);
  // a warp per request
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = warp; i < a.n; i += kPoolThreads / 32) {
    const int row = a.rows[i];
    const int keep = a.lens ? a.lens[i] : 0;
    if (row < 0 || row >= p.max_rows || s_first[row] != i || keep < 0) {
      if (lane == 0) record_error(a.device_error, DASH_DEV_BAD_ROW, 98, row);
      continue;
    }
    const int have = held_blocks(p, row);
    for (int b = keep + lane; b < have; b += 32) {
      int32_t* e = p.block_table + (int64_t)row * p.bt_stride + b;
      const int page = *e;
      *e = -1;
      if (page < 0 || page >= p.num_pages) continue;
      const int was = atomicSub(p.ref + page, 1);
      if (was == 1) {
        atomicOr(freed + (page >> 5), 1u << (page & 31));
      } else if (was <= 0) {                       // not held: the count stays at 0
        atomicAdd(p.ref + page, 1);
        record_error(a.device_error, DASH_DEV_BAD_ROW, 99, page);
      }
    }
    __syncwarp();
    if (lane == 0 && keep < have) p.n_blocks[row] = keep;
  }
  __syncthreads();
  scan_words(freed, before, words, s_warp);
  const int n = min(before[words], p.num_pages - n_free);
  for (int w = threadIdx.x; w < words; w += kPoolThreads) {
    int at = before[w];
    for (uint32_t m = freed[w]; m; m &= m - 1, ++at)
      if (at < n) p.free_list[n_free + at] = w * 32 + __ffs(m) - 1;
  }
  if (threadIdx.x == 0) *p.n_free = n_free + n;
}

__global__ void __launch_bounds__(kPoolThreads) pages_compact_kernel(const DashPagesArgs a) {
  extern __shared__ int s_mem[];                   // held pages' bits, prefix sums
  __shared__ int s_warp[32];
  asm volatile("griddepcontrol.launch_dependents;");          // the copy's CTAs may take their places
  const DashPagePool &p = a.pool, &q = a.into;
  const int P = p.num_pages, words = (P + 31) / 32;
  uint32_t* held = reinterpret_cast<uint32_t*>(s_mem);
  int* before = s_mem + words;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int w = warp; w < words; w += kPoolThreads / 32) {
    const int page = w * 32 + lane;
    const uint32_t m = __ballot_sync(0xffffffffu, page < P && p.ref[page] > 0);
    if (lane == 0) held[w] = m;
  }
  __syncthreads();
  scan_words(held, before, words, s_warp);
  const int L = before[words];
  auto rank = [&](int page) { return before[page >> 5] + __popc(held[page >> 5] & ((1u << (page & 31)) - 1u)); };
  auto on = [&](int page) { return (held[page >> 5] >> (page & 31)) & 1u; };
  const int at_L = L < P ? rank(L) : L;            // held pages below L
  const int moves = L - at_L;
  for (int page = threadIdx.x; page < P; page += kPoolThreads) {
    if (page < L && !on(page)) a.copy_dst[page - rank(page)] = page;
    if (page >= L && on(page)) a.copy_src[rank(page) - at_L] = page;
  }
  for (int k = moves + threadIdx.x; k < P / 2; k += kPoolThreads) a.copy_src[k] = a.copy_dst[k] = -1;
  __syncthreads();                                 // the lists are read below (same CTA)
  // counts: a target takes its source's, pages >= L have none
  for (int page = threadIdx.x; page < P; page += kPoolThreads) {
    int c = 0;
    if (page < L) c = on(page) ? p.ref[page] : p.ref[a.copy_src[page - rank(page)]];
    // in place: a source (>= L) is cleared only after every target has read it
    if (page < L) q.ref[page] = c;
  }
  __syncthreads();
  for (int page = threadIdx.x; page < P; page += kPoolThreads) {
    if (page >= L) q.ref[page] = 0;
    q.free_list[page] = page < P - L ? P - 1 - page : -1;
    a.new_id[page] = page >= L && on(page) ? a.copy_dst[rank(page) - at_L] : page;
  }
  for (int r = threadIdx.x; r < p.max_rows; r += kPoolThreads) q.n_blocks[r] = p.n_blocks[r];
  if (threadIdx.x == 0) {
    *q.n_free = P - L;
    *a.n_moves = moves;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
// Descriptors of n tensors; items per pair by `per` (accesses of one tensor ->
// work items).  whole_pages: a page without gaps counts as one entry.
template <typename F>
static void make_set(TensorSet& ts, const DashCacheTensor* t, int n, bool whole_pages, F per) {
  ts.n = n;
  int at = 0;
  for (int i = 0; i < n; ++i) {
    TensorDesc& d = ts.t[i];
    d.base = reinterpret_cast<uint8_t*>(t[i].base);
    d.page_stride = t[i].page_stride;
    d.tok_stride = t[i].tok_stride;
    d.tok_bytes = t[i].tok_bytes;
    d.page_toks = t[i].page_toks;
    if (whole_pages && d.tok_stride == d.tok_bytes) {
      d.tok_bytes *= d.page_toks;
      d.tok_stride = d.tok_bytes;
      d.page_toks = 1;
    }
    // the widest access that every token's start and length allow
    const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(t[i].base) | (uint64_t)d.page_stride |
                         (uint64_t)d.tok_stride | (uint64_t)d.tok_bytes | 16u;
    d.log_vec = 0;
    while (!((all >> d.log_vec) & 1u)) ++d.log_vec;
    d.first = at;
    at += per(d);
  }
  ts.items = at;
}

static int copy_pages(const DashCacheTensor* t, int n_tensors, const int32_t* src, const int32_t* dst, int n,
                      const int32_t* count, int64_t num_pages, const TableMap& tm, cudaStream_t st) {
  TableMap map = tm;
  for (int i0 = 0; i0 < n_tensors; i0 += kMaxTensors) {
    TensorSet ts;
    make_set(ts, t + i0, n_tensors - i0 < kMaxTensors ? n_tensors - i0 : kMaxTensors, true, [](const TensorDesc& d) {
      const int64_t acc = ((int64_t)d.tok_bytes >> d.log_vec) * d.page_toks;
      return (int)((acc + kCopyThreads * kCopyBatch - 1) / (kCopyThreads * kCopyBatch));
    });
    int64_t units = (int64_t)n * ts.items;
    if (map.rows && units < kMapBlocks) units = kMapBlocks;
    if (units == 0) continue;
    const int64_t most = 148 * 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units < most ? units : most));
    cfg.blockDim = dim3(kCopyThreads);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, pages_copy_kernel, ts, src, dst, n, count, num_pages, map);
    if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "pages_copy_kernel launch failed: %s", cudaGetErrorString(e));
    count_launch();
    const int rc = check_launch("pages_copy_kernel");
    if (rc) return rc;
    map.rows = 0;                                  // once
  }
  return DASH_OK;
}

// Shared memory above the default limit (48 KB with a kernel's static part).  The
// limit belongs to the kernel, not to the call: it is set to what the largest pool
// needs, because a call that set its own need would take the limit from under a
// larger one that another thread is about to launch.
constexpr size_t kMaxRows = kPoolMaxRows, kMaxPageWords = kPoolMaxPages / 32;
template <typename K>
static int allow_smem(K kernel, size_t bytes, size_t most, const char* name) {
  if (bytes > 24 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
    return set_error(DASH_ERR_CUDA, "%s: %zu bytes of shared memory refused", name, most);
  return DASH_OK;
}

int launch_pages_copy(const DashPagesCopyArgs& a, cudaStream_t st) {
  if (!a.check) return copy_pages(a.tensors, a.n_tensors, a.src, a.dst, a.n, a.count, a.num_pages, TableMap{}, st);
  const size_t smem = (size_t)((a.num_pages + 31) / 32) * 3 * 4;
  int rc = allow_smem(pages_check_kernel, smem, kMaxPageWords * 3 * 4, "pages_check_kernel");
  if (rc) return rc;
  pages_check_kernel<<<1, kPoolThreads, smem, st>>>(a.src, a.dst, a.n, a.count, (int)a.num_pages, a.list,
                                                    a.device_error);
  count_launch();
  rc = check_launch("pages_check_kernel");
  if (rc) return rc;
  return copy_pages(a.tensors, a.n_tensors, a.list, a.list + a.n, a.n, nullptr, a.num_pages, TableMap{}, st);
}

int launch_draft_commit(const DashCommitArgs& a, cudaStream_t st) {
  for (int i0 = 0; i0 < a.n_tensors; i0 += kMaxTensors) {
    TensorSet ts;
    make_set(ts, a.tensors + i0, a.n_tensors - i0 < kMaxTensors ? a.n_tensors - i0 : kMaxTensors, false,
             [](const TensorDesc& d) { return d.tok_bytes >> d.log_vec; });
    if (ts.items == 0) continue;
    const dim3 grid((unsigned)((ts.items + kCommitThreads - 1) / kCommitThreads), (unsigned)a.n_seq);
    draft_commit_kernel<<<grid, kCommitThreads, 0, st>>>(ts, a);
    count_launch();
    const int rc = check_launch("draft_commit_kernel");
    if (rc) return rc;
  }
  return DASH_OK;
}

int launch_pages_reserve(const DashPagesArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)a.pool.max_rows * 4;
  const int rc = allow_smem(pages_reserve_kernel, smem, kMaxRows * 4, "pages_reserve_kernel");
  if (rc) return rc;
  pages_reserve_kernel<<<1, kPoolThreads, smem, st>>>(a);
  count_launch();
  return check_launch("pages_reserve_kernel");
}

int launch_pages_fork(const DashPagesArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)a.pool.max_rows * 4;
  const int rc = allow_smem(pages_fork_kernel, smem, kMaxRows * 4, "pages_fork_kernel");
  if (rc) return rc;
  pages_fork_kernel<<<1, kPoolThreads, smem, st>>>(a);
  count_launch();
  const int rl = check_launch("pages_fork_kernel");
  return rl || a.n_tensors == 0 ? rl
                                : copy_pages(a.tensors, a.n_tensors, a.copy_src, a.copy_dst, a.n, nullptr,
                                             a.pool.num_pages, TableMap{}, st);
}

int launch_pages_free(const DashPagesArgs& a, cudaStream_t st) {
  const size_t words = (size_t)(a.pool.num_pages + 31) / 32;
  const size_t smem = ((size_t)a.pool.max_rows + 2 * words + 1) * 4;
  const int rc = allow_smem(pages_free_kernel, smem, (kMaxRows + 2 * kMaxPageWords + 1) * 4, "pages_free_kernel");
  if (rc) return rc;
  pages_free_kernel<<<1, kPoolThreads, smem, st>>>(a);
  count_launch();
  return check_launch("pages_free_kernel");
}

int launch_pages_compact(const DashPagesArgs& a, cudaStream_t st) {
  const size_t words = (size_t)(a.pool.num_pages + 31) / 32;
  const size_t smem = (2 * words + 1) * 4;
  const int rc = allow_smem(pages_compact_kernel, smem, (2 * kMaxPageWords + 1) * 4, "pages_compact_kernel");
  if (rc) return rc;
  pages_compact_kernel<<<1, kPoolThreads, smem, st>>>(a);
  count_launch();
  const int rl = check_launch("pages_compact_kernel");
  if (rl) return rl;
  // the data and the table's ids, in one launch (64 tensors each); a call without
  // tensors still maps the table
  const TableMap map = {a.pool.block_table, a.into.block_table, a.new_id, a.pool.bt_stride, a.into.bt_stride,
                        a.pool.max_rows, a.pool.bt_width};
  static const DashCacheTensor none = {};
  return a.n_tensors ? copy_pages(a.tensors, a.n_tensors, a.copy_src, a.copy_dst, a.pool.num_pages / 2, a.n_moves,
                                  a.pool.num_pages, map, st)
                     : copy_pages(&none, 1, a.copy_src, a.copy_dst, 0, a.n_moves, a.pool.num_pages, map, st);
}

}  // namespace dash
