// Pages of a cache on the device: sequences that go on from others (beams, freed
// and fresh sequences), and the packing of the pages that are held.
//
// Reference: continuous_batching/ (paging and page copies on the host); here the
// table, the lengths and the reference counts stay on the device, so that a
// decode loop with beams runs, and is captured, without the host.
//
// A page's reference count is the number of table entries (of any table over the
// pool) that hold it; 0 is free.  A reorder, in terms of whole tables:
//   1. k_reorder_tables: every sequence takes its parent's entries (in place: a
//      workgroup owns all rows of a few columns), and the counts follow: an old
//      entry counts once for each child that keeps it instead of once.
//   2. k_reorder_plan (one workgroup): the page a sequence writes next has to be
//      its own.  Of the sequences on one such page, in their order, all but the
//      last leave it for a fresh page while anyone else holds it; fresh pages are
//      the lowest free numbers in the order (sequence, page).
//   3. k_cache_copy: the rows already on a page that was left, in every array.
// All counts are integers, so the order of the atomics leaves no trace.
#include <algorithm>

#include "bq_device.hpp"
#include "bq_kernels.hpp"
#include "bq_pages.hpp"

namespace bq {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kTileEntries = 8192;  // LDS entries of k_reorder_tables (32 KiB)

struct CopyItem {
  int32_t src, dst, rows, pad;
};

// workspace: header {copies, 0, 0, 0}, then the copies
struct CopyList {
  int32_t count, pad[3];
  CopyItem item[1];
};

__global__ __launch_bounds__(256) void k_reorder_tables(ReorderArgs a, int cols) {
  extern __shared__ int32_t lds[];
  int32_t* tile = lds;                               // [num_seqs][cols] page numbers
  int32_t* shares = lds + (size_t)a.num_seqs * cols;  // children of each sequence
  int32_t* writes = shares + a.num_seqs;              // of these, with a page to write
  const int j0 = blockIdx.x * cols, n = a.num_seqs;
  for (int i = threadIdx.x; i < n; i += blockDim.x) shares[i] = writes[i] = 0;
  for (int e = threadIdx.x; e < n * cols; e += blockDim.x) {
    const int s = e / cols, j = j0 + e % cols;
    tile[e] = j < a.max_pages
                  ? page_number(a.base_rows[(int64_t)s * a.max_pages + j], a.page_shift, a.num_pages)
                  : -1;
  }
  __syncthreads();
  auto plan_of = [&](int i) {
    const int p = a.parents[i];
    return seq_plan(p, n, p >= 0 && p < n ? a.lens[p] : 0, a.grow ? a.grow[i] : 0, a.max_pages,
                    a.page_shift);
  };
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const SeqPlan s = plan_of(i);
    if (s.parent >= 0) {
      atomicAdd(&shares[s.parent], 1);
      if (s.full < s.end) atomicAdd(&writes[s.parent], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < n * cols; e += blockDim.x) {
    const int s = e / cols, j = j0 + e % cols;
    if (j >= a.max_pages) continue;
    if (tile[e] >= 0) {  // the old entry
      const SeqPlan own = seq_plan(s, n, a.lens[s], 0, a.max_pages, a.page_shift);
      const int d = (j < own.full ? shares[s] : j == own.full ? writes[s] : 0) - 1;
      if (d) atomicAdd(&a.refs[tile[e]], d);
    }
    const SeqPlan p = plan_of(s);  // the new one
    const int page = seq_keeps(p, j) ? tile[p.parent * cols + e % cols] : -1;
    a.base_rows[(int64_t)s * a.max_pages + j] = page >= 0 ? page << a.page_shift : -1;
  }
}

// inclusive scan over the workgroup; total in *sum
__device__ inline int block_scan(int v, int* wsum, int* sum) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int inc = wave_incl_scan(v);
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    const int x = wsum[w];
    before += w < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *sum = all;
  return inc + before;
}

__global__ __launch_bounds__(kPlanThreads) void k_reorder_plan(ReorderArgs a) {
  __shared__ int wsum[kPlanThreads / 64];
  __shared__ int32_t last[kMaxCacheSeqs], offset[kMaxCacheSeqs + 1];
  __shared__ int ncopy, nfree;
  CopyList* list = static_cast<CopyList*>(a.workspace);
  const int n = a.num_seqs, i = threadIdx.x;
  SeqPlan p{};
  int page = -1;
  if (i < n) {
    const int par = a.parents[i];
    p = seq_plan(par, n, par >= 0 && par < n ? a.lens[par] : 0, a.grow ? a.grow[i] : 0,
                 a.max_pages, a.page_shift);
    if (p.full < p.end)
      page = page_number(a.base_rows[(int64_t)i * a.max_pages + p.full], a.page_shift, a.num_pages);
    last[i] = page;
  }
  if (i == 0) ncopy = nfree = 0;
  __syncthreads();
  if (i < n) a.lens[i] = p.len;  // every length has been read
  bool leaves = false;
  if (page >= 0) {
    int earlier = 0;
    for (int k = 0; k < i; ++k) earlier += last[k] == page;
    leaves = a.refs[page] - earlier > 1;
  }
  int fresh = p.end - p.full;
  if (i >= n) fresh = 0;
  if (page >= 0 && !leaves) --fresh;
  int total;
  const int incl = block_scan(fresh, wsum, &total);
  if (i < n) offset[i] = incl - fresh;
  if (i == 0) offset[n] = total;
  if (leaves) atomicAdd(&a.refs[page], -1);  // it stays above 0: the last one keeps it
  __syncthreads();

  // the first `total` free pages, lowest numbers first
  int got = 0;
  for (int base = 0; base < a.num_pages && got < total; base += kPlanThreads) {
    const int q = base + i;
    const int free_ = q < a.num_pages && a.refs[q] == 0;
    int found;
    const int k = got + block_scan(free_, wsum, &found) - free_;
    if (free_ && k < total) {
      int lo = 0, hi = n - 1;  // the sequence: the last one with offset <= k
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offset[mid] <= k) lo = mid;
        else hi = mid - 1;
      }
      const int par = a.parents[lo];
      // its length is in lens already
      const SeqPlan s = seq_plan(par >= 0 && par < n ? 0 : -1, n, a.lens[lo], a.grow ? a.grow[lo] : 0,
                                 a.max_pages, a.page_shift);
      const int count = offset[lo + 1] - offset[lo];
      const int j = s.end - count + (k - offset[lo]);
      a.refs[q] = 1;
      a.base_rows[(int64_t)lo * a.max_pages + j] = q << a.page_shift;
      const int rows = s.len & ((1 << a.page_shift) - 1);
      if (j == s.full && last[lo] >= 0 && rows) {
        const int at = atomicAdd(&ncopy, 1);
        list->item[at] = CopyItem{last[lo] << a.page_shift, q << a.page_shift, rows, 0};
      }
    }
    got += found;
  }
  if (got > total) got = total;
  // entries that found no page
  for (int k = got + i; k < total; k += kPlanThreads) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offset[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    const int par = a.parents[lo];
    const SeqPlan s = seq_plan(par >= 0 && par < n ? 0 : -1, n, a.lens[lo], a.grow ? a.grow[lo] : 0,
                               a.max_pages, a.page_shift);
    const int count = offset[lo + 1] - offset[lo];
    a.base_rows[(int64_t)lo * a.max_pages + s.end - count + (k - offset[lo])] = -1;
  }
  __syncthreads();
  if (i == 0) {
    list->count = ncopy;
    a.info[0] = got;
    a.info[1] = ncopy;
    a.info[2] = total - got;
    a.info[3] = 0;
  }
}

// Page numbers after packing: with `live` pages held, the i-th free page below
// `live` takes the i-th held page from `live` on.
__global__ __launch_bounds__(kPlanThreads) void k_compact_plan(CompactArgs a) {
  __shared__ int wsum[kPlanThreads / 64];
  const int i = threadIdx.x;
  CopyList* list = static_cast<CopyList*>(a.workspace);
  int32_t* to = reinterpret_cast<int32_t*>(list->item + (a.num_pages / 2 + 1));
  int mine = 0, live;
  for (int q = i; q < a.num_pages; q += kPlanThreads) mine += a.refs[q] != 0;
  block_scan(mine, wsum, &live);
  int holes = 0, movers = 0;
  for (int base = 0; base < a.num_pages; base += kPlanThreads) {
    const int q = base + i;
    const bool in = q < a.num_pages;
    const bool held = in && a.refs[q] != 0;
    const int hole = in && !held && q < live, mover = held && q >= live;
    int nh, nm;
    const int kh = holes + block_scan(hole, wsum, &nh) - hole;
    const int km = movers + block_scan(mover, wsum, &nm) - mover;
    if (hole) list->item[kh].dst = q;
    if (mover) list->item[km].src = q;
    if (in) to[q] = q;
    holes += nh;
    movers += nm;
  }
  __syncthreads();
  for (int k = i; k < movers; k += kPlanThreads) {
    const int src = list->item[k].src, dst = list->item[k].dst;
    to[src] = dst;
    a.refs[dst] = a.refs[src];
    a.refs[src] = 0;
    list->item[k] = CopyItem{src << a.page_shift, dst << a.page_shift, 1 << a.page_shift, 0};
  }
  if (i == 0) {
    list->count = movers;
    a.info[0] = live;
    a.info[1] = movers;
    a.info[2] = a.info[3] = 0;
  }
}

__global__ __launch_bounds__(256) void k_compact_tables(CompactArgs a) {
  const CopyList* list = static_cast<const CopyList*>(a.workspace);
  const int32_t* to = reinterpret_cast<const int32_t*>(list->item + (a.num_pages / 2 + 1));
  if (list->count == 0) return;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (int64_t)a.num_seqs * a.max_pages) return;
  const int page = page_number(a.base_rows[e], a.page_shift, a.num_pages);
  if (page >= 0) a.base_rows[e] = to[page] << a.page_shift;
}

// Rows of pages in every array: a work item is kSegment bytes of one copy of one
// array.
constexpr int64_t kSegment = 32768;

template <typename W>
__device__ inline void copy_bytes(uint8_t* d, const uint8_t* s, int64_t bytes) {
  const int64_t n = bytes / (int64_t)sizeof(W);
  for (int64_t k = threadIdx.x; k < n; k += 256)
    reinterpret_cast<W*>(d)[k] = reinterpret_cast<const W*>(s)[k];
}

__global__ __launch_bounds__(256) void k_cache_copy(CacheArrays arrays, const void* workspace,
                                                    int segments) {
  const CopyList* list = static_cast<const CopyList*>(workspace);
  const int64_t per = (int64_t)arrays.n * segments, total = (int64_t)list->count * per;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const CopyItem it = list->item[w / per];
    const int r = (int)(w % per);
    const int64_t row = arrays.row_bytes[r / segments];
    uint8_t* data = static_cast<uint8_t*>(arrays.data[r / segments]);
    const int64_t at = (r % segments) * kSegment, bytes = (int64_t)it.rows * row;
    if (at >= bytes) continue;
    const int64_t len = bytes - at < kSegment ? bytes - at : kSegment;
    uint8_t* d = data + it.dst * row + at;
    const uint8_t* s = data + it.src * row + at;
    const uint64_t align = reinterpret_cast<uint64_t>(data) | (uint64_t)row;
    if ((align & 15) == 0) copy_bytes<v4i>(d, s, len);
    else if ((align & 3) == 0) copy_bytes<uint32_t>(d, s, len);
    else copy_bytes<uint8_t>(d, s, len);
  }
}

hipError_t launch_copy(const CacheArrays& arrays, void* workspace, int max_items, int page_shift,
                       hipStream_t st) {
  if (arrays.n == 0 || max_items == 0) return hipSuccess;
  int64_t most = 0;
  for (int i = 0; i < arrays.n; ++i) most = std::max(most, arrays.row_bytes[i] << page_shift);
  const int64_t segments = (most + kSegment - 1) / kSegment;
  if (segments * arrays.n > INT32_MAX) return hipErrorInvalidValue;
  const int64_t items = std::min<int64_t>((int64_t)max_items * arrays.n * segments, 4096);
  k_cache_copy<<<(int)items, 256, 0, st>>>(arrays, workspace, (int)segments);
  return hipGetLastError();
}

}  // namespace

size_t reorder_workspace(int num_seqs) { return 16 + (size_t)num_seqs * sizeof(CopyItem); }
size_t compact_workspace(int num_pages) {
  return 16 + ((size_t)num_pages / 2 + 1) * sizeof(CopyItem) + (size_t)num_pages * 4;
}

hipError_t launch_cache_reorder(const ReorderArgs& a, const CacheArrays& arrays, hipStream_t st) {
  const int cols = std::max(1, std::min(64, kTileEntries / a.num_seqs));
  const int blocks = (a.max_pages + cols - 1) / cols;
  const size_t lds = ((size_t)a.num_seqs * cols + 2 * (size_t)a.num_seqs) * 4;
  k_reorder_tables<<<blocks, 256, lds, st>>>(a, cols);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k_reorder_plan<<<1, kPlanThreads, 0, st>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  return launch_copy(arrays, a.workspace, a.num_seqs, a.page_shift, st);
}

hipError_t launch_cache_compact(const CompactArgs& a, const CacheArrays& arrays, hipStream_t st) {
  k_compact_plan<<<1, kPlanThreads, 0, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t entries = (int64_t)a.num_seqs * a.max_pages;
  k_compact_tables<<<(int)((entries + 255) / 256), 256, 0, st>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  return launch_copy(arrays, a.workspace, a.num_pages / 2, a.page_shift, st);
}

}  // namespace bq
