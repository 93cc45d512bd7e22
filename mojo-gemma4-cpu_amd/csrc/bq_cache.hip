// Pages of a cache on the device: sequences that go on from others (beams, freed
// and fresh sequences), and the packing of the pages that are held.
//
// Reference: continuous_batching/ (paging and page copies on the host); here the
// table, the lengths and the reference counts stay on the device, so that a
// decode loop with beams runs, and is captured, without the host.
//
// A page's reference count is the number of table entries (of any table over the
// pool) that hold it; 0 is free.  A reorder, in terms of whole tables:
//   1. Every sequence takes its parent's entries, and the counts follow: an old entry
//      counts once for each child that keeps it instead of once.
//   2. The page a sequence writes next has to be its own.  Of the sequences on one
//      such page, in their order, all but the last leave it for a fresh page while
//      anyone else holds it; fresh pages are the lowest free numbers in the order
//      (sequence, page).
//   3. The rows already on a page that was left are copied in every array.
// All counts are integers, so the order of atomics leaves no trace.
//
// Pools whose tables and counts fit LDS (k_reorder_plan<true>, k_compact<true>) take one
// launch: every workgroup works the whole plan out for itself from the old state, marks
// that it has read it, and copies its share; the last to mark writes the new state.
// Larger ones are planned by launches of their own, then copied (k_cache_copy).
#include <algorithm>

#include "bq_half.hpp"
#include "bq_kernels.hpp"
#include "bq_pages.hpp"

namespace bq {

namespace {

constexpr int kPlanThreads = 1024, kWaves = kPlanThreads / 64;
constexpr int kTableThreads = 512;
constexpr int kBatch = 8;           // loads of a thread that are on their way at once
constexpr int kOwned = 2048;        // wanted pages whose sequences k_reorder_plan lists
constexpr int kTileEntries = 1024;  // table entries of a k_reorder_tables workgroup
constexpr int64_t kOneMoves = 64 << 20;  // bytes that a one-launch compaction may have to move
constexpr int64_t kOneBytes = 128 << 10;  // tables and counts of a one-launch plan (LDS)

struct CopyItem {
  int32_t src, dst, rows, pad;
};

// workspace: the marks of a launch's workgroups, or the plan for the next launch
constexpr int kMaxPlanBlocks = 256;
struct CopyList {
  int32_t count, pad[3];
  CopyItem item[1];
};

// inclusive scan over the workgroup; total in *sum
__device__ inline int block_scan(int v, int* wsum, int* sum) {
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int inc = wave_incl_scan(v);
  if (lane == 63) wsum[wave] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int x = wsum[w];
    before += w < wave ? x : 0;
    all += x;
  }
  __syncthreads();
  *sum = all;
  return inc + before;
}

// What a workgroup keeps in LDS of each sequence: where it comes from, and how many
// go on from it.
struct SeqLds {
  int32_t parent, len, full, end;  // SeqPlan
  int32_t own_full;                // whole pages it had itself
  int32_t shares, writes;          // its children, and those with a page to write
};

__device__ inline SeqPlan plan_of(const SeqLds& q) {
  return SeqPlan{q.parent, q.len, q.full, q.end};
}

// every sequence's plan; to be followed by a barrier and count_children
__device__ inline void load_seqs(const ReorderArgs& a, SeqLds* seq, int threads) {
  for (int i = threadIdx.x; i < a.num_seqs; i += threads) {
    const int p = a.parents[i];
    const SeqPlan s = seq_plan(p, a.num_seqs, p >= 0 && p < a.num_seqs ? a.lens[p] : 0,
                               a.grow ? a.grow[i] : 0, a.max_pages, a.page_shift);
    const SeqPlan own = seq_plan(i, a.num_seqs, a.lens[i], 0, a.max_pages, a.page_shift);
    seq[i] = SeqLds{s.parent, s.len, s.full, s.end, own.full, 0, 0};
  }
}

__device__ inline void count_children(const ReorderArgs& a, SeqLds* seq, int threads) {
  for (int i = threadIdx.x; i < a.num_seqs; i += threads) {
    const int p = seq[i].parent;
    if (p >= 0) {
      atomicAdd(&seq[p].shares, 1);
      if (seq[i].full < seq[i].end) atomicAdd(&seq[p].writes, 1);
    }
  }
}

// kBatch strided loads of a thread, asked for together; `get` says what element e is
template <typename Get>
__device__ inline void ask(int32_t (&v)[kBatch], int e0, int n, int threads, Get&& get) {
#pragma unroll
  for (int u = 0; u < kBatch; ++u) v[u] = e0 + u * threads < n ? get(e0 + u * threads) : 0;
}
template <typename Put>
__device__ inline void give_to(const int32_t (&v)[kBatch], int e0, int n, int threads, Put&& put) {
#pragma unroll
  for (int u = 0; u < kBatch; ++u)
    if (e0 + u * threads < n) put(e0 + u * threads, v[u]);
}

// columns [j0, j0 + width) of the tables: old page numbers to LDS ...
__device__ inline int32_t tile_entry(const ReorderArgs& a, int e, int j0, int width) {
  const int s = e / width;
  return a.base_rows[(int64_t)s * a.max_pages + j0 + (e - s * width)];
}
__device__ inline void load_tile(const ReorderArgs& a, int32_t* tile, int j0, int width,
                                 int threads) {
  const int n = a.num_seqs * width;
  for (int e0 = threadIdx.x; e0 < n; e0 += kBatch * threads) {
    int32_t v[kBatch];
    ask(v, e0, n, threads, [&](int e) { return tile_entry(a, e, j0, width); });
    give_to(v, e0, n, threads,
            [&](int e, int32_t base) { tile[e] = page_number(base, a.page_shift, a.num_pages); });
  }
}

// ... and the counts and new entries (row bases) from there, the latter to `to` with rows
// `to_width` apart
__device__ inline void new_tile(const ReorderArgs& a, int32_t* refs, const SeqLds* seq,
                                const int32_t* tile, int32_t* to, int to_width, int j0, int width,
                                int threads) {
  for (int e = threadIdx.x; e < a.num_seqs * width; e += threads) {
    const int s = e / width, c = e - s * width, j = j0 + c;
    const SeqLds q = seq[s];
    if (tile[e] >= 0) {
      const int d = (j < q.own_full ? q.shares : j == q.own_full ? q.writes : 0) - 1;
      if (d) atomicAdd(&refs[tile[e]], d);
    }
    const int page = seq_keeps(plan_of(q), j) ? tile[q.parent * width + c] : -1;
    to[(int64_t)s * to_width + j] = page >= 0 ? page << a.page_shift : -1;
  }
}

// the pool's counts from element e0 on to LDS, what is past the last page as held
__device__ inline void load_refs(const int32_t* from, int32_t* refs, int pages, int pages4, int e0) {
  for (; e0 < pages4; e0 += kBatch * kPlanThreads) {
    int32_t v[kBatch];
    ask(v, e0, pages, kPlanThreads, [&](int q) { return from[q]; });
    give_to(v, e0, pages4, kPlanThreads, [&](int q, int32_t r) { refs[q] = q < pages ? r : 1; });
  }
}

__global__ __launch_bounds__(kTableThreads) void k_reorder_tables(ReorderArgs a, int cols) {
  extern __shared__ int32_t lds[];
  SeqLds* seq = reinterpret_cast<SeqLds*>(lds);                     // [num_seqs]
  int32_t* tile = lds + (size_t)a.num_seqs * (sizeof(SeqLds) / 4);  // [num_seqs][width]
  const int j0 = blockIdx.x * cols, width = min(cols, a.max_pages - j0);
  load_seqs(a, seq, kTableThreads);
  load_tile(a, tile, j0, width, kTableThreads);
  __syncthreads();
  count_children(a, seq, kTableThreads);
  __syncthreads();
  new_tile(a, a.refs, seq, tile, a.base_rows, a.max_pages, j0, width, kTableThreads);
}

// Rows of pages in every array: a work item is a segment of one copy of one array,
// four 16-byte loads a thread ahead of its stores, which go past the caches (127
// MB in copies of 0 to 256 KiB: 54 us, 4.7 TB/s; through them 60).  Items are ordered by
// segment first, then by array: the missing ones of short copies and the small ones of
// narrow arrays come one after the other, and no workgroup gets more of them than another
// (66 us the other way round).  More workgroups than run at once
// gain 1 us there, and cost a call without copies 1.5.
__host__ __device__ constexpr int64_t segment_bytes(int threads) { return threads == 256 ? 32768 : 65536; }
constexpr int kCopyBlocks = 2048;

template <typename W, int THREADS>
__device__ inline void copy_bytes(uint8_t* d, const uint8_t* s, int64_t bytes) {
  constexpr int U = 4;
  const int n = (int)(bytes / (int64_t)sizeof(W));
  W* dw = reinterpret_cast<W*>(d);
  const W* sw = reinterpret_cast<const W*>(s);
  for (int k = threadIdx.x; k < n; k += THREADS * U) {
    W w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * THREADS < n) w[u] = sw[k + u * THREADS];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * THREADS < n) __builtin_nontemporal_store(w[u], dw + k + u * THREADS);
  }
}

// share `share` of `shares` of the copies, in segments of 128 bytes a thread (64 where a
// workgroup has 1024 threads)
template <int THREADS>
__device__ inline void copy_share(const CacheArrays& arrays, const CopyItem* items, int copies,
                                  int segments, int share, int shares) {
  const int64_t pairs = (int64_t)copies * arrays.n, total = pairs * segments;
  for (int64_t w = share; w < total; w += shares) {
    const int segment = (int)(w / pairs), r = (int)(w - segment * pairs);
    const int array = r / copies;
    const CopyItem it = items[r - array * copies];
    const int64_t row = arrays.row_bytes[array];
    uint8_t* data = static_cast<uint8_t*>(arrays.data[array]);
    const int64_t at = segment * segment_bytes(THREADS), bytes = (int64_t)it.rows * row;
    if (at >= bytes) continue;
    const int64_t len = bytes - at < segment_bytes(THREADS) ? bytes - at : segment_bytes(THREADS);
    uint8_t* d = data + it.dst * row + at;
    const uint8_t* s = data + it.src * row + at;
    const uint64_t align = reinterpret_cast<uint64_t>(data) | (uint64_t)row;
    if ((align & 15) == 0) copy_bytes<v4i, THREADS>(d, s, len);
    else if ((align & 3) == 0) copy_bytes<uint32_t, THREADS>(d, s, len);
    else copy_bytes<uint8_t, THREADS>(d, s, len);
  }
}

// ONE: the whole reorder, tables and counts in LDS and the copies too; else what
// k_reorder_tables leaves to plan.
template <bool ONE>
__global__ __launch_bounds__(kPlanThreads) void k_reorder_plan(ReorderArgs a, CacheArrays arrays,
                                                               int segments) {
  extern __shared__ __align__(16) int32_t lds[];
  const int n = a.num_seqs, i = threadIdx.x, entries = n * a.max_pages;
  const int pages4 = (a.num_pages + 3) & ~3;
  int32_t* refs = ONE ? lds : a.refs;                                 // [num_pages]
  CopyItem* items = ONE ? reinterpret_cast<CopyItem*>(lds + pages4)   // [num_seqs]
                        : static_cast<CopyList*>(a.workspace)->item;
  SeqLds* seq = ONE ? reinterpret_cast<SeqLds*>(items + n) : reinterpret_cast<SeqLds*>(lds);
  int32_t* tile = reinterpret_cast<int32_t*>(seq + n);                // ONE: [num_seqs][max_pages]
  int32_t* rows = ONE ? tile + entries : a.base_rows;                 // the new table, as wide
  __shared__ int wsum[kWaves], said;
  __shared__ __align__(16) int32_t last[kMaxCacheSeqs];
  __shared__ int32_t offset[kMaxCacheSeqs + 1], given[kMaxCacheSeqs], early[kMaxCacheSeqs];
  __shared__ int16_t owner[kOwned];
  early[i] = 0;
  if constexpr (ONE) {  // all first loads before any is used
    int32_t base[kBatch], count[kBatch];
    ask(base, i, entries, kPlanThreads, [&](int e) { return tile_entry(a, e, 0, a.max_pages); });
    ask(count, i, a.num_pages, kPlanThreads, [&](int q) { return a.refs[q]; });
    load_seqs(a, seq, kPlanThreads);
    give_to(base, i, entries, kPlanThreads, [&](int e, int32_t v) {
      tile[e] = page_number(v, a.page_shift, a.num_pages);
    });
    give_to(count, i, pages4, kPlanThreads,
            [&](int q, int32_t r) { refs[q] = q < a.num_pages ? r : 1; });
    for (int e = i + kBatch * kPlanThreads; e < entries; e += kPlanThreads)
      tile[e] = page_number(tile_entry(a, e, 0, a.max_pages), a.page_shift, a.num_pages);
    load_refs(a.refs, refs, a.num_pages, pages4, i + kBatch * kPlanThreads);
    __syncthreads();
    count_children(a, seq, kPlanThreads);
    __syncthreads();
    new_tile(a, refs, seq, tile, rows, a.max_pages, 0, a.max_pages, kPlanThreads);
  } else {
    load_seqs(a, seq, kPlanThreads);
  }
  SeqPlan p{};
  int page = -1;
  if (i < n) {
    p = plan_of(seq[i]);
    if (p.full < p.end) {
      if constexpr (ONE)
        page = p.parent >= 0 ? tile[p.parent * a.max_pages + p.full] : -1;
      else
        page = page_number(a.base_rows[(int64_t)i * a.max_pages + p.full], a.page_shift,
                           a.num_pages);
    }
  }
  last[i] = page;
  given[i] = -1;
  __syncthreads();  // every length has been read, every count changed
  if (!ONE && i < n) a.lens[i] = p.len;
  // earlier sequences on the same page, counted by 1024 / n threads each
  int np = 64;
  while (np < n) np <<= 1;
  {
    const int who = i & (np - 1), step = 4 * (kPlanThreads / np), mine = last[who];
    int earlier = 0;
    if (mine >= 0)
#pragma unroll 2
      for (int k = 4 * (i / np); k < who; k += step) {
        const v4i l = *reinterpret_cast<const v4i*>(last + k);
#pragma unroll
        for (int u = 0; u < 4; ++u) earlier += l[u] == mine && k + u < who;
      }
    if (earlier) atomicAdd(&early[who], earlier);
  }
  __syncthreads();
  const bool leaves = page >= 0 && refs[page] - early[i] > 1;
  __syncthreads();  // before counts fall
  int fresh = i < n ? p.end - p.full : 0;
  if (page >= 0 && !leaves) --fresh;
  int total;
  const int incl = block_scan(fresh, wsum, &total);
  if (i < n) offset[i] = incl - fresh;
  if (i == 0) offset[n] = total;
  if (total <= kOwned)
    for (int k = incl - fresh; k < incl; ++k) owner[k] = (int16_t)i;
  if (leaves) atomicAdd(&refs[page], -1);  // it stays above 0: the last one keeps it
  __syncthreads();

  // the k-th page that is wanted: a sequence's, from a list or (many pages for a few
  // sequences) by bisection of the offsets
  auto give = [&](int k, int page_) {
    int lo = 0;
    if (total <= kOwned) {
      lo = owner[k];
    } else {
      for (int hi = n - 1; lo < hi;) {  // the last sequence with offset <= k
        const int mid = (lo + hi + 1) >> 1;
        if (offset[mid] <= k) lo = mid;
        else hi = mid - 1;
      }
    }
    const int j = seq[lo].end - (offset[lo + 1] - k);
    rows[(int64_t)lo * a.max_pages + j] = page_ >= 0 ? page_ << a.page_shift : -1;
    if (j == seq[lo].full) given[lo] = page_;
  };
  // the first `total` free pages, lowest numbers first, four a thread
  int got = 0;
  for (int base = 0; base < a.num_pages && got < total; base += 4 * kPlanThreads) {
    const int q = base + 4 * i;
    int free_ = 0, found;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (q + u < a.num_pages && refs[q + u] == 0) free_ |= 1 << u;
    int k = got + block_scan(__popc(free_), wsum, &found) - __popc(free_);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (free_ >> u & 1) {
        if (k < total) {
          refs[q + u] = 1;
          give(k, q + u);
        }
        ++k;
      }
    got += found;
  }
  if (got > total) got = total;
  for (int k = got + i; k < total; k += kPlanThreads) give(k, -1);  // no page left for these
  __syncthreads();
  // what a left page held goes to the page that was given instead
  const int held = p.len & ((1 << a.page_shift) - 1);
  const int copy = leaves && held && given[i] >= 0;
  int copies;
  const int at = block_scan(copy, wsum, &copies) - copy;
  if (copy) items[at] = CopyItem{page << a.page_shift, given[i] << a.page_shift, held, 0};
  const bool done = !ONE || last_of(static_cast<uint64_t*>(a.workspace), 1, gridDim.x, blockIdx.x,
                                    a.tag, &said);
  if (done) {
    if constexpr (ONE) {
      for (int q = i; q < a.num_pages; q += kPlanThreads) a.refs[q] = refs[q];
      for (int e = i; e < entries; e += kPlanThreads) a.base_rows[e] = rows[e];
      if (i < n) a.lens[i] = p.len;
    }
    if (i == 0) {
      if constexpr (!ONE) static_cast<CopyList*>(a.workspace)->count = copies;
      a.info[0] = got;
      a.info[1] = copies;
      a.info[2] = total - got;
      a.info[3] = 0;
    }
  }
  if constexpr (ONE)  // last_of's barriers stand between the items and this
    copy_share<kPlanThreads>(arrays, items, copies, segments, blockIdx.x, gridDim.x);
}

// Packing: with `live` pages held, the i-th free page below `live` takes the i-th held
// page from `live` on.  ONE: all of it, the plan in LDS; else the plan alone.
template <bool ONE>
__global__ __launch_bounds__(kPlanThreads) void k_compact(CompactArgs a, CacheArrays arrays,
                                                          int segments) {
  extern __shared__ __align__(16) int32_t lds[];
  __shared__ int wsum[kWaves], said;
  const int i = threadIdx.x, pages4 = (a.num_pages + 3) & ~3;
  int32_t* refs = ONE ? lds : a.refs;  // [num_pages]
  CopyItem* items = ONE ? reinterpret_cast<CopyItem*>(lds + pages4)  // [num_pages / 2 + 1]
                        : static_cast<CopyList*>(a.workspace)->item;
  int32_t* to = reinterpret_cast<int32_t*>(items + (a.num_pages / 2 + 1));  // [num_pages]
  if constexpr (ONE) {
    load_refs(a.refs, refs, a.num_pages, pages4, i);
    __syncthreads();
  }
  auto held4 = [&](int q) {  // which of four pages are held, as bits
    int m = 0;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (q + u < a.num_pages && refs[q + u] != 0) m |= 1 << u;
    return m;
  };
  int mine = 0, live;
  for (int q = 4 * i; q < a.num_pages; q += 4 * kPlanThreads) mine += __popc(held4(q));
  block_scan(mine, wsum, &live);
  int holes = 0, movers = 0;
  for (int base = 0; base < a.num_pages; base += 4 * kPlanThreads) {
    const int q = base + 4 * i, held = held4(q);
    const int in = min(max(a.num_pages - q, 0), 4), low = min(max(live - q, 0), 4);
    const int hole = ~held & ((1 << low) - 1), mover = held & ~((1 << low) - 1);
    int both;  // at most 4096 of each: two counts in one scan
    const int mineboth = __popc(hole) | __popc(mover) << 16;
    const int before = block_scan(mineboth, wsum, &both) - mineboth;
    int kh = holes + (before & 0xFFFF), km = movers + (before >> 16);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (hole >> u & 1) items[kh++].dst = q + u;
      if (mover >> u & 1) items[km++].src = q + u;
      if (u < in) to[q + u] = q + u;
    }
    holes += both & 0xFFFF;
    movers += both >> 16;
  }
  __syncthreads();
  for (int k = i; k < movers; k += kPlanThreads) {
    const int src = items[k].src, dst = items[k].dst;
    to[src] = dst;
    refs[dst] = refs[src];
    refs[src] = 0;
    items[k] = CopyItem{src << a.page_shift, dst << a.page_shift, 1 << a.page_shift, 0};
  }
  // The last to have read the counts writes; were two to write, the second would find
  // every entry where it belongs.
  const bool done = !ONE || last_of(static_cast<uint64_t*>(a.workspace), 1, gridDim.x, blockIdx.x,
                                    a.tag, &said);
  if (done) {
    if constexpr (ONE) {
      for (int q = i; q < a.num_pages; q += kPlanThreads) a.refs[q] = refs[q];
      if (movers)
        for (int e = i; e < a.num_seqs * a.max_pages; e += kPlanThreads) {
          const int page = page_number(a.base_rows[e], a.page_shift, a.num_pages);
          if (page >= live) a.base_rows[e] = to[page] << a.page_shift;
        }
    }
    if (i == 0) {
      if constexpr (!ONE) static_cast<CopyList*>(a.workspace)->count = movers;
      a.info[0] = live;
      a.info[1] = movers;
      a.info[2] = a.info[3] = 0;
    }
  }
  if constexpr (ONE)
    copy_share<kPlanThreads>(arrays, items, movers, segments, blockIdx.x, gridDim.x);
}

// The first `table_blocks` workgroups (compaction) carry the tables over to the new
// page numbers, the others copy.
__global__ __launch_bounds__(256) void k_cache_copy(CacheArrays arrays, const void* workspace,
                                                    int segments, CompactArgs t, int table_blocks) {
  const CopyList* list = static_cast<const CopyList*>(workspace);
  if (list->count == 0) return;
  if (blockIdx.x < table_blocks) {
    const int32_t* to = reinterpret_cast<const int32_t*>(list->item + (t.num_pages / 2 + 1));
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= (int64_t)t.num_seqs * t.max_pages) return;
    const int page = page_number(t.base_rows[e], t.page_shift, t.num_pages);
    if (page >= 0) t.base_rows[e] = to[page] << t.page_shift;
    return;
  }
  copy_share<256>(arrays, list->item, list->count, segments, blockIdx.x - table_blocks,
                  gridDim.x - table_blocks);
}

// segments of the widest array's page
int64_t copy_segments(const CacheArrays& arrays, int page_shift, int threads) {
  int64_t most = 0;
  for (int i = 0; i < arrays.n; ++i) most = std::max(most, arrays.row_bytes[i] << page_shift);
  const int64_t each = segment_bytes(threads);
  return std::max<int64_t>(1, (most + each - 1) / each);
}

hipError_t launch_copy(const CacheArrays& arrays, void* workspace, int max_items, int64_t segments,
                       hipStream_t st, const CompactArgs* t = nullptr) {
  const int64_t entries = t ? (int64_t)t->num_seqs * t->max_pages : 0;
  const int64_t table_blocks = (entries + 255) / 256;
  const int64_t copies = std::min<int64_t>((int64_t)max_items * arrays.n * segments, kCopyBlocks);
  if (copies == 0 && table_blocks == 0) return hipSuccess;
  k_cache_copy<<<(int)(table_blocks + std::max<int64_t>(copies, 1)), 256, 0, st>>>(
      arrays, workspace, (int)segments, t ? *t : CompactArgs{}, (int)table_blocks);
  return hipGetLastError();
}

// a plan of `bytes` of LDS, by a workgroup for every two pieces that there may be to copy
template <typename K, typename A>
hipError_t launch_one(K kernel, A a, const CacheArrays& arrays, int64_t bytes, int max_items,
                      int64_t segments, hipStream_t st) {
  if (bytes > 40960) {  // with 20 KiB of fixed LDS
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) return e;
  }
  const int64_t blocks = std::min<int64_t>(std::min(tune().cus, kMaxPlanBlocks),
                                           (int64_t)max_items * arrays.n * segments / 2);
  a.tag = launch_tag();
  kernel<<<(int)std::max<int64_t>(blocks, 1), kPlanThreads, (size_t)bytes, st>>>(a, arrays,
                                                                               (int)segments);
  return hipGetLastError();
}

}  // namespace

size_t reorder_workspace(int num_seqs) {
  return std::max(16 + (size_t)num_seqs * sizeof(CopyItem), kMaxPlanBlocks * sizeof(uint64_t));
}
size_t compact_workspace(int num_pages) {
  return std::max(16 + ((size_t)num_pages / 2 + 1) * sizeof(CopyItem) + (size_t)num_pages * 4,
                  kMaxPlanBlocks * sizeof(uint64_t));
}

hipError_t launch_cache_reorder(const ReorderArgs& a, const CacheArrays& arrays, hipStream_t st) {
  const int64_t segments = copy_segments(arrays, a.page_shift, 256);
  const int64_t large = copy_segments(arrays, a.page_shift, kPlanThreads);
  if (segments * kMaxCacheArrays > INT32_MAX) return hipErrorInvalidValue;
  const int64_t seqs = (int64_t)sizeof(SeqLds) * a.num_seqs, pages4 = (a.num_pages + 3) & ~3;
  const int64_t one = seqs + (int64_t)sizeof(CopyItem) * a.num_seqs +
                      4 * (pages4 + 2 * (int64_t)a.num_seqs * a.max_pages);
  if (one <= kOneBytes)
    return launch_one(&k_reorder_plan<true>, a, arrays, one, a.num_seqs, large, st);
  const int cols = std::max(1, std::min(a.max_pages, kTileEntries / a.num_seqs));
  k_reorder_tables<<<(a.max_pages + cols - 1) / cols, kTableThreads,
                     (size_t)seqs + (size_t)cols * a.num_seqs * 4, st>>>(a, cols);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  k_reorder_plan<false><<<1, kPlanThreads, (size_t)seqs, st>>>(a, arrays, 0);
  e = hipGetLastError();
  return e != hipSuccess ? e : launch_copy(arrays, a.workspace, a.num_seqs, segments, st);
}

hipError_t launch_cache_compact(const CompactArgs& a, const CacheArrays& arrays, hipStream_t st) {
  const int64_t segments = copy_segments(arrays, a.page_shift, 256);
  const int64_t large = copy_segments(arrays, a.page_shift, kPlanThreads);
  if (segments * kMaxCacheArrays > INT32_MAX) return hipErrorInvalidValue;
  const int64_t pages4 = (a.num_pages + 3) & ~3;
  const int64_t one = 8 * pages4 + (int64_t)sizeof(CopyItem) * (a.num_pages / 2 + 1);
  // Where much may move, the copies of a launch of their own, in small workgroups, make up
  // for it: 64 sequences of 2000 positions, an eighth retired, 470 MB: 117 and 121 us.
  int64_t page = 0;
  for (int i = 0; i < arrays.n; ++i) page += arrays.row_bytes[i] << a.page_shift;
  if (one <= kOneBytes && page * (a.num_pages / 2) <= kOneMoves)
    return launch_one(&k_compact<true>, a, arrays, one, a.num_pages / 2, large, st);
  k_compact<false><<<1, kPlanThreads, 0, st>>>(a, arrays, 0);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess
             ? e
             : launch_copy(arrays, a.workspace, a.num_pages / 2, segments, st, &a);
}

}  // namespace bq
