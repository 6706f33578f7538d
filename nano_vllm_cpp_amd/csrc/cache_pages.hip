// Pages of a paged KV cache: copied, shared by a forked sequence, given back, moved together.
//
// A page is block_size rows of every cache of a model (K and V of each layer).  Its state is one
// int32 reference count: 0 is free, n is held by n block-table entries.  There is no free list:
// a fork takes the lowest free pages, which the count array names, so the same calls give the
// same pages on every run.
//
// The page operations are copies, bound by HBM: 16-byte vectors, 16 KiB a workgroup.  180 pages of 256 KiB
// in 16 caches moved, whole calls: 290 us (4, 8, 32 and 64 KiB: 302, 294, 356 and 316; not streamed past the
// caches: 307), 279 with 1024 workgroups that walk the slices, 5.4 TB/s (a large copy 6.5).
#include <string.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "nvf_device.hpp"
#include "nvf_host.hpp"

namespace nvf {

constexpr int kPageThreads = 256;
constexpr int64_t kSliceBytes = 16384;  // of a page, one workgroup
constexpr int kMaxCaches = 128;         // in one launch's arguments
constexpr int kMaxPairs = 256;

struct CacheList {
  int n;
  uint8_t* base[kMaxCaches];
};
struct PairList {
  int n;
  int32_t a[kMaxPairs], b[kMaxPairs];
};

// bytes [begin, end) of a slice, 16-byte vectors or single bytes
template <bool VEC>
__device__ __forceinline__ void copy_bytes(uint8_t* __restrict__ dst, const uint8_t* __restrict__ src, int64_t n) {
  if constexpr (VEC) {
    constexpr int kPer = (int)(kSliceBytes / (16 * kPageThreads));
    u32x4 v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t at = 16 * ((int64_t)i * kPageThreads + threadIdx.x);
      if (at < n) v[i] = ld16_nt(src + at);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t at = 16 * ((int64_t)i * kPageThreads + threadIdx.x);
      if (at < n) st16_nt(dst + at, v[i]);
    }
  } else {
    for (int64_t at = threadIdx.x; at < n; at += kPageThreads) dst[at] = src[at];
  }
}

// workgroup = (pair, cache, slice)
template <bool VEC>
__global__ __launch_bounds__(kPageThreads) void copy_pages_kernel(const CacheList caches, const PairList pairs,
                                                                  int64_t page_bytes, int slices) {
  const int slice = (int)(blockIdx.x % slices), rest = (int)(blockIdx.x / slices);
  const int c = rest % caches.n, p = rest / caches.n;
  const int64_t at = slice * kSliceBytes;
  uint8_t* base = caches.base[c];
  copy_bytes<VEC>(base + pairs.b[p] * page_bytes + at, base + pairs.a[p] * page_bytes + at,
                  page_bytes - at < kSliceBytes ? page_bytes - at : kSliceBytes);
}

// ---------------------------------------------------------------------------
// Scans of the reference counts by one workgroup: thread i of 1024 takes 16 consecutive pages of
// each 16384.
constexpr int kScanThreads = 1024;
constexpr int kScanPer = 16;

// The number of set bits below this thread's, over the workgroup, and their total; `lds` holds a
// count for each wave.
__device__ __forceinline__ int scan_bits(int count, int* lds, int& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int sum = count;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  __syncthreads();  // the previous scan's reads of lds
  if (lane == 63) lds[w] = sum;
  __syncthreads();
  int below = 0;
  total = 0;
  for (int i = 0; i < kScanThreads / 64; ++i) {
    const int v = lds[i];
    below += i < w ? v : 0;
    total += v;
  }
  return below + sum - count;
}

// bit i: page at + i exists and pred(its count)
template <typename F>
__device__ __forceinline__ uint32_t page_bits(const int32_t* __restrict__ ref, int64_t at, int64_t end, F pred) {
  uint32_t bits = 0;
  int32_t v[kScanPer];
#pragma unroll
  for (int i = 0; i < kScanPer; ++i) v[i] = at + i < end ? ref[at + i] : 0;
#pragma unroll
  for (int i = 0; i < kScanPer; ++i) bits |= (at + i < end && pred(v[i])) ? 1u << i : 0u;
  return bits;
}

// Forks a[i] -> b[i] (parents, children).  The child takes its parent's full pages; for a partial last
// one the i-th fork that has one gets the i-th lowest free page (new_page[i]; -1: it needs none,
// -2: there is none, and the child ends with its full pages).  Where the parent's entry for the partial one is no page
// of the cache, there are no rows to copy and the child gets no page: one would show its last owner's.
__global__ __launch_bounds__(kScanThreads) void fork_plan_kernel(int32_t* __restrict__ tables,
                                                                 int32_t* __restrict__ key_len,
                                                                 int32_t* __restrict__ ref, const PairList forks,
                                                                 int32_t* __restrict__ new_page, int max_blocks,
                                                                 int64_t num_pages, int bs) {
  __shared__ int counts[kScanThreads / 64];
  __shared__ int32_t page_of[kMaxPairs], len_of[kMaxPairs];
  const int i = threadIdx.x;
  const int len = i < forks.n ? max(key_len[forks.a[i]], 0) : 0;
  const bool partial = i < forks.n && len % bs != 0 && len / bs < max_blocks;
  const int32_t last = partial ? tables[(int64_t)forks.a[i] * max_blocks + len / bs] : -1;
  const bool needs = last >= 0 && last < num_pages;
  if (i < kMaxPairs) {
    page_of[i] = -2;
    len_of[i] = len;
  }
  int wanted = 0;
  const int rank = scan_bits(needs ? 1 : 0, counts, wanted);
  int found = 0;
  for (int64_t p0 = 0; p0 < num_pages && found < wanted; p0 += kScanThreads * kScanPer) {
    const int64_t at = p0 + (int64_t)i * kScanPer;
    uint32_t bits = page_bits(ref, at, num_pages, [](int32_t r) { return r == 0; });
    int total = 0, k = found + scan_bits(__popc(bits), counts, total);
    for (; bits && k < wanted; bits &= bits - 1, ++k) page_of[k] = (int32_t)(at + __builtin_ctz(bits));
    found += total;
  }
  __syncthreads();
  // (every count has been read)
  if (i < forks.n) {
    const int32_t page = needs ? page_of[rank] : -1;
    new_page[i] = page;
    if (page >= 0) ref[page] = 1;
    key_len[forks.b[i]] = page == -2 ? len / bs * bs : len;
    if (partial) tables[(int64_t)forks.b[i] * max_blocks + len / bs] = page >= 0 ? page : -1;
  }
  for (int64_t x = i; x < (int64_t)forks.n * max_blocks; x += kScanThreads) {  // (fork, block)
    const int f = (int)(x / max_blocks), c = (int)(x - (int64_t)f * max_blocks), n = len_of[f], full = n / bs;
    if (c == full && n % bs != 0) continue;  // the partial page, above
    const int32_t e = c < full ? tables[(int64_t)forks.a[f] * max_blocks + c] : -1;
    const bool held = e >= 0 && e < num_pages;
    tables[(int64_t)forks.b[f] * max_blocks + c] = held ? e : -1;
    if (held) atomicAdd(ref + e, 1);
  }
}

// workgroup = (fork, cache, slice): the used rows of the parent's last page to the child's
template <bool VEC>
__global__ __launch_bounds__(kPageThreads) void fork_copy_kernel(const CacheList caches, const PairList forks,
                                                                 const int32_t* __restrict__ tables,
                                                                 const int32_t* __restrict__ key_len,
                                                                 const int32_t* __restrict__ new_page, int max_blocks,
                                                                 int64_t num_pages, int bs, int64_t row_bytes,
                                                                 int slices) {
  const int slice = (int)(blockIdx.x % slices), rest = (int)(blockIdx.x / slices);
  const int c = rest % caches.n, f = rest / caches.n;
  const int32_t to = new_page[f];
  if (to < 0) return;
  const int len = key_len[forks.a[f]];
  const int32_t from = tables[(int64_t)forks.a[f] * max_blocks + len / bs];
  if (from < 0 || from >= num_pages) return;
  const int64_t at = slice * kSliceBytes, used = len % bs * row_bytes - at, page_bytes = bs * row_bytes;
  if (used <= 0) return;
  uint8_t* base = caches.base[c];
  copy_bytes<VEC>(base + to * page_bytes + at, base + from * page_bytes + at, used < kSliceBytes ? used : kSliceBytes);
}

// One workgroup a sequence.  window < 0: all of its pages.  Otherwise those whose keys the next
// token (key count key_len + 1) does not see: no key below sinks, none from key_len + 1 - window on.
__global__ __launch_bounds__(kPageThreads) void free_pages_kernel(int32_t* __restrict__ tables,
                                                                  int32_t* __restrict__ key_len,
                                                                  int32_t* __restrict__ ref, const PairList seqs,
                                                                  int max_blocks, int64_t num_pages, int bs,
                                                                  int64_t window, int64_t sinks) {
  const int64_t s = seqs.a[blockIdx.x];
  const int64_t first = window < 0 ? INT64_MAX : (int64_t)key_len[s] + 1 - window;  // the oldest key in the window
  for (int c = threadIdx.x; c < max_blocks; c += kPageThreads) {
    const int64_t k0 = (int64_t)c * bs;
    if (window >= 0 && (k0 < sinks || k0 + bs > first)) continue;
    int32_t* e = tables + s * max_blocks + c;
    const int32_t page = *e;
    *e = -1;
    if (page < 0 || page >= num_pages) continue;
    if (atomicSub(ref + page, 1) <= 0) atomicAdd(ref + page, 1);  // a count below zero would never be free again
  }
  if (window < 0 && threadIdx.x == 0) key_len[s] = 0;
}

// ---------------------------------------------------------------------------
// With n pages in use: the k-th used page from n on moves to the k-th free page below n.  `work`:
// [0] the number of moves, then the sources, the destinations and each page's place (int32,
// num_pages each).
__global__ __launch_bounds__(kScanThreads) void compact_plan_kernel(const int32_t* ref, int32_t* ref_out,
                                                                    int32_t* __restrict__ work,
                                                                    int32_t* __restrict__ moved, int64_t num_pages) {
  __shared__ int counts[kScanThreads / 64];
  int32_t* src = work + 1;
  int32_t* dst = src + num_pages;
  int32_t* place = dst + num_pages;
  const auto in_use = [](int32_t r) { return r > 0; };
  int64_t used = 0;
  for (int64_t p0 = 0; p0 < num_pages; p0 += kScanThreads * kScanPer) {
    int total = 0;
    scan_bits(__popc(page_bits(ref, p0 + threadIdx.x * kScanPer, num_pages, in_use)), counts, total);
    used += total;
  }
  int64_t holes = 0, movers = 0;
  for (int64_t p0 = 0; p0 < num_pages; p0 += kScanThreads * kScanPer) {
    const int64_t at = p0 + threadIdx.x * kScanPer;
    const uint32_t in = page_bits(ref, at, num_pages, in_use);
    const int64_t left = (at < num_pages - kScanPer ? at + kScanPer : num_pages) - at;  // this thread's pages
    const uint32_t all = left >= kScanPer ? 0xffffu : left > 0 ? (1u << left) - 1 : 0u;
    const uint32_t low = used - at >= kScanPer ? 0xffffu : used > at ? (1u << (used - at)) - 1 : 0u;
    uint32_t hole = ~in & all & low, mover = in & ~low;
    int total = 0;
    int64_t k = holes + scan_bits(__popc(hole), counts, total);
    holes += total;
    for (; hole; hole &= hole - 1) dst[k++] = (int32_t)(at + __builtin_ctz(hole));
    k = movers + scan_bits(__popc(mover), counts, total);
    movers += total;
    for (; mover; mover &= mover - 1) src[k++] = (int32_t)(at + __builtin_ctz(mover));
    for (int i = 0; i < left && i < kScanPer; ++i) place[at + i] = in >> i & 1 ? (int32_t)(at + i) : -1;
  }
  __syncthreads();  // (as many holes as movers)
  for (int64_t k = threadIdx.x; k < movers; k += kScanThreads) place[src[k]] = dst[k];
  if (ref_out != ref)
    for (int64_t p = threadIdx.x; p < num_pages; p += kScanThreads) ref_out[p] = ref[p];
  __syncthreads();
  for (int64_t k = threadIdx.x; k < movers; k += kScanThreads) {
    const int32_t n = ref[src[k]];
    ref_out[dst[k]] = n;
    ref_out[src[k]] = 0;
  }
  if (threadIdx.x == 0) {
    work[0] = (int32_t)movers;
    if (moved) moved[0] = (int32_t)movers;
  }
}

// The moves, (move, cache, slice) items in turn, and the block tables' entries.
template <bool VEC>
__global__ __launch_bounds__(kPageThreads) void compact_move_kernel(const CacheList caches, const int32_t* tables,
                                                                    int32_t* tables_out,
                                                                    const int32_t* __restrict__ work,
                                                                    int64_t entries, int64_t num_pages,
                                                                    int64_t page_bytes, int slices) {
  const int32_t* src = work + 1;
  const int32_t* dst = src + num_pages;
  const int32_t* place = dst + num_pages;
  for (int64_t e = (int64_t)blockIdx.x * kPageThreads + threadIdx.x; e < entries;
       e += (int64_t)gridDim.x * kPageThreads) {
    const int32_t p = tables[e];
    tables_out[e] = p >= 0 && p < num_pages ? place[p] : -1;
  }
  // the next item's pages are read while this one is copied
  const int64_t items = (int64_t)work[0] * caches.n * slices;
  const auto move_of = [&](int64_t x) { return x / ((int64_t)caches.n * slices); };
  int64_t x = blockIdx.x;
  int32_t from = 0, to = 0;
  if (x < items) {
    from = src[move_of(x)];
    to = dst[move_of(x)];
  }
  while (x < items) {
    const int64_t next = x + gridDim.x, within = x % ((int64_t)caches.n * slices);
    int32_t from_next = 0, to_next = 0;
    if (next < items) {
      from_next = src[move_of(next)];
      to_next = dst[move_of(next)];
    }
    const int64_t at = within % slices * kSliceBytes;
    uint8_t* base = caches.base[within / slices];
    copy_bytes<VEC>(base + to * page_bytes + at, base + from * page_bytes + at,
                    page_bytes - at < kSliceBytes ? page_bytes - at : kSliceBytes);
    x = next;
    from = from_next;
    to = to_next;
  }
}

// Host lists of n values: all in [0, limit); those of `once` not twice, and none of `other` among them.
static int check_lists(const char* who, const char* once_name, const int32_t* once, const char* other_name,
                       const int32_t* other, int64_t n, int64_t limit) {
  std::vector<int32_t> sorted;
  try {
    sorted.assign(once, once + n);
  } catch (const std::exception&) {
    return fail(NVF_ERR_INVALID, "%s: no host memory for %lld entries", who, (long long)n);
  }
  std::sort(sorted.begin(), sorted.end());
  for (int64_t i = 0; i < n; ++i) {
    if (once[i] < 0 || once[i] >= limit)
      return fail(NVF_ERR_INVALID, "%s: %s %d is outside [0, %lld)", who, once_name, once[i], (long long)limit);
    if (i > 0 && sorted[(size_t)i] == sorted[(size_t)i - 1])
      return fail(NVF_ERR_INVALID, "%s: %s %d comes twice", who, once_name, sorted[(size_t)i]);
  }
  for (int64_t i = 0; other && i < n; ++i) {
    if (other[i] < 0 || other[i] >= limit)
      return fail(NVF_ERR_INVALID, "%s: %s %d is outside [0, %lld)", who, other_name, other[i], (long long)limit);
    if (std::binary_search(sorted.begin(), sorted.end(), other[i]))
      return fail(NVF_ERR_INVALID, "%s: %d is a %s and a %s", who, other[i], other_name, once_name);
  }
  return NVF_OK;
}

static int check_caches(const char* who, void* const* caches, int n_caches, int64_t num_pages, int64_t page_bytes) {
  if (n_caches < 0 || num_pages < 0 || num_pages > INT32_MAX || page_bytes <= 0 ||
      (page_bytes + kSliceBytes - 1) / kSliceBytes > INT32_MAX / (kMaxPairs * kMaxCaches))
    return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  if (n_caches > 0 && !caches) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  std::vector<uintptr_t> at;
  try {
    at.assign(reinterpret_cast<const uintptr_t*>(caches), reinterpret_cast<const uintptr_t*>(caches) + n_caches);
  } catch (const std::exception&) {
    return fail(NVF_ERR_INVALID, "%s: no host memory for %d caches", who, n_caches);
  }
  std::sort(at.begin(), at.end());
  for (int i = 0; i < n_caches; ++i) {
    if (!at[(size_t)i]) return fail(NVF_ERR_INVALID, "%s: NULL cache", who);
    if (i > 0 && at[(size_t)i] - at[(size_t)i - 1] < (uint64_t)(num_pages * page_bytes))
      return fail(NVF_ERR_INVALID, "%s: two caches overlap", who);
  }
  return NVF_OK;
}

// Calls f(caches of one launch, whether all are 16-byte vectors).
template <typename F>
static void by_caches(void* const* caches, int n_caches, bool vec, F f) {
  for (int c0 = 0; c0 < n_caches; c0 += kMaxCaches) {
    CacheList list{};
    list.n = std::min(kMaxCaches, n_caches - c0);
    bool v = vec;
    for (int i = 0; i < list.n; ++i) {
      list.base[i] = static_cast<uint8_t*>(caches[c0 + i]);
      v = v && aligned16(caches[c0 + i]);
    }
    f(list, v);
  }
}
template <typename F>
static void by_pairs(const int32_t* a, const int32_t* b, int64_t n, F f) {
  for (int64_t p0 = 0; p0 < n; p0 += kMaxPairs) {
    PairList list{};
    list.n = (int)std::min<int64_t>(kMaxPairs, n - p0);
    memcpy(list.a, a + p0, list.n * sizeof(int32_t));
    if (b) memcpy(list.b, b + p0, list.n * sizeof(int32_t));
    f(list, p0);
  }
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int nvf_copy_pages(void* const* caches_host, int n_caches, const int32_t* src_host, const int32_t* dst_host,
                   int64_t n, int64_t num_pages, int64_t page_bytes, void* stream) {
  const char* who = "nvf_copy_pages";
  int rc = check_caches(who, caches_host, n_caches, num_pages, page_bytes);
  if (rc != NVF_OK) return rc;
  if (n < 0 || n > num_pages) return fail(NVF_ERR_INVALID, "%s: bad number of pages", who);
  if (n > 0 && (!src_host || !dst_host)) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if ((rc = check_lists(who, "destination", dst_host, "source", src_host, n, num_pages)) != NVF_OK) return rc;
  if (n == 0 || n_caches == 0) return NVF_OK;
  const int slices = (int)((page_bytes + kSliceBytes - 1) / kSliceBytes);
  by_caches(caches_host, n_caches, page_bytes % 16 == 0, [&](const CacheList& caches, bool vec) {
    by_pairs(src_host, dst_host, n, [&](const PairList& pairs, int64_t) {
      const dim3 grid((unsigned)(pairs.n * caches.n * slices));
      const auto kernel = vec ? copy_pages_kernel<true> : copy_pages_kernel<false>;
      kernel<<<grid, kPageThreads, 0, as_stream(stream)>>>(caches, pairs, page_bytes, slices);
    });
  });
  return launch_status("copy_pages");
}

int nvf_fork_pages(void* const* caches_host, int n_caches, int32_t* block_tables, int32_t* key_len,
                   int32_t* ref_count, const int32_t* parent_host, const int32_t* child_host, int64_t n,
                   int32_t* new_page, int64_t table_rows, int max_blocks, int64_t num_pages, int block_size,
                   int64_t row_bytes, void* stream) {
  const char* who = "nvf_fork_pages";
  if (block_size <= 0 || row_bytes <= 0 || row_bytes > INT32_MAX) return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  const int64_t page_bytes = block_size * row_bytes;
  int rc = check_caches(who, caches_host, n_caches, num_pages, page_bytes);
  if (rc != NVF_OK) return rc;
  if (max_blocks <= 0 || table_rows < 0 || n < 0 || n > table_rows)
    return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  if (n == 0) return NVF_OK;
  if (!block_tables || !key_len || !ref_count || !parent_host || !child_host || !new_page)
    return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if ((rc = check_lists(who, "child", child_host, "parent", parent_host, n, table_rows)) != NVF_OK) return rc;
  const int slices = (int)((page_bytes + kSliceBytes - 1) / kSliceBytes);
  by_pairs(parent_host, child_host, n, [&](const PairList& forks, int64_t at) {
    fork_plan_kernel<<<dim3(1), kScanThreads, 0, as_stream(stream)>>>(block_tables, key_len, ref_count, forks,
                                                                     new_page + at, max_blocks, num_pages, block_size);
    by_caches(caches_host, n_caches, row_bytes % 16 == 0, [&](const CacheList& caches, bool vec) {
      const dim3 grid((unsigned)(forks.n * caches.n * slices));
      const auto kernel = vec ? fork_copy_kernel<true> : fork_copy_kernel<false>;
      kernel<<<grid, kPageThreads, 0, as_stream(stream)>>>(caches, forks, block_tables, key_len, new_page + at,
                                                           max_blocks, num_pages, block_size, row_bytes, slices);
    });
  });
  return launch_status("fork_pages");
}

int nvf_free_pages(int32_t* block_tables, int32_t* key_len, int32_t* ref_count, const int32_t* seqs_host, int64_t n,
                   int64_t table_rows, int max_blocks, int64_t num_pages, int block_size, int64_t window,
                   int64_t sinks, void* stream) {
  const char* who = "nvf_free_pages";
  if (max_blocks <= 0 || table_rows < 0 || n < 0 || n > table_rows || num_pages < 0 || block_size <= 0 || sinks < 0)
    return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  if (n == 0) return NVF_OK;
  if (!block_tables || !key_len || !ref_count || !seqs_host) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  const int rc = check_lists(who, "sequence", seqs_host, "", nullptr, n, table_rows);
  if (rc != NVF_OK) return rc;
  by_pairs(seqs_host, nullptr, n, [&](const PairList& seqs, int64_t) {
    free_pages_kernel<<<dim3((unsigned)seqs.n), kPageThreads, 0, as_stream(stream)>>>(
        block_tables, key_len, ref_count, seqs, max_blocks, num_pages, block_size, window, sinks);
  });
  return launch_status("free_pages");
}

int64_t nvf_compact_pages_workspace_size(int64_t num_pages) {
  return num_pages < 0 ? 0 : (3 * num_pages + 1) * (int64_t)sizeof(int32_t);
}

int nvf_compact_pages(void* const* caches_host, int n_caches, const int32_t* block_tables, const int32_t* ref_count,
                      int32_t* tables_out, int32_t* ref_out, int32_t* moved, int64_t table_rows, int max_blocks,
                      int64_t num_pages, int64_t page_bytes, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "nvf_compact_pages";
  const int rc = check_caches(who, caches_host, n_caches, num_pages, page_bytes);
  if (rc != NVF_OK) return rc;
  if (table_rows < 0 || max_blocks < 0) return fail(NVF_ERR_INVALID, "%s: bad shape", who);
  const int64_t entries = table_rows * max_blocks;
  if (!ref_count || !ref_out || !workspace || (entries > 0 && (!block_tables || !tables_out)))
    return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if (workspace_bytes < nvf_compact_pages_workspace_size(num_pages))
    return fail(NVF_ERR_INVALID, "%s: the workspace is too small", who);
  int32_t* work = static_cast<int32_t*>(workspace);
  hipStream_t st = as_stream(stream);
  compact_plan_kernel<<<dim3(1), kScanThreads, 0, st>>>(ref_count, ref_out, work, moved, num_pages);
  const int slices = (int)((page_bytes + kSliceBytes - 1) / kSliceBytes);
  const dim3 grid(1024);  // the moves' number is the device's: workgroups take them in turn (2048 of them: 290 us for 280)
  bool first = true;
  by_caches(caches_host, n_caches, page_bytes % 16 == 0, [&](const CacheList& caches, bool vec) {
    const auto kernel = vec ? compact_move_kernel<true> : compact_move_kernel<false>;
    kernel<<<grid, kPageThreads, 0, st>>>(caches, block_tables, tables_out, work, first ? entries : 0, num_pages,
                                          page_bytes, slices);
    first = false;
  });
  if (first)  // no caches: the tables alone
    compact_move_kernel<true><<<grid, kPageThreads, 0, st>>>(CacheList{}, block_tables, tables_out, work, entries,
                                                            num_pages, page_bytes, slices);
  return launch_status("compact_pages");
}

}  // extern "C"
