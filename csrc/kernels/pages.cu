// Page pool of a paged cache, kept on the device: fork, extend, truncate, compact, copy.
//
// State (int32, one reference count per page, one bit per free page, one length and one
// page-table row per slot).  Page 0 is the padding page: a table entry 0 means "no page".
// Every operation has one result, whatever the order of its threads: pages are handed out
// lowest free id first in request order, counts and bits change by integer atomics.
//
//   fork     child = parent's tokens: whole pages below min(length, share) are shared
//            (reference + 1), the rest is copied into fresh pages.
//   extend   a slot grows to new_len: fresh pages behind its last one; a partly filled last
//            page that others refer to is copied first (copy on write).
//   truncate a slot shrinks to new_len (0: it ends); a page without references is free.
//   compact  the n live pages end up with the ids below n (the j-th live page >= n moves to
//            the j-th free page < n), their data with them, and every table follows.
//
// fork, extend and compact are two launches: a plan by one CTA (requests are checked, counted
// and given pages; nothing changes when one is bad or pages are short) and an apply over the
// whole GPU (table rows, counts, page data).  The data is what bounds them: every copied page
// is read and written once in each layer of each cache.
#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace pages {

constexpr int T = 1024;
constexpr int kCopyThreads = 256;
constexpr int kPiece = kCopyThreads * 16 * 4;  // bytes of one copy work item: 4 x 16 per thread

// Scratch header (ints).
enum Head { kCopies = 0, kRequests = 1, kLive = 2, kHeadInts = 8 };

struct Scratch {
  int *head, *claim, *full, *off, *src, *dst, *remap;
};

__host__ __device__ inline Scratch scratch_of(const PagePoolArgs& a) {
  Scratch s;
  s.head = a.scratch;
  s.claim = s.head + kHeadInts;       // [slots], zero between calls
  s.full = s.claim + a.num_slots;     // [slots] first entry of a request that wants a page
  s.off = s.full + a.num_slots;       // [slots + 1] fresh pages before each request
  s.src = s.off + a.num_slots + 1;    // [pages] copies
  s.dst = s.src + a.num_pages;
  s.remap = s.dst + a.num_pages;      // [pages] compact: new id of a moved page
  return s;
}

ZS_DEVICE int pages_for(const PagePoolArgs& a, int tokens) { return tokens / a.page_size + (tokens % a.page_size > 0); }

// Exclusive prefix sums over the block (T threads) of two counts at once; *total gets the sums.
struct Two {
  int x, y;
};
ZS_DEVICE Two block_scan(Two v, Two* red, Two* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Two s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffff, s.x, o), y = __shfl_up_sync(0xffffffff, s.y, o);
    if (lane >= o) s.x += x, s.y += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  Two before = lane < warp ? red[lane] : Two{0, 0}, all = red[lane];
  before.x = (int)__reduce_add_sync(0xffffffff, (unsigned)before.x);
  before.y = (int)__reduce_add_sync(0xffffffff, (unsigned)before.y);
  total->x = (int)__reduce_add_sync(0xffffffff, (unsigned)all.x);
  total->y = (int)__reduce_add_sync(0xffffffff, (unsigned)all.y);
  return Two{before.x + s.x - v.x, before.y + s.y - v.y};
}

// This thread's words of the free map: contiguous, so ranks follow page ids.
struct Words {
  int w0, w1;
};
ZS_DEVICE Words my_words(const PagePoolArgs& a) {
  const int n = (a.num_pages + 31) / 32, per = (n + T - 1) / T;
  Words w;
  w.w0 = min(n, (int)threadIdx.x * per);
  w.w1 = min(n, w.w0 + per);
  return w;
}

// One reference of page p is dropped; without references it is free.
ZS_DEVICE void release(const PagePoolArgs& a, int p) {
  if (p <= 0 || p >= a.num_pages) {
    report_error(a.err, kErrBadShape);
    return;
  }
  const int old = atomicSub(a.refcount + p, 1);
  if (old == 1) {
    atomicOr(a.free_bits + (p >> 5), 1u << (p & 31));
  } else if (old <= 0) {  // was free: the tables did not agree with the counts
    atomicAdd(a.refcount + p, 1);
    report_error(a.err, kErrBadShape);
  }
}

// A request of a fork or extend: how many fresh pages it wants (-1: it cannot be served), from which
// table entry on, and the length that it gives its slot (-1: as it is).
struct Want {
  int pages, full, len;
};
ZS_DEVICE Want want(const PagePoolArgs& a, const Scratch& s, int i, bool fork) {
  const Want no = {-1, 0, -1};
  const int slot = a.slots[i], from = fork ? a.parents[i] : slot, lens = a.lens != nullptr ? a.lens[i] : 0x7FFFFFFF;
  if (slot < 0 || slot >= a.num_slots || from < 0 || from >= a.num_slots) return no;
  const int claimed = atomicExch(s.claim + slot, i + 1), own = a.seq_len[slot], len = a.seq_len[from];
  const long long most = (long long)a.max_pages * a.page_size;
  if (claimed != 0 || lens < 0 || len < 0 || len > most) return no;
  if (fork) {
    if (own != 0) return no;
    const int full = min(len, lens) / a.page_size;
    return Want{pages_for(a, len) - full, full, len};
  }
  if (lens > most) return no;
  const int have = pages_for(a, len);
  if (lens <= len) return Want{0, have, -1};
  int full = have;
  if (len % a.page_size != 0) {
    const int tail = a.page_table[(size_t)slot * a.max_pages + have - 1];
    if (tail < 0 || tail >= a.num_pages) return no;
    if (a.refcount[tail] > 1) full = have - 1;  // copy on write: the last page too
  }
  return Want{pages_for(a, lens) - full, full, lens};
}

// A thread per request, then a thread per fresh page: every chain of loads is walked once, side by
// side (256 forks of 32 prompts, then one of each grown, with the copies: 124 us with a warp per request
// in turn, 117 us so).
__global__ void __launch_bounds__(T) plan_kernel(const PagePoolArgs a, bool fork) {
  pdl_wait();
  pdl_trigger();
  __shared__ Two red[32];
  __shared__ int carry, off_near[T + 1];
  const Scratch s = scratch_of(a);
  const int tid = threadIdx.x;
  if (tid == 0) carry = 0;
  int* const off = a.n <= T ? off_near : s.off;  // fresh pages before each request
  const Words words = my_words(a);
  Two mine = {0, 0}, sum;
  for (int i = words.w0; i < words.w1; ++i) mine.y += __popc(a.free_bits[i]);
  Want first = {0, 0, -1};
  int bad = 0, rank = 0, have = 0;  // free pages before this thread's, of all
  for (int i0 = 0; i0 < a.n; i0 += T) {
    const int i = i0 + tid;
    Want w = {0, 0, -1};
    if (i < a.n) {
      w = want(a, s, i, fork);
      if (w.pages < 0) bad = 1, w.pages = 0;
      s.full[i] = w.full;
    }
    mine.x = w.pages;
    const Two before = block_scan(mine, red, &sum);
    const int base = carry;
    if (i < a.n) off[i] = base + before.x;
    if (i0 == 0) {
      first = w;
      rank = before.y;
      have = sum.y;
      mine.y = 0;
    }
    __syncthreads();
    if (tid == 0) carry = (int)min((long long)base + sum.x, 1ll << 30);  // more than any pool has
  }
  const bool valid = __syncthreads_or(bad) == 0;
  const int total = carry;
  const bool ok = valid && total <= have;
  for (int i = tid; i < a.n; i += T) {  // claims are given back before anyone else runs
    const int slot = a.slots[i];
    if (slot >= 0 && slot < a.num_slots) s.claim[slot] = 0;
  }
  if (tid == 0) {
    s.head[kCopies] = ok ? total : 0;
    s.head[kRequests] = ok ? a.n : 0;
    if (!ok) report_error(a.err, valid ? kErrNoPages : kErrBadShape);
    off[a.n] = total;
  }
  if (!ok) return;
  // The lowest free pages are taken.
  for (int i = words.w0; i < words.w1 && rank < total; ++i) {
    uint32_t bits = a.free_bits[i];
    while (bits != 0 && rank < total) {
      const int b = __ffs(bits) - 1;
      bits &= bits - 1;
      s.dst[rank++] = i * 32 + b;
    }
    a.free_bits[i] = bits;
  }
  __syncthreads();
  // Fresh pages into the tables; pages with old contents are listed for the copy.
  for (int k = tid; k < total; k += T) {
    int i = 0;  // its request: the last with off <= k, which is one with pages
    for (int hi = a.n; hi - i > 1;) {
      const int mid = (i + hi) >> 1;
      if (off[mid] <= k) i = mid;
      else hi = mid;
    }
    const int slot = a.slots[i], from = fork ? a.parents[i] : slot, j = s.full[i] + k - off[i], p = s.dst[k];
    const int q = j < pages_for(a, a.seq_len[from]) ? a.page_table[(size_t)from * a.max_pages + j] : 0;
    s.src[k] = q;  // 0: nothing to copy
    a.refcount[p] = 1;
    a.page_table[(size_t)slot * a.max_pages + j] = p;
    if (!fork && q != 0) release(a, q);  // the shared last page that this slot leaves
  }
  __syncthreads();
  // Lengths are written once all are read.
  for (int i = tid + T; i < a.n; i += T) {
    const int len = a.seq_len[fork ? a.parents[i] : a.slots[i]];
    off[i] = fork ? len : max(len, a.lens[i]);
  }
  __syncthreads();
  for (int i = tid; i < a.n; i += T) {
    const int len = i == tid ? first.len : off[i];
    if (len >= 0) a.seq_len[a.slots[i]] = len;
  }
}

// Copies the listed pages: a work item is kPiece bytes of one page in one layer of one cache, four
// loads of every thread on their way before its stores.  At the memory's rate: 7.0 TB/s read and
// written for the 359 MB of 256 forks (102 us), 6.2 TB/s for a compaction that moves 167 MB (54 us).
ZS_DEVICE void copy_pages(const PagePoolArgs& a, const int* src, const int* dst, int copies) {
  int per_page = 0;
  for (int c = 0; c < a.num_caches; ++c)
    per_page += a.cache_layers[c] * (int)((a.cache_page_bytes[c] + kPiece - 1) / kPiece);
  const long long items = (long long)copies * per_page;
  for (long long it = blockIdx.x; it < items; it += gridDim.x) {
    const int k = (int)(it / per_page);
    int rest = (int)(it % per_page), c = 0, pieces = 0;
    for (; c < a.num_caches; ++c) {
      pieces = (int)((a.cache_page_bytes[c] + kPiece - 1) / kPiece);
      if (rest < a.cache_layers[c] * pieces) break;
      rest -= a.cache_layers[c] * pieces;
    }
    const int from = src[k], to = dst[k];
    if (from <= 0 || from >= a.num_pages || to <= 0 || to >= a.num_pages) {
      if (from != 0 && threadIdx.x == 0) report_error(a.err, kErrBadShape);
      continue;
    }
    const size_t bytes = (size_t)a.cache_page_bytes[c];
    char* layer = static_cast<char*>(a.cache[c]) + (size_t)(rest / pieces) * a.num_pages * bytes;
    const size_t at = (size_t)(rest % pieces) * kPiece;
    const uint4* in = reinterpret_cast<const uint4*>(layer + from * bytes + at);
    uint4* out = reinterpret_cast<uint4*>(layer + to * bytes + at);
    const int n = (int)(min((size_t)kPiece, bytes - at) / 16);
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = threadIdx.x + j * kCopyThreads;
      if (x < n) v[j] = __ldcs(in + x);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int x = threadIdx.x + j * kCopyThreads;
      if (x < n) __stcs(out + x, v[j]);
    }
  }
}

__global__ void __launch_bounds__(kCopyThreads) apply_kernel(const PagePoolArgs a, bool fork) {
  pdl_wait();
  pdl_trigger();
  const Scratch s = scratch_of(a);
  const int n = s.head[kRequests];
  if (fork) {
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
      const int* old = a.page_table + (size_t)a.parents[i] * a.max_pages;
      int* row = a.page_table + (size_t)a.slots[i] * a.max_pages;
      for (int j = threadIdx.x; j < s.full[i]; j += kCopyThreads) {
        const int p = old[j];
        row[j] = p;
        if (p > 0 && p < a.num_pages) atomicAdd(a.refcount + p, 1);
        else report_error(a.err, kErrBadShape);
      }
    }
  }
  copy_pages(a, s.src, s.dst, s.head[kCopies]);
}

// One CTA per request.  Entries are taken out with an exchange, so a slot named twice ends at
// the shorter length and every page is released once.  Bound by its chain of atomics: 4.2 us for 48
// sequences of up to a few dozen pages, one page a thread.
__global__ void __launch_bounds__(128) truncate_kernel(const PagePoolArgs a) {
  pdl_wait();
  pdl_trigger();
  const int slot = a.slots[blockIdx.x], to = a.lens != nullptr ? a.lens[blockIdx.x] : 0;
  if (slot < 0 || slot >= a.num_slots || to < 0) {
    if (threadIdx.x == 0) report_error(a.err, kErrBadShape);
    return;
  }
  __shared__ int len;
  if (threadIdx.x == 0) len = atomicMin(a.seq_len + slot, to);
  __syncthreads();
  int* row = a.page_table + (size_t)slot * a.max_pages;
  const int end = min(pages_for(a, len), a.max_pages);
  for (int j = pages_for(a, to) + threadIdx.x; j < end; j += 128) {
    const int p = atomicExch(row + j, 0);
    if (p != 0) release(a, p);
  }
}

// Bound by its chain of loads and scans, 7.1 us for a pool of 4096 pages as for one of 256.
__global__ void __launch_bounds__(T) compact_plan_kernel(const PagePoolArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ Two red[32];
  const Scratch s = scratch_of(a);
  const Words w = my_words(a);
  Two mine = {0, 0}, sum;
  for (int i = w.w0; i < w.w1; ++i) mine.x += __popc(a.free_bits[i]);
  block_scan(mine, red, &sum);
  const int live = a.num_pages - sum.x;
  // Free pages below `live` and live pages from `live` on, each in id order: equally many.
  auto below = [&](int word) -> uint32_t {  // bits of the ids < live
    const int n = live - word * 32;
    return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
  };
  auto exists = [&](int word) -> uint32_t {
    const int n = a.num_pages - word * 32;
    return n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u;
  };
  mine.x = 0;  // holes; y: pages that move
  for (int i = w.w0; i < w.w1; ++i) {
    const uint32_t f = a.free_bits[i];
    mine.x += __popc(f & below(i));
    mine.y += __popc(~f & exists(i) & ~below(i));
  }
  const Two before = block_scan(mine, red, &sum);
  const int total = sum.x;
  int hole = before.x, mover = before.y;
  for (int i = w.w0; i < w.w1; ++i) {
    const uint32_t f = a.free_bits[i];
    for (uint32_t b = f & below(i); b != 0; b &= b - 1) s.dst[hole++] = i * 32 + __ffs(b) - 1;
    for (uint32_t b = ~f & exists(i) & ~below(i); b != 0; b &= b - 1) s.src[mover++] = i * 32 + __ffs(b) - 1;
    a.free_bits[i] = exists(i) & ~below(i);
  }
  __syncthreads();
  for (int k = threadIdx.x; k < total; k += T) {
    const int from = s.src[k], to = s.dst[k];
    s.remap[from] = to;
    a.refcount[to] = a.refcount[from];
    a.refcount[from] = 0;
  }
  if (threadIdx.x == 0) {
    s.head[kCopies] = total;
    s.head[kLive] = live;
  }
}

__global__ void __launch_bounds__(kCopyThreads) compact_apply_kernel(const PagePoolArgs a) {
  pdl_wait();
  pdl_trigger();
  const Scratch s = scratch_of(a);
  const int copies = s.head[kCopies], live = s.head[kLive];
  if (copies == 0) return;
  for (int slot = blockIdx.x; slot < a.num_slots; slot += gridDim.x) {
    int* row = a.page_table + (size_t)slot * a.max_pages;
    const int end = min(pages_for(a, a.seq_len[slot]), a.max_pages);
    for (int j = threadIdx.x; j < end; j += kCopyThreads) {
      const int p = row[j];
      if (p >= live && p < a.num_pages) row[j] = s.remap[p];
    }
  }
  copy_pages(a, s.src, s.dst, copies);
}

__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const PagePoolArgs a) {
  pdl_wait();
  pdl_trigger();
  copy_pages(a, a.copy_src, a.copy_dst, a.n);
}

int check(const PagePoolArgs& a) {
  if (a.num_pages < 1 || a.num_slots < 1 || a.max_pages < 1 || a.page_size < 1 || a.n < 0) return -1;
  if (a.num_caches < 0 || a.num_caches > ZS_POOL_MAX_CACHES || a.scratch == nullptr) return -1;
  for (int c = 0; c < a.num_caches; ++c)
    if (a.cache[c] == nullptr || a.cache_layers[c] < 1 || a.cache_page_bytes[c] < 16 || a.cache_page_bytes[c] % 16 != 0 ||
        reinterpret_cast<uintptr_t>(a.cache[c]) % 16 != 0)
      return -1;
  return 0;
}

constexpr int kGrid = 148 * 8;  // copy CTAs: 8 of 256 threads fill an SM

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : -2; }

}  // namespace pages
}  // namespace zs

extern "C" long long zs_pool_scratch_ints(int num_pages, int num_slots) {
  return zs::pages::kHeadInts + 3ll * num_slots + 1 + 3ll * num_pages;
}

extern "C" int zs_pool_fork(const PagePoolArgs* args, cudaStream_t stream) {
  const PagePoolArgs& a = *args;
  if (int e = zs::pages::check(a)) return e;
  if (a.n == 0) return 0;
  if (a.n > a.num_slots || a.parents == nullptr || a.slots == nullptr) return -1;
  zs_launch(zs::pages::plan_kernel, 1, zs::pages::T, 0, stream, a, true);
  zs_launch(zs::pages::apply_kernel, zs::pages::kGrid, zs::pages::kCopyThreads, 0, stream, a, true);
  return zs::pages::launched();
}

extern "C" int zs_pool_extend(const PagePoolArgs* args, cudaStream_t stream) {
  const PagePoolArgs& a = *args;
  if (int e = zs::pages::check(a)) return e;
  if (a.n == 0) return 0;
  if (a.n > a.num_slots || a.slots == nullptr || a.lens == nullptr) return -1;
  zs_launch(zs::pages::plan_kernel, 1, zs::pages::T, 0, stream, a, false);
  zs_launch(zs::pages::apply_kernel, zs::pages::kGrid, zs::pages::kCopyThreads, 0, stream, a, false);
  return zs::pages::launched();
}

extern "C" int zs_pool_truncate(const PagePoolArgs* args, cudaStream_t stream) {
  const PagePoolArgs& a = *args;
  if (int e = zs::pages::check(a)) return e;
  if (a.n == 0) return 0;
  if (a.slots == nullptr) return -1;
  zs_launch(zs::pages::truncate_kernel, a.n, 128, 0, stream, a);
  return zs::pages::launched();
}

extern "C" int zs_pool_compact(const PagePoolArgs* args, cudaStream_t stream) {
  const PagePoolArgs& a = *args;
  if (int e = zs::pages::check(a)) return e;
  zs_launch(zs::pages::compact_plan_kernel, 1, zs::pages::T, 0, stream, a);
  zs_launch(zs::pages::compact_apply_kernel, zs::pages::kGrid, zs::pages::kCopyThreads, 0, stream, a);
  return zs::pages::launched();
}

extern "C" int zs_pool_copy(const PagePoolArgs* args, cudaStream_t stream) {
  const PagePoolArgs& a = *args;
  if (int e = zs::pages::check(a)) return e;
  if (a.n == 0) return 0;
  if (a.copy_src == nullptr || a.copy_dst == nullptr) return -1;
  zs_launch(zs::pages::copy_kernel, zs::pages::kGrid, zs::pages::kCopyThreads, 0, stream, a);
  return zs::pages::launched();
}
