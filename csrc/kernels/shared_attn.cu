// Gated GQA attention over a paged cache whose sequences share leading pages.
//
// The step's rows attend through segments: a segment is a list of rows and a range of page
// positions that all of them share (a common prompt's pages, or one sequence's own).  Row r
// sees key t of a segment when t < seq_lens[r]; its output is the softmax over the keys of all
// its segments, merged from records (o, m, l) per (row, head) and part of a segment:
//   s_t = scale * q . k_t,  m = max s_t,  l = sum exp(s_t - m),  o = sum exp(s_t - m) v_t
//   out = sigmoid(gate) * (sum_j exp(m_j - M) o_j) / (sum_j exp(m_j - M) l_j),  M = max m_j.
// A row that sees no key gives 0.  Cache blocks are those of attention.cu.
//
// Work: a unit is (segment, kv head, up to 128 / G rows: 128 query slots = row x head of the
// GQA group), its keys go through 64-key tiles.  The tiles of all units, one after the other,
// are divided evenly over the CTAs (one per SM), so a CTA works on the end of one unit, some
// whole ones and the start of another; each such fragment leaves one record per slot, and a
// last kernel merges a row's records.  A prefix's pages are read once for 128 query slots
// instead of once per row; tails and prefixes run in one launch without a tail of idle SMs.
#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace sattn {

constexpr int D = 256;
constexpr int PAGE = 16;
constexpr int PREC = D + 4;              // record: o[256], m, l, padding to 16 bytes
constexpr int BLOCK = PAGE * D * 2;      // bytes of a (page, kv head) block
constexpr int SLOTS = ZS_SHARED_SLOTS;   // query slots of a unit
constexpr int TILE = 64;                 // keys of a tile
constexpr int TPAGES = TILE / PAGE;
constexpr int STAGE = TPAGES * BLOCK;    // one tile of K or V: 32 KiB
constexpr int STAGES = 4;
constexpr int COMPUTE = 128;             // softmax threads (warps 0-3), then a copy and an MMA warp
constexpr int THREADS = COMPUTE + 64;
constexpr int CTAS = ZS_SHARED_CTAS;
constexpr int MAX_SEGS = ZS_SHARED_MAX_SEGS;

// The plan (ints): header, then per segment its end page, tiles per unit, page-table row and
// longest row, the first tile of every segment, and the first segment of every CTA.
struct Work {
  int *total, *pend, *nt, *slot, *len, *tile0, *cta_seg;
};
__host__ __device__ inline Work work_of(const SharedAttnArgs& a) {
  Work w;
  w.total = a.work;
  w.pend = a.work + 4;
  w.nt = w.pend + a.num_segs;
  w.slot = w.nt + a.num_segs;
  w.len = w.slot + a.num_segs;
  w.tile0 = w.len + a.num_segs;
  w.cta_seg = w.tile0 + a.num_segs + 1;
  return w;
}

ZS_DEVICE int group_of(const SharedAttnArgs& a) { return a.num_q_heads / a.num_kv_heads; }
// First tile of CTA c when `total` tiles are divided over n CTAs, and the CTA of a tile.
ZS_DEVICE int first_tile(int total, int n, int c) { return (int)((long long)total * c / n); }
ZS_DEVICE int cta_of(int total, int n, int tile) { return (int)(((long long)(tile + 1) * n - 1) / total); }
ZS_DEVICE int active_ctas(int total) { return min(CTAS, total); }

// One CTA: the longest row of every segment decides how many pages it has; tiles are counted and
// the CTAs' ranges laid over them.
__global__ void __launch_bounds__(1024) plan_kernel(const SharedAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ unsigned long long longest[MAX_SEGS];  // (length, ~row)
  __shared__ int tile0[MAX_SEGS + 1];
  __shared__ long long red[32];
  const Work w = work_of(a);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int s = tid; s < a.num_segs; s += 1024) longest[s] = 0;
  __syncthreads();
  for (int e = tid; e < a.entries; e += 1024) {
    const int row = a.seg_rows[e];
    const int len = max(a.seq_lens[row], 0);
    atomicMax(&longest[a.entry_seg[e]], ((unsigned long long)len << 32) | (uint32_t)~row);
  }
  __syncthreads();
  const int rpu = SLOTS / group_of(a);
  long long carry = 0;
  for (int s0 = 0; s0 < a.num_segs; s0 += 1024) {
    const int s = s0 + tid;
    long long tiles = 0;
    if (s < a.num_segs) {
      const int len = (int)(longest[s] >> 32), row = (int)~(uint32_t)longest[s], p0 = a.seg_page0[s], p1 = a.seg_page1[s];
      int pend = (int)(((long long)len + PAGE - 1) / PAGE);
      if (p1 >= 0) pend = min(pend, p1);
      const int nt = (max(pend - p0, 0) + TPAGES - 1) / TPAGES;
      const int rows = a.seg_start[s + 1] - a.seg_start[s];
      tiles = (long long)nt * ((rows + rpu - 1) / rpu) * a.num_kv_heads;
      w.pend[s] = pend;
      w.nt[s] = nt;
      w.slot[s] = a.row_slot[row];
      w.len[s] = (int)min((long long)len, (long long)pend * PAGE);
    }
    long long x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffff, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) red[warp] = x;
    __syncthreads();
    long long before = carry, sum = carry;
    for (int j = 0; j < 32; ++j) {
      if (j < warp) before += red[j];
      sum += red[j];
    }
    if (s < a.num_segs) tile0[s] = w.tile0[s] = (int)(before + x - tiles);
    carry = sum;
  }
  const bool fits = carry < (1ll << 30);  // lengths beyond any cache: nothing is read
  if (tid == 0) {
    if (!fits) report_error(a.err, kErrBadShape);
    tile0[a.num_segs] = w.tile0[a.num_segs] = fits ? (int)carry : 0;
    *w.total = fits ? (int)carry : 0;
  }
  if (!fits) {
    for (int s = tid; s < a.num_segs; s += 1024) w.nt[s] = w.tile0[s] = 0;
    return;
  }
  __syncthreads();
  const int total = (int)carry, n = active_ctas(total);
  for (int c = tid; c < n; c += 1024) {
    const int t = first_tile(total, n, c);
    int lo = 0, hi = a.num_segs;  // the last segment with tile0 <= t (empty ones before it share its tile0)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile0[mid] <= t) lo = mid; else hi = mid;
    }
    w.cta_seg[c] = lo;
  }
}

// A CTA's part of one unit: tiles [t0, t1).
struct Fragment {
  int seg, kvh, e0, slots, t0, t1, p0, pend, len;
  const int* pt;
  bool first;  // holds the unit's first tile
};

struct Walk {
  int pos, end, seg, rpu, group;
  ZS_DEVICE bool next(const SharedAttnArgs& a, const Work& w, Fragment& f) {
    if (pos >= end) return false;
    while (pos >= w.tile0[seg + 1]) ++seg;
    const int nt = w.nt[seg], at = pos - w.tile0[seg], u = at / nt;
    const int e0 = a.seg_start[seg], rows = a.seg_start[seg + 1] - e0, nq = (rows + rpu - 1) / rpu;
    const int qt = u % nq;  // the units of one kv head follow one another: they read the same pages
    f.seg = seg;
    f.kvh = u / nq;
    f.e0 = e0 + qt * rpu;
    f.slots = min(rpu, rows - qt * rpu) * group;
    f.t0 = at - u * nt;
    f.t1 = min(nt, f.t0 + end - pos);
    f.p0 = a.seg_page0[seg];
    f.pend = w.pend[seg];
    f.len = w.len[seg];
    f.pt = a.page_table + (size_t)w.slot[seg] * a.max_pages;
    f.first = f.t0 == 0;
    pos += f.t1 - f.t0;
    return true;
  }
};

struct Smem {
  uint8_t q[D / 64][SLOTS * 128];   // Q: 128 slots, K-major, 4 chunks of 64 dims (128-byte swizzle)
  uint8_t ring[STAGES][STAGE];      // tiles as page images: K, V, K, V, ...
  uint8_t p[2][SLOTS * 128];        // P: 128 slots x 64 keys bf16, K-major
  float factor[SLOTS];
  int vote[2][4];
  int again[2];                     // the P in this buffer is followed by its rounding errors
  int least;                        // shortest visible length among a fragment's rows
  volatile int abort;
  uint32_t tmem;
  uint64_t full[STAGES], empty[STAGES], s_full[2], s_empty[2], p_full[2], p_empty[2], q_full;
};

// Waits give up when one of them in the CTA has run out (the error word is set then).
ZS_DEVICE bool wait_for(Smem& s, uint64_t* bar, uint32_t phase, int* err) {
  for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (s.abort) return false;
    if (i > 64) __nanosleep(64);
  }
  report_error(err, kErrMbarTimeout);
  s.abort = 1;
  return false;
}

ZS_DEVICE void compute_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
ZS_DEVICE bool compute_any(bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)x)
      : "memory");
  return r != 0;
}

ZS_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
ZS_DEVICE uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
ZS_DEVICE void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
ZS_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Byte offset of (key k, 16-byte piece pc of its 512-byte row) in a tile's page images.
ZS_DEVICE int tile_offset(int k, int pc) {
  return (k >> 4) * BLOCK + ((k >> 3) & 1) * 4096 + (pc >> 3) * 1024 + (k & 7) * 128 + (((pc & 7) ^ (k & 7)) << 4);
}
ZS_DEVICE bool not_finite(uint32_t two) {  // either of two bf16 is an infinity or NaN
  return (two & 0x7F80u) == 0x7F80u || (two & 0x7F800000u) == 0x7F800000u;
}

constexpr uint32_t kTmemO = 128;     // TMEM columns: S of two tiles, then O^T (2 x 128 dims, a column per slot)
constexpr uint32_t kTmemCols = 512;
constexpr float kGrow = 8.f;         // O is rescaled when a maximum grows by more than 2^8

// One CTA per SM; S = Q K^T (M = 128 slots, N = 64 keys) and O^T += V^T P^T (M = 128 dims twice,
// N = slots in use) on tcgen05.  Thread s of the softmax warps owns query slot s: a row of S is
// one TMEM lane, so maximum and sum need no exchange between threads.
//  * copy warp: page ids, then one bulk copy per (page, kv head) block into a ring of four 32 KiB
//    stages, running ahead across tiles and fragments;
//  * MMA warp: S of the next tile is issued before O of this one, so it runs under the softmax;
//  * softmax warps: P = 2^(s - m) with a reference m that follows the running maximum only when
//    that grows by more than 2^8 (P stays below 2^8, O and l in fp32), so O in TMEM is rescaled
//    rarely; the next fragment's Q is fetched during the last tile.
// P is rounded to bf16 for the tensor cores, 2^-8 of a weight; over many keys those errors
// average out, and where a weight is more than a quarter of the sum before its tile (first
// tiles, few keys, peaked rows) a second product adds what the rounding lost.  l sums the
// weights before they are rounded.
__global__ void __launch_bounds__(THREADS, 1) tiles_kernel(const SharedAttnArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 5) {
    tmem_alloc(&s.tmem, kTmemCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&s.full[i], 1);
      mbar_init(&s.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.s_empty[i], COMPUTE);
      mbar_init(&s.p_full[i], COMPUTE);
      mbar_init(&s.p_empty[i], 1);
    }
    mbar_init(&s.q_full, COMPUTE);
    s.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  pdl_wait();
  pdl_trigger();
  const Work w = work_of(a);
  const int total = *w.total, n = active_ctas(total), cta = blockIdx.x;
  Walk walk{0, 0, 0, SLOTS / group_of(a), group_of(a)};
  if (cta < n) {
    walk.pos = first_tile(total, n, cta);
    walk.end = first_tile(total, n, cta + 1);
    walk.seg = w.cta_seg[cta];
  }
  Fragment f;

  if (warp == 4) {
    // ------------------------------------------------------------------ copies
    // Lane j holds the page id of the tile's page j and issues its K and V blocks.
    const char* kc = static_cast<const char*>(a.k_cache);
    const char* vc = static_cast<const char*>(a.v_cache);
    int i = 0, issued = 0;  // tiles, stage uses
    bool ok = true;
    while (ok && walk.next(a, w, f)) {
      auto page_of = [&](int t) {
        const int p = f.p0 + t * TPAGES + lane;
        if (lane >= TPAGES || p >= f.pend) return 0;
        return p < a.max_pages ? __ldg(f.pt + p) : -1;  // a length behind the table row: a bad page
      };
      int page = page_of(f.t0);
      for (int t = f.t0; ok && t < f.t1; ++t, ++i) {
        const int after = t + 1 < f.t1 ? page_of(t + 1) : 0;
        const int np = min(TPAGES, f.pend - (f.p0 + t * TPAGES));
        if (page < 0 || page >= a.num_pages) {
          report_error(a.err, kErrBadShape);
          page = 0;
        }
        const size_t at = ((size_t)page * a.num_kv_heads + f.kvh) * BLOCK;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int st = (2 * i + kv) & (STAGES - 1);
          if (i >= 2) ok = ok && wait_for(s, &s.empty[st], ((i >> 1) - 1) & 1, a.err);
          ok = __all_sync(0xffffffff, ok);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&s.full[st], np * BLOCK);
          __syncwarp();
          if (lane < np) bulk_load(s.ring[st] + lane * BLOCK, (kv ? vc : kc) + at, BLOCK, &s.full[st]);
          ++issued;
        }
        page = after;
      }
    }
    // Copies in flight land before the CTA gives its shared memory back.
    if (lane == 0)
      for (int m = max(0, issued - STAGES); m < issued; ++m) mbar_wait(&s.full[m & (STAGES - 1)], (m / STAGES) & 1, nullptr);
  } else if (warp == 5) {
    // -------------------------------------------------------------------- MMA
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc_bf16(SLOTS, TILE, 0, 0);
      int ns = 0, no = 0;  // issued products: S of a tile, O of a round of P
      auto scores = [&](int i) {  // S of tile i
        const int st = (2 * i) & (STAGES - 1), b = i & 1;
        if (!wait_for(s, &s.full[st], (i >> 1) & 1, a.err)) return false;
        if (i >= 2 && !wait_for(s, &s.s_empty[b], ((i >> 1) - 1) & 1, a.err)) return false;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_bf16(tmem + b * TILE, make_smem_desc(smem_u32(s.q[c]) + k * 32, 16, 1024, 2),
                     make_smem_desc(smem_u32(s.ring[st] + c * 1024) + k * 32, 16, 4096, 2), idesc_s, (c | k) ? 1u : 0u);
        tc_commit(&s.empty[st]);
        tc_commit(&s.s_full[b]);
        ++ns;
        return true;
      };
      auto output = [&](int i, bool fresh, uint32_t idesc) {  // O^T of tile i: one or two rounds of P
        const int st = (2 * i + 1) & (STAGES - 1);
        if (!wait_for(s, &s.full[st], (i >> 1) & 1, a.err)) return false;
        for (bool again = true; again; fresh = false, ++no) {
          const int b = no & 1;
          if (!wait_for(s, &s.p_full[b], (no >> 1) & 1, a.err)) return false;
          tc_fence_after();
          again = s.again[b] != 0;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int k = 0; k < TPAGES; ++k)
              mma_bf16(tmem + kTmemO + mt * SLOTS, make_smem_desc(smem_u32(s.ring[st] + 2 * mt * 1024) + k * BLOCK, 1024, 4096, 2),
                       make_smem_desc(smem_u32(s.p[b]) + k * 32, 16, 1024, 2), idesc, (!fresh || k > 0) ? 1u : 0u);
          if (!again) tc_commit(&s.empty[st]);
          tc_commit(&s.p_empty[b]);
        }
        return true;
      };
      int i = 0, nf = 0;
      bool ok = true;
      for (; ok && walk.next(a, w, f); ++nf) {
        const uint32_t idesc_o = make_idesc_bf16(128, (f.slots + 15) & ~15, 1, 0);
        ok = wait_for(s, &s.q_full, nf & 1, a.err) && scores(i);
        for (int t = f.t0; ok && t < f.t1; ++t, ++i) {
          if (t + 1 < f.t1) ok = scores(i + 1);
          ok = ok && output(i, t == f.t0, idesc_o);
        }
      }
      // The issued products end before TMEM is released.
      if (ns > 0) mbar_wait(&s.s_full[(ns - 1) & 1], ((ns - 1) >> 1) & 1, nullptr);
      if (no > 0) mbar_wait(&s.p_empty[(no - 1) & 1], ((no - 1) >> 1) & 1, nullptr);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const float qscale = a.sm_scale * 1.4426950408889634f;  // exp2 domain
    const int group = walk.group;
    // Q of a fragment, 512 bytes a slot: slot = warp, warp + 4, ..
    auto fetch_q = [&](const Fragment& g) {
      for (int sl = warp; sl < g.slots; sl += 4) {
        const int row = a.seg_rows[g.e0 + sl / group];
        const char* src = static_cast<const char*>(a.q) + (((size_t)row * a.num_q_heads + g.kvh * group + sl % group) * D + lane * 8) * 2;
        cp_async16(smem_u32(s.q[lane >> 3]) + sl * 128 + (((lane & 7) ^ (sl & 7)) << 4), src);
      }
    };
    auto q_ready = [&]() {
      cp_async_wait();
      fence_proxy_async_shared();
      mbar_arrive(&s.q_full);
    };
    // After a wait that gave up these warps go on to the end with whatever is there (the error word
    // is set, every later wait gives up at once): their barriers always meet.
    bool more = walk.next(a, w, f);
    if (more) {
      fetch_q(f);
      q_ready();
    }
    int i = 0, pr = 0;  // tiles, rounds of P
    while (more) {
      Fragment g;
      const bool used = tid < f.slots, busy = warp * 32 < f.slots;
      const int limit = used ? min(a.seq_lens[a.seg_rows[f.e0 + tid / group]], f.len) : 0x7FFFFFFF;  // keys this slot sees
      {
        const int least = __reduce_min_sync(0xffffffff, limit);
        if (tid == 0) s.least = 0x7FFFFFFF;
        compute_sync();
        if (lane == 0) atomicMin(&s.least, least);
        compute_sync();
      }
      const int least = s.least;
      float m = -INFINITY, l = 0.f;  // reference maximum (raw scores) and sum of this slot
      for (int t = f.t0; t < f.t1; ++t, ++i) {
        const int b = i & 1, key0 = (f.p0 + t * TPAGES) * PAGE;
        wait_for(s, &s.s_full[b], (i >> 1) & 1, a.err);
        tc_fence_after();
        const bool last = t + 1 == f.t1;
        if (last) {  // every product with Q is done: the next fragment's Q can come
          more = walk.next(a, w, g);
          if (more) fetch_q(g);
        }
        uint32_t r[2][32];
        float mt = -INFINITY;
        const int valid = limit - key0;
        if (busy) {
          tmem_ld_32x32b_x32(tmem + b * TILE + lane_off, r[0]);
          tmem_ld_32x32b_x32(tmem + b * TILE + 32 + lane_off, r[1]);
          tmem_ld_wait();
          if (valid < TILE) {
#pragma unroll
            for (int j = 0; j < TILE; ++j)
              if (j >= valid) r[j >> 5][j & 31] = 0xFF800000u;  // -inf
          }
          float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < TILE; ++j) x[j & 3] = fmaxf(x[j & 3], __uint_as_float(r[j >> 5][j & 31]));
          mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        }
        tc_fence_before();
        mbar_arrive(&s.s_empty[b]);
        // The reference follows the maximum when that outgrew it (and at first).
        const bool grow = used && (m == -INFINITY ? mt > -INFINITY : (mt - m) * qscale > kGrow);
        float fac = 1.f;
        if (grow) {
          fac = m == -INFINITY ? 0.f : ex2((m - mt) * qscale);
          l *= fac;
          m = mt;
        }
        // A weight above a quarter of the sum so far: its bf16 rounding (2^-8) would show.
        const bool sharp = used && mt > -INFINITY && ex2((mt - m) * qscale) * 4.f > l;
        {
          const int any = (__any_sync(0xffffffff, grow) ? 1 : 0) | (__any_sync(0xffffffff, sharp) ? 2 : 0);
          if (lane == 0) s.vote[b][warp] = any;
          compute_sync();
        }
        const int votes = s.vote[b][0] | s.vote[b][1] | s.vote[b][2] | s.vote[b][3];
        const bool fine = (votes & 2) != 0;
        if ((votes & 1) && t > f.t0) {
          s.factor[tid] = fac;
          wait_for(s, &s.p_empty[(pr - 1) & 1], ((pr - 1) >> 1) & 1, a.err);  // O holds every tile before this one
          compute_sync();
          tc_fence_after();
          for (int c0 = 0; c0 < f.slots; c0 += 16)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t o[16];
              const uint32_t at = tmem + kTmemO + h * SLOTS + c0 + lane_off;
              tmem_ld_32x32b_x16(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * s.factor[c0 + j]);
              tmem_st_32x32b_x16(at, o);
            }
          tmem_st_wait();
          compute_sync();
        }
        int pb = pr & 1;
        if (pr >= 2) wait_for(s, &s.p_empty[pb], ((pr >> 1) - 1) & 1, a.err);  // the buffer's last P is read
        if (busy) {
          const float off = m == -INFINITY ? 0.f : m * qscale;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < TILE / 8; ++c) {
            uint32_t pk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = c * 8 + j * 2;
              const float lo = ex2(fmaf(__uint_as_float(r[k >> 5][k & 31]), qscale, -off));
              const float hi = ex2(fmaf(__uint_as_float(r[k >> 5][(k & 31) + 1]), qscale, -off));
              sum[j] += lo + hi;
              pk[j] = pack_bf16(lo, hi);
              r[k >> 5][k & 31] = __float_as_uint(lo);
              r[k >> 5][(k & 31) + 1] = __float_as_uint(hi);
            }
            *reinterpret_cast<uint4*>(s.p[pb] + tid * 128 + ((c ^ (tid & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        if (tid == 0) s.again[pb] = fine;
        // Values that a row does not see must not meet its zero weights as NaN or infinity.  Rows
        // of the tile that nobody sees are zeroed.  Rows that only some see are looked at: those
        // with such a value are zeroed too, and added by hand to the slots that see them.
        const int end = f.len - key0;  // keys of the tile that some row sees
        uint64_t odd = 0;
        if (end < TILE || least < key0 + TILE) {
          const int st = (2 * i + 1) & (STAGES - 1);
          wait_for(s, &s.full[st], (i >> 1) & 1, a.err);
          const int from = max(0, min(least - key0, TILE)), stop = min(end, TILE);
          bool found = false;
          for (int x = from * 32 + tid; x < stop * 32; x += COMPUTE) {
            const uint4 v = *reinterpret_cast<const uint4*>(s.ring[st] + tile_offset(x >> 5, x & 31));
            found |= not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w);
          }
          if (from < stop && compute_any(found)) {
            for (int k = from; k < stop; ++k) {  // 512 bytes a key, 4 a thread
              uint32_t* at = reinterpret_cast<uint32_t*>(s.ring[st] + tile_offset(k, tid >> 2)) + (tid & 3);
              if (compute_any(not_finite(*at))) {
                odd |= 1ull << k;
                *at = 0;
              }
            }
          }
          for (int x = max(end, 0) * 32 + tid; x < TILE * 32; x += COMPUTE)
            *reinterpret_cast<uint4*>(s.ring[st] + tile_offset(x >> 5, x & 31)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_shared();
        tc_fence_before();
        mbar_arrive(&s.p_full[pb]);
        ++pr;
        if (fine) {  // a second round: what the first one's rounding lost
          pb = pr & 1;
          if (pr >= 2) wait_for(s, &s.p_empty[pb], ((pr >> 1) - 1) & 1, a.err);
          if (busy) {
#pragma unroll
            for (int c = 0; c < TILE / 8; ++c) {
              uint32_t pk[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int k = c * 8 + j * 2;
                const float lo = __uint_as_float(r[k >> 5][k & 31]), hi = __uint_as_float(r[k >> 5][(k & 31) + 1]);
                const uint32_t x = pack_bf16(lo, hi);
                pk[j] = pack_bf16(lo - __uint_as_float(x << 16), hi - __uint_as_float(x & 0xFFFF0000u));
              }
              *reinterpret_cast<uint4*>(s.p[pb] + tid * 128 + ((c ^ (tid & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
          if (tid == 0) s.again[pb] = 0;
          fence_proxy_async_shared();
          mbar_arrive(&s.p_full[pb]);
          ++pr;
        }
        if (odd != 0) {
          wait_for(s, &s.p_empty[pb], ((pr - 1) >> 1) & 1, a.err);
          tc_fence_after();
          for (int c0 = 0; c0 < f.slots; c0 += 16)
            for (int h = 0; h < 2; ++h) {
              uint32_t o[16];
              const uint32_t at = tmem + kTmemO + h * SLOTS + c0 + lane_off;
              tmem_ld_32x32b_x16(at, o);
              tmem_ld_wait();
              for (int k = 0; k < TILE; ++k) {
                if (!(odd >> k & 1)) continue;
                const int at_page = (key0 + k) / PAGE, d = h * 128 + tid;
                const int page = at_page < a.max_pages ? f.pt[at_page] : -1;
                if (page < 0 || page >= a.num_pages) continue;
                const uint8_t* blk = static_cast<const uint8_t*>(a.v_cache) + ((size_t)page * a.num_kv_heads + f.kvh) * BLOCK;
                const float v = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(blk + tile_offset(k & 15, d >> 3) + (d & 7) * 2));
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  const int sl = c0 + j;
                  const int pat = sl * 128 + (((k >> 3) ^ (sl & 7)) << 4) + (k & 7) * 2;
                  float p = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(s.p[pb] + pat));
                  if (fine) p += __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(s.p[pb ^ 1] + pat));
                  if (p != 0.f) o[j] = __float_as_uint(__uint_as_float(o[j]) + p * v);
                }
              }
              tmem_st_32x32b_x16(at, o);
            }
          tmem_st_wait();
          tc_fence_before();
          compute_sync();  // all have read P before anyone writes the next
        }
      }
      if (more) q_ready();
      // ---- the fragment's records
      wait_for(s, &s.p_empty[(pr - 1) & 1], ((pr - 1) >> 1) & 1, a.err);
      tc_fence_after();
      float* rec = a.partial + (f.first ? ((size_t)f.e0 * a.num_q_heads + f.kvh * group) * PREC
                                        : ((size_t)a.entries * a.num_q_heads + (size_t)cta * SLOTS) * PREC);
      // Records of the unit's first fragment lie by (entry, head), those of a later one by slot.
      auto at = [&](int sl) { return rec + (f.first ? ((size_t)(sl / group) * a.num_q_heads + sl % group) : (size_t)sl) * PREC; };
      for (int c0 = 0; c0 < f.slots; c0 += 16)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(tmem + kTmemO + h * SLOTS + c0 + lane_off, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < f.slots) at(c0 + j)[h * 128 + tid] = __uint_as_float(o[j]);
        }
      if (used) {
        at(tid)[D] = m * qscale;
        at(tid)[D + 1] = l;
      }
      tc_fence_before();
      f = g;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
}

// One CTA per (row, q head), thread = dim.
__global__ void __launch_bounds__(D) merge_kernel(const SharedAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const Work w = work_of(a);
  const int row = blockIdx.x, h = blockIdx.y, d = threadIdx.x, group = group_of(a), rpu = SLOTS / group;
  const int total = *w.total, n = active_ctas(total);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int j = 0; j < a.levels; ++j) {
    const int e = a.row_entry[row * a.levels + j];
    if (e < 0) break;
    const int seg = a.entry_seg[e], nt = w.nt[seg];
    if (nt == 0) continue;
    const int at = e - a.seg_start[seg], nq = (a.seg_start[seg + 1] - a.seg_start[seg] + rpu - 1) / rpu;
    const int first = w.tile0[seg] + ((h / group) * nq + at / rpu) * nt;
    const int c0 = cta_of(total, n, first), c1 = cta_of(total, n, first + nt - 1);
    const float* rec = a.partial + ((size_t)e * a.num_q_heads + h) * PREC;
    const float* more = a.partial + ((size_t)a.entries * a.num_q_heads + (at % rpu) * group + h % group) * PREC;
    for (int c = c0; c <= c1; ++c) {
      if (c > c0) rec = more + (size_t)c * SLOTS * PREC;
      const float mr = rec[D];
      if (mr == -INFINITY) continue;
      const float mn = fmaxf(m, mr), s0 = m == -INFINITY ? 0.f : exp2f(m - mn), s1 = exp2f(mr - mn);
      l = l * s0 + rec[D + 1] * s1;
      o = o * s0 + rec[d] * s1;
      m = mn;
    }
  }
  float y = m == -INFINITY ? 0.f : o / l;
  const size_t at = ((size_t)row * a.num_q_heads + h) * D + d;
  if (a.gate != nullptr) y *= sigmoidf_(__bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[at]));
  if (a.out_bf16 != nullptr) static_cast<__nv_bfloat16*>(a.out_bf16)[at] = __float2bfloat16_rn(y);
  if (a.out_q != nullptr) {
    const uint8_t code = mx_scale_e8m0(warp_max(fabsf(y)));
    a.out_q[at] = f32_to_e4m3(y * mx_inv_scale(code));
    if ((d & 31) == 0) {
      const int kb = h * (D / 32) + (d >> 5);
      a.out_sf[((size_t)(row >> 7) * (a.num_q_heads * D >> 7) + (kb >> 2)) * 512 + sf_atom_offset(row & 127, kb & 3)] = code;
    }
  }
}

int check(const SharedAttnArgs& a) {
  if (a.num_kv_heads < 1 || a.num_q_heads % a.num_kv_heads != 0 || a.num_q_heads / a.num_kv_heads > ZS_SHARED_MAX_GROUP) return -1;
  if (a.head_dim != D || a.page_size != PAGE || a.levels < 1 || a.num_segs < 0 || a.num_segs > MAX_SEGS || a.rows < 0) return -1;
  if (a.work == nullptr || a.max_pages < 1 || a.max_pages > (1 << 26)) return -1;
  return 0;
}

}  // namespace sattn
}  // namespace zs

extern "C" int zs_shared_attn_plan(const SharedAttnArgs* args, cudaStream_t stream) {
  const SharedAttnArgs& a = *args;
  if (int e = zs::sattn::check(a)) return e;
  if (a.rows == 0) return 0;
  zs_launch(zs::sattn::plan_kernel, 1, 1024, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_shared_attn(const SharedAttnArgs* args, cudaStream_t stream) {
  const SharedAttnArgs& a = *args;
  if (int e = zs::sattn::check(a)) return e;
  if (a.partial == nullptr || !(a.sm_scale > 0.f) || a.num_pages < 1) return -1;
  if (a.rows == 0) return 0;
  const size_t smem = sizeof(zs::sattn::Smem) + 1024;
  cudaFuncSetAttribute(zs::sattn::tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  zs_launch(zs::sattn::tiles_kernel, zs::sattn::CTAS, zs::sattn::THREADS, smem, stream, a);
  zs_launch(zs::sattn::merge_kernel, dim3(a.rows, a.num_q_heads), zs::sattn::D, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
