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
// Work: a unit is up to 128 / G rows (128 query slots = row x head of the GQA group) and a kv
// head.  It goes through its pieces, the segments of those rows one after the other, in 64-key
// tiles: a common prompt fills a unit or several, the own tokens of many sequences are pieces of
// one.  The tiles of all units, one after the other, are divided evenly over the CTAs (one per
// SM); a CTA's part of a unit leaves one record per slot that had tiles there, and a last kernel
// merges a row's records.  A prefix's pages are read once for 128 query slots instead of once per
// row, and tails and prefixes run in one launch without a tail of idle SMs.
#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace sattn {

constexpr int D = 256;
constexpr int PAGE = 16;
constexpr int PREC = D + 4;              // record: o[256], m, l of either half of the keys, padding to 16 bytes
constexpr int BLOCK = PAGE * D * 2;      // bytes of a (page, kv head) block
constexpr int SLOTS = ZS_SHARED_SLOTS;   // query slots of a unit
constexpr int TILE = 64;                 // keys of a tile
constexpr int TPAGES = TILE / PAGE;
constexpr int STAGE = TPAGES * BLOCK;    // one tile of K or V: 32 KiB
constexpr int STAGES = 2;                // of K, and of V
constexpr int COMPUTE = 256;             // softmax threads (warps 0-7), then K copy, MMA, lookup and V copy warps
constexpr int THREADS = COMPUTE + 128;
constexpr int AHEAD = 3;                 // pieces known at a time
constexpr int CTAS = ZS_SHARED_CTAS;
constexpr int MAX_SEGS = ZS_SHARED_MAX_SEGS;
constexpr int MAX_PIECES = ZS_SHARED_MAX_PIECES;

// The plan (ints): header (cost of one kv head), a Piece for each piece and one behind the last (its
// cost0 alone), per entry and kv head the first CTA and the number of CTAs that have tiles of it and
// its first slot, and the range of costs and first piece of every CTA.
struct Piece {
  int cost0, nt, over, e0;    // cost before it, tiles, cost of the unit that it starts (or 0), the unit's first entry
  int rows, r0, r1, p0;       // rows of the unit, the piece's rows in it, first page
  int pend, len, table, pad;  // last page + 1, its longest row's length (at most that end) and page-table row
};
struct Work {
  int* head;
  Piece* piece;
  int4 *entry, *cta;
};
__host__ __device__ inline Work work_of(const SharedAttnArgs& a) {
  Work w;
  w.head = a.work;
  w.piece = reinterpret_cast<Piece*>(a.work + 4);
  w.entry = reinterpret_cast<int4*>(w.piece + a.num_pieces + 1);
  w.cta = w.entry + (size_t)a.entries * a.num_kv_heads;
  return w;
}

ZS_DEVICE int group_of(const SharedAttnArgs& a) { return a.num_q_heads / a.num_kv_heads; }
// The last i in [0, n) with x[i] <= v (x ascending, x[0] <= v).
ZS_DEVICE int last_at(const int* x, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (x[mid] <= v) lo = mid; else hi = mid;
  }
  return lo;
}

// One CTA: the longest row of every segment decides how many pages it has; costs are counted and
// the CTAs' ranges laid over them.
__global__ void __launch_bounds__(1024) plan_kernel(const SharedAttnArgs a) {
  pdl_trigger();
  __shared__ unsigned long long longest[MAX_SEGS];  // (length, ~entry)
  __shared__ int table[MAX_SEGS];
  __shared__ int cost0[MAX_PIECES + 1], start[CTAS + 1];
  __shared__ uint8_t over[MAX_PIECES];
  __shared__ long long red[32];
  const Work w = work_of(a);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int s = tid; s < a.num_segs; s += 1024) longest[s] = 0;
  // The plan's own tensors do not change: what a thread needs of them first is read before the wait.
  const bool e_in = tid < a.entries, p_in = tid < a.num_pieces;
  const int row = e_in ? a.seg_rows[tid] : 0, seg = e_in ? a.entry_seg[tid] : 0, slot = e_in ? a.row_slot[row] : 0;
  // (entry, kv head) pair `tid`
  const int of = tid / a.num_kv_heads, of_piece = of < a.entries ? a.entry_piece[of] : 0, of_unit = of < a.entries ? a.pieces[8 * of_piece + 1] : 0;
  const int4 px = p_in ? reinterpret_cast<const int4*>(a.pieces)[2 * tid] : make_int4(0, 0, 0, 0);
  const int4 py = p_in ? reinterpret_cast<const int4*>(a.pieces)[2 * tid + 1] : make_int4(0, 0, 0, 0);
  __syncthreads();
  pdl_wait();
  auto key = [&](int e, int r) { return ((unsigned long long)max(a.seq_lens[r], 0) << 32) | (uint32_t)~e; };
  const unsigned long long mine = e_in ? key(tid, row) : 0;
  if (e_in) atomicMax(&longest[seg], mine);
  for (int e = tid + 1024; e < a.entries; e += 1024) atomicMax(&longest[a.entry_seg[e]], key(e, a.seg_rows[e]));
  __syncthreads();
  if (e_in && longest[seg] == mine) table[seg] = slot;
  for (int e = tid + 1024; e < a.entries; e += 1024) {
    const int s = a.entry_seg[e];
    if ((uint32_t)longest[s] == (uint32_t)~e) table[s] = a.row_slot[a.seg_rows[e]];
  }
  __syncthreads();
  const int group = group_of(a);
  long long carry = 0;
  for (int i0 = 0; i0 < a.num_pieces; i0 += 1024) {
    const int i = i0 + tid;
    long long cost = 0;
    Piece g = {};
    if (i < a.num_pieces) {
      // (segment, unit's first entry, unit's rows, unit's first piece), (the next unit's first piece, its
      // rows r0 << 16 | r1 of the unit, pages p0..p1)
      const int4 x = i0 == 0 ? px : reinterpret_cast<const int4*>(a.pieces)[2 * i];
      const int4 y = i0 == 0 ? py : reinterpret_cast<const int4*>(a.pieces)[2 * i + 1];
      const int len = (int)(longest[x.x] >> 32);
      g.e0 = x.y;
      g.rows = x.z;
      // What a piece costs besides its tiles, in tiles of 1.1 us: another Q, 0.9 us; for a unit's first
      // one also the last unit's records and a pipeline that starts anew, 6 to 7 us with 128 slots
      // (eight prompts: 36.9 us the call with 6 tiles for it, 39.8 with 4, 36.7 with 7; four rows a
      // sequence: 57.3, 57.3, 58.2).
      g.over = x.w == i ? 4 + x.z * group / 64 : 1;
      g.r0 = y.y >> 16;
      g.r1 = y.y & 0xFFFF;
      g.p0 = y.z;
      g.pend = (int)(((long long)len + PAGE - 1) / PAGE);
      if (y.w >= 0) g.pend = min(g.pend, y.w);
      g.nt = (max(g.pend - g.p0, 0) + TPAGES - 1) / TPAGES;
      g.len = (int)min((long long)len, (long long)g.pend * PAGE);
      g.table = table[x.x];
      if (g.nt == 0 && x.w != i) g.over = 0;
      cost = g.nt + g.over;
    }
    long long x = cost;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffff, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) red[warp] = x;
    __syncthreads();
    long long before = lane < warp ? red[lane] : 0, sum = red[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffff, before, o);
      sum += __shfl_xor_sync(0xffffffff, sum, o);
    }
    if (i < a.num_pieces) {
      g.cost0 = (int)(carry + before + x - cost);
      cost0[i] = g.cost0;
      over[i] = (uint8_t)g.over;
      w.piece[i] = g;
    }
    carry += sum;
    __syncthreads();
  }
  const bool fits = carry * a.num_kv_heads < (1ll << 30);  // lengths beyond any cache: nothing is read
  const int each = fits ? (int)carry : 0, total = each * a.num_kv_heads, n = min(CTAS, total);
  if (tid == 0) {
    if (!fits) report_error(a.err, kErrBadShape);
    cost0[a.num_pieces] = w.piece[a.num_pieces].cost0 = each;
    w.head[0] = each;
  }
  __syncthreads();
  // Equal shares; a border within what a unit's start costs moves to the start, which then costs
  // nobody anything.
  int at = total, in = 0;
  if (tid < n) {
    at = total / n * tid + total % n * tid / n;
    const int rel = at % each;
    in = last_at(cost0, a.num_pieces, rel);
    if (over[in] > 1 && rel < cost0[in] + over[in]) at += cost0[in] - rel;
  }
  if (tid <= CTAS) start[tid] = at;
  __syncthreads();
  if (tid < CTAS) w.cta[tid] = make_int4(at, start[tid + 1], in, 0);
  for (int x = tid; x < a.entries * a.num_kv_heads; x += 1024) {
    const int e = x == tid ? of : x / a.num_kv_heads, i = x == tid ? of_piece : a.entry_piece[e];
    const int first = (x - e * a.num_kv_heads) * each + cost0[i] + over[i], nt = fits ? max(0, cost0[i + 1] - cost0[i] - over[i]) : 0;
    const int c0 = nt > 0 ? last_at(start, CTAS, first) : 0, c1 = nt > 0 ? last_at(start, CTAS, first + nt - 1) : -1;
    w.entry[x] = make_int4(c0, c1 - c0 + 1, (e - (x == tid ? of_unit : a.pieces[8 * i + 1])) * group, 0);
  }
}

// A CTA's part of a piece: tiles [t0, t1) for the slots [s0, s1) of its unit.
struct Fragment {
  int kvh, e0, slots, s0, s1, t0, t1, p0, pend, len, table;
  int first;  // of the unit in this CTA
};

struct Walk {
  int pos, end, i, each, group;
  int kvh, e0;
  ZS_DEVICE bool next(const SharedAttnArgs& a, const Work& w, Fragment& f) {
    while (pos < end) {
      const int4* at4 = reinterpret_cast<const int4*>(w.piece + i);
      const int4 x = __ldg(at4), y = __ldg(at4 + 1), z = __ldg(at4 + 2);
      const int head = pos / each, at = pos - head * each - x.x;
      if (at >= __ldg(&w.piece[i + 1].cost0) - x.x) {  // behind this piece: the next one
        ++i;
        continue;
      }
      const int cost = x.y + x.z;
      f.t0 = max(0, at - x.z);
      f.t1 = min(x.y, at - x.z + end - pos);
      pos += min(cost - at, end - pos);
      if (pos == (head + 1) * each) i = 0;  // the next kv head
      if (f.t1 <= f.t0) continue;
      f.first = head != kvh || x.w != e0;
      f.kvh = kvh = head;
      f.e0 = e0 = x.w;
      f.slots = y.x * group;
      f.s0 = y.y * group;
      f.s1 = y.z * group;
      f.p0 = y.w;
      f.pend = z.x;
      f.len = z.y;
      f.table = z.z;
      return true;
    }
    return false;
  }
};

struct Smem {
  uint8_t ring[2][STAGES][STAGE];   // tiles of K, and of V, as page images
  uint8_t way[SLOTS][528];          // Q on its way to TMEM, 512 bytes a slot
  float stage[8][32][20];           // a warp's 32 slots x 16 dims of O on their way out
  float top[2][2][SLOTS];           // per half of a tile's keys, the largest score of every slot
  Fragment frag[AHEAD];             // t1 == 0: no more
  int limit[AHEAD][SLOTS];          // keys that each slot sees (0: unused)
  int least[AHEAD];                 // the fewest among the piece's slots
  volatile int abort;
  uint32_t tmem;
  uint64_t full[2][STAGES], empty[2][STAGES], s_full[2], p_full[2], o_full[2], q_full, f_full[AHEAD], f_empty[AHEAD], r_full[AHEAD], way_full[2], way_empty[2];
};
constexpr int SMEM = (int)sizeof(Smem);
static_assert(SMEM <= 232448, "shared memory of one CTA");

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

ZS_DEVICE void compute_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
ZS_DEVICE bool compute_any(bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 256, p;\n\t"
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
// Towards zero, so that what is left of a positive number is not negative.
ZS_DEVICE uint32_t pack_bf16_down(float lo, float hi) {
  uint32_t r;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// c ? x : y, opaque: a chain of them over an array is not turned into an indexed load, which
// would move the whole array from registers to local memory.
ZS_DEVICE float pick(bool c, float x, float y) {
  float r;
  asm("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\tselp.f32 %0, %1, %2, p;\n\t}" : "=f"(r) : "f"(x), "f"(y), "r"((int)c));
  return r;
}
ZS_DEVICE void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Arrives on the barrier when the thread's copies so far have landed.
ZS_DEVICE void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
ZS_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// One tcgen05.mma with A in TMEM.  The B descriptors of a product differ in their low words alone
// (start address, leading offset): the high word (stride, version, 128-byte swizzle) is a constant.
constexpr uint32_t desc_hi(uint32_t stride) { return (stride >> 4) | (1u << 14) | (2u << 29); }
ZS_DEVICE uint32_t desc_lo(const void* p, uint32_t lead) { return (smem_u32(p) >> 4) | ((lead >> 4) << 16); }
constexpr uint32_t kHiB = desc_hi(4096);  // 8-key groups of a tile are 4 KiB apart
ZS_DEVICE void mma_step(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((int)add), "n"(kHiB)
      : "memory");
}
// The same for some rows of D: lanes whose bit in `off` is set keep what they hold.
ZS_DEVICE void mma_step_rows(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, const uint32_t (&off)[4], bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, {%6, %7, %8, %9}, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((int)add), "n"(kHiB), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
      : "memory");
}

// Byte offset of (key k, 16-byte piece pc of its 512-byte row) in a tile's page images.
ZS_DEVICE int tile_offset(int k, int pc) {
  return (k >> 4) * BLOCK + ((k >> 3) & 1) * 4096 + (pc >> 3) * 1024 + (k & 7) * 128 + (((pc & 7) ^ (k & 7)) << 4);
}
ZS_DEVICE bool not_finite(uint32_t two) {  // either of two bf16 is an infinity or NaN
  return (two & 0x7F80u) == 0x7F80u || (two & 0x7F800000u) == 0x7F800000u;
}

// TMEM columns: two S buffers of 64 (P as bf16 pairs takes their place: 32 columns, then 32 for its
// rounding errors), Q as bf16 pairs, O.
constexpr uint32_t kTmemQ = 128, kTmemO = 256, kTmemCols = 512;
constexpr float kGrow = 8.f;         // O is rescaled when a maximum grows by more than 2^8

// One CTA per SM; S = Q K^T (M = 128 slots, N = 64 keys, K-major) and O += P V (M = 128 slots,
// N = 256 dims, V read MN-major) on tcgen05, with Q and P as the TMEM operand: shared memory
// then carries only the copies in and one read of K and V per tile (with Q and P^T there the
// kernel was bound by shared-memory bandwidth).  A row of S, P and O is one TMEM lane; thread
// (half, slot) of the softmax warps owns half of the keys of a tile, and of the dims of O.
//  * copy warps, K and V: page ids, then one bulk copy per (page, kv head) block into two 32 KiB
//    stages each, running ahead across tiles and pieces;
//  * MMA warp: S of the next tile is issued before O of this one, so it runs under the softmax;
//  * lookup warp: the next fragments, their rows and lengths, and their Q into shared memory;
//  * softmax warps: P = 2^(s - m) with a reference m that follows the running maximum only when
//    that grows by more than 2^8 (P stays below 2^8, O and l in fp32), so O in TMEM is rescaled
//    rarely; the next fragment's Q goes to TMEM during this one's last tile.
// The tensor cores take P as bf16, so it goes through them twice: cut to bf16, and what the cut left
// (2^-17 of a weight is lost then).  A single product loses 2^-9 of every weight, and as values of
// either sign cancel in the output as much as those errors do, that is 2^-9 of the output too, as much
// again as its own rounding (0.0021 of the result's norm at 2000 and 33000 keys, 0.0017 so).  Left out
// where no weight is above a quarter of the sum so far, the second product saved 0, 3 and 4 % of a call
// (eight prompts, the same with four rows a sequence, a long document).  l sums the weights before
// they are cut.  Both parts are positive, so that an infinite value that a row sees stays that infinity.
// Long pieces run at 1.0 to 1.1 us a tile and CTA; the three products take 0.8 us of it (1536
// clocks at 4096 multiply-adds a clock).  A copy takes 2 us from its issue to its S, and two of K are on
// their way at a time; S and P in places of their own, so that the next S need not wait for O, gave
// 1.15 us.  What short calls pay for is the way to the first tile (5 us from the plan's end: range,
// piece, rows, Q) and a unit's records (3.6 us for 128 slots, 5.5 TB/s over all SMs).
__global__ void __launch_bounds__(THREADS, 1) tiles_kernel(const SharedAttnArgs a) {
  extern __shared__ __align__(1024) uint8_t raw[];
  Smem& s = *reinterpret_cast<Smem*>(raw);
  if ((smem_u32(raw) & 1023) != 0) {  // the swizzled images need it
    report_error(a.err, kErrBadShape);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 9) {
    tmem_alloc(&s.tmem, kTmemCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int kv = 0; kv < 2; ++kv)
      for (int i = 0; i < STAGES; ++i) {
        mbar_init(&s.full[kv][i], 1);
        mbar_init(&s.empty[kv][i], 1);
      }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], COMPUTE);
      mbar_init(&s.o_full[i], 1);
    }
    mbar_init(&s.q_full, COMPUTE);
    for (int i = 0; i < AHEAD; ++i) {
      mbar_init(&s.f_full[i], 1);
      mbar_init(&s.r_full[i], 32);
      mbar_init(&s.f_empty[i], COMPUTE / 32 + 3);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.way_full[i], 32);
      mbar_init(&s.way_empty[i], COMPUTE);
    }
    s.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  if (warp >= COMPUTE / 32) {  // the softmax warps have something to do first
    pdl_wait();
    pdl_trigger();
  }
  const int cta = blockIdx.x, group = group_of(a);
  // Fragment k of the CTA, once the lookup warp has it; false when there is none (or a wait gave up).
  int fk = 0;
  uint32_t fph = 0;
  auto next_fragment = [&](Fragment& f) {
    // The softmax warps give its place back when they are through with the piece (they also read the
    // limits there), the copy and MMA warps as soon as they have read it: none of them may be so far
    // behind that the lookup warp writes the next piece over one that it has yet to read.
    const bool reader = warp >= COMPUTE / 32;
    bool ok = wait_for(s, &s.f_full[fk], fph, a.err);
    if (reader) ok = __all_sync(0xffffffff, ok);
    if (!ok) return false;
    f = s.frag[fk];
    if (reader) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&s.f_empty[fk]);
    }
    if (++fk == AHEAD) {
      fk = 0;
      fph ^= 1;
    }
    return f.t1 > 0;
  };
  Fragment f;

  if (warp == 8 || warp == 11) {
    // ------------------------------------------------------------------ copies
    // Warp 8 brings K, warp 11 V.  Lane j holds the page id of the tile's page j and issues its block.
    const int kv = warp == 8 ? 0 : 1;
    const char* cache = static_cast<const char*>(kv ? a.v_cache : a.k_cache);
    int i = 0;  // tiles asked for
    bool ok = true;
    while (ok && __all_sync(0xffffffff, next_fragment(f))) {
      const int* pt = a.page_table + (size_t)f.table * a.max_pages;
      auto page_of = [&](int t) {
        const int p = f.p0 + t * TPAGES + lane;
        if (lane >= TPAGES || p >= f.pend) return 0;
        return p < a.max_pages ? __ldg(pt + p) : -1;  // a length behind the table row: a bad page
      };
      int page = page_of(f.t0);
      for (int t = f.t0; t < f.t1; ++t, ++i) {
        const int after = t + 1 < f.t1 ? page_of(t + 1) : 0;
        const int np = min(TPAGES, f.pend - (f.p0 + t * TPAGES)), st = i & 1;
        if (page < 0 || page >= a.num_pages) {
          report_error(a.err, kErrBadShape);
          page = 0;
        }
        if (i >= STAGES) ok = wait_for(s, &s.empty[kv][st], ((i >> 1) - 1) & 1, a.err);
        ok = __all_sync(0xffffffff, ok);
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&s.full[kv][st], np * BLOCK);
        __syncwarp();
        if (lane < np)
          bulk_load(s.ring[kv][st] + lane * BLOCK, cache + ((size_t)page * a.num_kv_heads + f.kvh) * BLOCK, BLOCK, &s.full[kv][st]);
        page = after;
      }
    }
    // Copies in flight land before the CTA gives its shared memory back.
    if (lane == 0)
      for (int m = max(0, i - STAGES); m < i; ++m) mbar_wait(&s.full[kv][m & 1], (m >> 1) & 1, nullptr);
  } else if (warp == 9) {
    // -------------------------------------------------------------------- MMA
    // The warp stays together; one elected lane issues.
    const bool leader = elect_one();
    const uint32_t idesc_s = make_idesc_bf16(SLOTS, TILE, 0, 0), idesc_o = make_idesc_bf16(SLOTS, D, 0, 1);
    const uint32_t k_lo = desc_lo(s.ring[0], 16), v_lo = desc_lo(s.ring[1], 1024);
    int ns = 0, no = 0;  // issued products
    auto scores = [&](int i) {  // S of tile i
      const int st = i & 1;
      if (!wait_for(s, &s.full[0][st], (i >> 1) & 1, a.err)) return false;
      // It takes the place of the P two tiles before: products with different accumulators have
      // no order of their own.
      if (i >= 2 && !wait_for(s, &s.o_full[i & 1], ((i >> 1) - 1) & 1, a.err)) return false;
      tc_fence_after();
      const uint32_t k_at = k_lo + st * (STAGE / 16), d = tmem + (i & 1) * TILE;
      if (leader) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)  // 16 dims each: 4 in a 64-dim chunk, 8 columns of Q
          mma_step(d, tmem + kTmemQ + x * 8, k_at + (x >> 2) * (1024 / 16) + (x & 3) * 2, idesc_s, x > 0);
        tc_commit(&s.empty[0][st]);
        tc_commit(&s.s_full[i & 1]);
      }
      ++ns;
      return true;
    };
    // O of tile i, for the rows of its piece alone: the others' stay as they are, whatever the tile holds.
    uint32_t off[4];
    auto output = [&](int i, bool fresh) {
      const int st = i & 1, b = i & 1;
      if (!wait_for(s, &s.full[1][st], (i >> 1) & 1, a.err)) return false;
      if (!wait_for(s, &s.p_full[b], (i >> 1) & 1, a.err)) return false;
      tc_fence_after();
      const uint32_t v_at = v_lo + st * (STAGE / 16), p_at = tmem + b * TILE;
      if (leader) {
#pragma unroll
        for (int k = 0; k < TPAGES; ++k)  // a page each: 16 keys
          mma_step_rows(tmem + kTmemO, p_at + k * 8, v_at + k * (BLOCK / 16), idesc_o, off, !fresh || k > 0);
#pragma unroll
        for (int k = 0; k < TPAGES; ++k)  // what the rounding of P to bf16 left
          mma_step_rows(tmem + kTmemO, p_at + 32 + k * 8, v_at + k * (BLOCK / 16), idesc_o, off, true);
        tc_commit(&s.empty[1][st]);
        tc_commit(&s.o_full[b]);
      }
      ++no;
      return true;
    };
    int i = 0, nq = 1;
    bool more = __all_sync(0xffffffff, next_fragment(f));
    bool ok = more && __all_sync(0xffffffff, wait_for(s, &s.q_full, 0, a.err) && scores(0));
    while (ok && more) {
      const int t0 = f.t0, t1 = f.t1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int lo = min(max(f.s0 - 32 * j, 0), 32), hi = min(max(f.s1 - 32 * j, 0), 32);
        off[j] = ~((uint32_t)((1ull << hi) - 1) & ~(uint32_t)((1ull << lo) - 1));
      }
      for (int t = t0; ok && t < t1; ++t, ++i) {
        // S of the next tile, which may be the next unit's first, goes before O of this one.
        bool next = t + 1 < t1;
        if (!next) {
          next = more = __all_sync(0xffffffff, next_fragment(f));
          if (more) ok = wait_for(s, &s.q_full, nq++ & 1, a.err);
        }
        ok = ok && (!next || scores(i + 1)) && output(i, t == t0);
        ok = __all_sync(0xffffffff, ok);
      }
    }
    // The issued products end before TMEM is released.
    if (ns > 0) mbar_wait(&s.s_full[(ns - 1) & 1], ((ns - 1) >> 1) & 1, nullptr);
    if (no > 0) mbar_wait(&s.o_full[(no - 1) & 1], ((no - 1) >> 1) & 1, nullptr);
    __syncwarp();
  } else if (warp == 10) {
    // ----------------------------------------------------------------- lookup
    // The pieces ahead, their slots' lengths, and their queries to shared memory.
    const Work w = work_of(a);
    const int4 mine = __ldg(w.cta + cta);
    Walk walk{mine.x, mine.y, mine.z, max(1, __ldg(w.head)), group, -1, -1};
    const char* qbase = static_cast<const char*>(a.q);
    bool ok = true, more = true;
    int row[4], len[4], head[4], parts = 0;  // pieces whose Q was asked for
#pragma unroll
    for (int j = 0; j < 4; ++j) head[j] = (j * 32 + lane) % group;
    for (int at = 0, ph = 0; ok && more;) {
      more = walk.next(a, w, f);
      if (!more) f.t1 = 0;
      ok = __all_sync(0xffffffff, wait_for(s, &s.f_empty[at], ph ^ 1, a.err));  // passes at once in the first round
      if (lane == 0) {
        s.frag[at] = f;
        mbar_arrive(&s.f_full[at]);
      }
      if (!more || !ok) break;
      if (f.first) {
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = j * 32 + lane < f.slots ? a.seg_rows[f.e0 + (j * 32 + lane) / group] : -1;
      }
      // Queries of two pieces of a unit may be on their way (their slots differ); those of the next
      // unit wait until all of the last one's have left.
      if (parts >= 2) ok = wait_for(s, &s.way_empty[parts & 1], ((parts >> 1) - 1) & 1, a.err);
      if (f.first && parts >= 1) ok = ok && wait_for(s, &s.way_empty[(parts - 1) & 1], ((parts - 1) >> 1) & 1, a.err);
      ok = __all_sync(0xffffffff, ok);
      if (!ok) break;
      // The queries of the piece's slots (the softmax warps fetch the first piece's themselves), then
      // the lengths of its rows.
      // (Not bulk copies: those would wait behind the tiles that the copy warps asked for.)
#pragma unroll
      for (int j = 0; j < 4 && parts > 0; ++j) {
        const int index = row[j] * a.num_q_heads + f.kvh * group + head[j];
        const int lo = max(f.s0, j * 32), hi = min(f.s1, j * 32 + 32);
#pragma unroll 8
        for (int x = lo; x < hi; ++x)
          cp_async16(s.way[x] + lane * 16, qbase + (size_t)__shfl_sync(0xffffffff, index, x & 31) * (D * 2) + lane * 16);
      }
      cp_async_arrive(&s.way_full[parts & 1]);
      ++parts;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int sl = j * 32 + lane;
        len[j] = sl >= f.s0 && sl < f.s1 ? max(a.seq_lens[row[j]], 0) : 0;
      }
      int least = 0x7FFFFFFF;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int sl = j * 32 + lane;
        const bool in = sl >= f.s0 && sl < f.s1;
        s.limit[at][sl] = in ? min(len[j], f.len) : 0;
        if (in) least = min(least, min(len[j], f.len));
      }
      least = __reduce_min_sync(0xffffffff, least);
      if (lane == 0) s.least[at] = least;
      mbar_arrive(&s.r_full[at]);
      if (++at == AHEAD) {
        at = 0;
        ph ^= 1;
      }
    }
    cp_async_wait();
  } else {
    // ---------------------------------------------------------------- softmax
    const int half = warp >> 2, slot = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);  // this warp's quarter of TMEM
    const float qscale = a.sm_scale * 1.4426950408889634f;             // exp2 domain
    const int head = slot % group;
    auto way = [&](int r, int p) { return s.way[r] + ((half * 16 + p) << 4); };  // 16-byte piece p of the warp's half
    // The first piece's Q: every warp fetches what it will store, two slots' halves at a time, in a
    // quarter of the time that one warp takes for 128 slots while tiles arrive (4.1 us).
    auto fetch_q = [&](const Fragment& g) {
      const int index = (slot >= g.s0 && slot < g.s1 ? a.seg_rows[g.e0 + slot / group] : 0) * a.num_q_heads + g.kvh * group + head;
#pragma unroll
      for (int x = 0; x < 32; x += 2) {
        const int at = x + (lane >> 4), from = __shfl_sync(0xffffffff, index, at), to = (warp & 3) * 32 + at, c = half * 256 + (lane & 15) * 16;
        if (to >= g.s0 && to < g.s1) cp_async16(s.way[to] + c, static_cast<const char*>(a.q) + (size_t)from * (D * 2) + c);
      }
      cp_async_wait();
      __syncwarp();
    };
    auto store_q = [&](const Fragment& g, int k) {  // Q of piece k from the way to TMEM
      wait_for(s, &s.way_full[k & 1], (k >> 1) & 1, a.err);
      if ((warp & 3) * 32 < g.s1 && (warp & 3) * 32 + 32 > g.s0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t r[16];
#pragma unroll
          for (int x = 0; x < 4; ++x) *reinterpret_cast<uint4*>(r + 4 * x) = *reinterpret_cast<const uint4*>(way(slot, 4 * j + x));
          tmem_st_32x32b_x16(lanes + kTmemQ + half * 64 + j * 16, r);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      mbar_arrive(&s.q_full);
      mbar_arrive(&s.way_empty[k & 1]);
    };
    // After a wait that gave up these warps go on to the end of the fragment with whatever is there (the
    // error word is set, every later wait gives up at once) and leave together: their barriers always meet.
    // Before the plan is there, one tile is computed from whatever TMEM holds and nothing is kept of
    // it: the first real tile then finds its instructions in the cache (from its S to its P 1.3 us instead of 3.4).  A call of
    // four rows behind other work takes 25 us instead of 29, one that repeats 16.3 instead of 16.7; eight
    // prompts repeated 39.8 instead of 39.1.
    int dry;
    asm volatile("mov.u32 %0, 1;" : "=r"(dry));
    f = Fragment{0, 0, SLOTS, 0, SLOTS, 0, 1, 0, TPAGES, TILE, 0, 1};
    bool more = true;
    int kf = 0;  // place of the piece
    uint32_t kph = 0;
    int i = 0, parts = 1;
    float m = -INFINITY, l = 0.f;  // reference maximum (raw scores) of the slot, sum of this half's weights
    int rec = -1;                  // record of the slot, once it had a tile
    while (more) {
      if (!dry) wait_for(s, &s.r_full[kf], kph, a.err);
      const int limit = dry ? TILE : s.limit[kf][slot], least = dry ? TILE : s.least[kf];
      const bool used = slot >= f.s0 && slot < f.s1, busy = (warp & 3) * 32 < f.s1 && (warp & 3) * 32 + 32 > f.s0;
      if (used) {
        // The CTA with a piece's first tile keeps the record by (entry, head), the others by CTA and slot.
        rec = dry       ? -1
              : f.t0 == 0 ? (f.e0 + slot / group) * a.num_q_heads + f.kvh * group + head
                        : a.entries * a.num_q_heads + cta * SLOTS + slot;
        m = -INFINITY;
        l = 0.f;
      }
      Fragment g = {};
      for (int t = f.t0; t < f.t1; ++t, ++i) {
        const int b = i & 1, key0 = (f.p0 + t * TPAGES) * PAGE;
        if (!dry) wait_for(s, &s.s_full[b], (i >> 1) & 1, a.err);
        tc_fence_after();
        if (t + 1 == f.t1 && !dry) {
          more = !compute_any(!next_fragment(g));
          if (more) store_q(g, parts++);  // every product with this Q is done: the next takes its place
        }
        uint32_t r[32];
        float mt = -INFINITY;
        const int valid = limit - key0 - half * 32;
        if (busy) {
          tmem_ld_32x32b_x32(lanes + b * TILE + half * 32, r);
          tmem_ld_wait();
          if (valid < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j >= valid) r[j] = 0xFF800000u;  // -inf
          }
          float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j & 3] = fmaxf(x[j & 3], __uint_as_float(r[j]));
          mt = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          s.top[b][half][slot] = mt;
        }
        compute_sync();  // both halves' maxima are there, and S is read: P takes its place
        float fac = 1.f;
        bool grow = false;
        if (busy) {
          // The reference follows the maximum when that outgrew it (and at first); both halves agree.
          mt = fmaxf(mt, s.top[b][half ^ 1][slot]);
          grow = used && (m == -INFINITY ? mt > -INFINITY : (mt - m) * qscale > kGrow);
          if (grow) {
            fac = m == -INFINITY ? 0.f : ex2((m - mt) * qscale);
            l *= fac;
            m = mt;
          }
        }
        if (__any_sync(0xffffffff, grow) && t > f.t0) {
          wait_for(s, &s.o_full[(i - 1) & 1], ((i - 1) >> 1) & 1, a.err);  // O holds every tile before this one
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            uint32_t o[16];
            const uint32_t at = lanes + kTmemO + half * 128 + c;
            tmem_ld_32x32b_x16(at, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * fac);
            tmem_st_32x32b_x16(at, o);
          }
        }
        if (busy) {
          const float off = m == -INFINITY ? 0.f : m * qscale;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t pk[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float lo = ex2(fmaf(__uint_as_float(r[2 * j]), qscale, -off));
            const float hi = ex2(fmaf(__uint_as_float(r[2 * j + 1]), qscale, -off));
            sum[j & 3] += lo + hi;
            pk[j] = pack_bf16_down(lo, hi);
            r[2 * j] = __float_as_uint(lo);
            r[2 * j + 1] = __float_as_uint(hi);
          }
          tmem_st_32x32b_x16(lanes + b * TILE + half * 16, pk);
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
          for (int j = 0; j < 16; ++j)  // above 0 by the smallest step at least: an infinite value times 0 would be NaN
            pk[j] = pack_bf16(__uint_as_float(r[2 * j]) - __uint_as_float(pk[j] << 16),
                              __uint_as_float(r[2 * j + 1]) - __uint_as_float(pk[j] & 0xFFFF0000u)) | 0x00010001u;
          tmem_st_32x32b_x16(lanes + b * TILE + 32 + half * 16, pk);
          tmem_st_wait();
        }
        // Values that a row does not see must not meet its zero weights as NaN or infinity.  Rows
        // of the tile that nobody sees are zeroed.  Rows that only some see are looked at: those
        // with such a value are zeroed too, and added by hand to the slots that see them.
        const int end = f.len - key0;  // keys of the tile that some row sees
        unsigned long long odd = 0;
        if (end < TILE || least < key0 + TILE) {
          uint8_t* const vt = s.ring[1][b];
          wait_for(s, &s.full[1][b], (i >> 1) & 1, a.err);
          const int from = max(0, min(least - key0, TILE)), stop = min(end, TILE);
          bool found = false;
          for (int x = from * 32 + tid; x < stop * 32; x += COMPUTE) {
            const uint4 v = *reinterpret_cast<const uint4*>(vt + tile_offset(x >> 5, x & 31));
            found |= not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w);
          }
          if (from < stop && compute_any(found)) {
            for (int k = from; k < stop; ++k) {  // 512 bytes a key: 4 for each of 128 threads
              uint32_t* at = reinterpret_cast<uint32_t*>(vt + tile_offset(k, (tid & 127) >> 2)) + (tid & 3);
              if (compute_any(not_finite(*at))) {
                odd |= 1ull << k;
                *at = 0;
              }
            }
          }
          for (int x = max(end, 0) * 32 + tid; x < TILE * 32; x += COMPUTE)
            *reinterpret_cast<uint4*>(vt + tile_offset(x >> 5, x & 31)) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_shared();
        }
        tc_fence_before();
        if (!dry) mbar_arrive(&s.p_full[b]);
        if (odd != 0) {
          wait_for(s, &s.o_full[b], (i >> 1) & 1, a.err);
          tc_fence_after();
          for (int k = 0; k < TILE; ++k) {
            if (!(odd >> k & 1)) continue;
            compute_sync();
            if (busy && (k >> 5) == half) {
              float p = 0.f;
#pragma unroll
              for (int j = 0; j < 32; ++j) p = pick(j == (k & 31), __uint_as_float(r[j]), p);
              s.top[b][0][slot] = p;
            }
            compute_sync();
            const int at_page = (key0 + k) / PAGE, page = at_page < a.max_pages ? a.page_table[(size_t)f.table * a.max_pages + at_page] : -1;
            if (!busy || page < 0 || page >= a.num_pages) continue;
            const uint8_t* blk = static_cast<const uint8_t*>(a.v_cache) + ((size_t)page * a.num_kv_heads + f.kvh) * BLOCK;
            const float p = s.top[b][0][slot];
            for (int c = 0; c < 128; c += 16) {
              uint32_t o[16];
              const uint32_t at = lanes + kTmemO + half * 128 + c;
              tmem_ld_32x32b_x16(at, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const int d = half * 128 + c + j;
                const float v = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(blk + tile_offset(k & 15, d >> 3) + (d & 7) * 2));
                if (p != 0.f) o[j] = __float_as_uint(__uint_as_float(o[j]) + p * v);
              }
              tmem_st_32x32b_x16(at, o);
              tmem_st_wait();
            }
          }
          tc_fence_before();
        }
      }
      if (!more || g.first || dry) {
        // ---- the unit's records, through shared memory so that the stores are whole lines.
        if (!dry) wait_for(s, &s.o_full[(i - 1) & 1], ((i - 1) >> 1) & 1, a.err);
        tc_fence_after();
        const uint32_t has = __ballot_sync(0xffffffff, rec >= 0);
        float* to = a.partial + (size_t)max(rec, 0) * PREC;
        if (has != 0 || dry) {
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(lanes + kTmemO + half * 128 + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
              for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<uint4*>(&s.stage[warp][lane][j]) =
                    make_uint4(o[q * 16 + j], o[q * 16 + j + 1], o[q * 16 + j + 2], o[q * 16 + j + 3]);
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 4; ++j) {  // 8 rows of 64 bytes an instruction
                const int x = 8 * j + (lane >> 2), rx = __shfl_sync(0xffffffff, rec, x);
                if (rx >= 0)
                  *reinterpret_cast<uint4*>(a.partial + (size_t)rx * PREC + half * 128 + c + q * 16 + (lane & 3) * 4) =
                      *reinterpret_cast<const uint4*>(&s.stage[warp][x][(lane & 3) * 4]);
              }
              __syncwarp();
            }
          }
        }
        if (rec >= 0) {
          if (half == 0) *reinterpret_cast<float2*>(to + D) = make_float2(m * qscale, l);
          else to[D + 2] = l;
        }
        rec = -1;
        tc_fence_before();
      }
      __syncwarp();
      if (dry) {
        pdl_wait();
        pdl_trigger();
        dry = i = 0;
        m = -INFINITY;
        l = 0.f;
        more = !compute_any(!next_fragment(f));
        if (more) {
          fetch_q(f);
          store_q(f, 0);
        }
        continue;
      }
      if (lane == 0) mbar_arrive(&s.f_empty[kf]);
      if (++kf == AHEAD) {
        kf = 0;
        kph ^= 1;
      }
      f = g;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, kTmemCols);
}

constexpr int MERGE_WARPS = 8, AT_ONCE = 2;
// The join of a (row, q head) pair's records, read once from L2 (4.2 us for 1824 pairs' 20 MB after
// the tiles' end; latencies bound it).  A lane owns dims 4 lane .. + 3 and 128 + 4 lane .. + 3.  Records
// are found and weighed 32 at a time (one a lane), then added in order, AT_ONCE on their way together;
// with PARTS warps on a pair, warp p takes every PARTS-th record and the parts are joined in order.
// 64 registers, so that four CTAs share an SM, are worth more than more loads in flight (1824 pairs:
// 40.5 us the whole call with 2, 40.9 with 3; with 4 and 80 registers 45.4).
template <int PARTS>
__global__ void __launch_bounds__(MERGE_WARPS * 32, 4) merge_kernel(const SharedAttnArgs a) {
  const Work w = work_of(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % PARTS;
  const int at_item = blockIdx.x * (MERGE_WARPS / PARTS) + warp / PARTS, item = min(at_item, a.rows * a.num_q_heads - 1);
  const int row = item / a.num_q_heads, h = item % a.num_q_heads, group = group_of(a);
  float m = -INFINITY, l = 0.f, o[8] = {};
  uint2 gate[2] = {};
  for (int j0 = 0; j0 < a.levels; j0 += 32) {
    // A lane per segment of the row: where its records are.  before = records of the segments before.
    const int e = j0 + lane < a.levels ? __ldg(a.row_entry + row * a.levels + j0 + lane) : -1;
    int c0 = 0, cnt = 0, slot = 0;
    if (e >= 0) {
      const int4 u = __ldcg(w.entry + (size_t)e * a.num_kv_heads + h / group);
      c0 = u.x;
      cnt = u.y;
      slot = u.z + h % group;
    }
    int before = cnt;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const int y = __shfl_up_sync(0xffffffff, before, x);
      if (lane >= x) before += y;
    }
    const int records = __shfl_sync(0xffffffff, before, 31);
    before -= cnt;
    // Where record r is, counted over this group of segments.
    auto place = [&](int r) {
      int j = 0;  // its segment: the last with before <= r and records
      for (int x = 1; x < 32; ++x) {
        const int bx = __shfl_sync(0xffffffff, before, x), cx = __shfl_sync(0xffffffff, cnt, x);
        if (cx > 0 && bx <= r) j = x;
        if (j0 + x + 1 >= a.levels) break;
      }
      const int c = __shfl_sync(0xffffffff, c0, j) + r - __shfl_sync(0xffffffff, before, j);
      const int sl = __shfl_sync(0xffffffff, slot, j), ej = __shfl_sync(0xffffffff, e, j);
      return r == __shfl_sync(0xffffffff, before, j) ? ej * a.num_q_heads + h
                                                    : a.entries * a.num_q_heads + c * SLOTS + sl;
    };
    int at = place(part + lane * PARTS);  // this lane's record
    if (j0 == 0) {
      // What came so far is from kernels that had ended when the tiles began (their CTAs let this
      // kernel start after their own wait); the records are not.
      if (a.gate != nullptr) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          gate[k] = __ldcg(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.gate) + (size_t)item * D + k * 128 + lane * 4));
      }
      pdl_wait();
      pdl_trigger();
    }
    for (int r0 = part; r0 < records; r0 += 32 * PARTS) {
      const int r = r0 + lane * PARTS;
      if (r0 > part) at = place(r);
      const float4 ml = r < records ? *reinterpret_cast<const float4*>(a.partial + (size_t)at * PREC + D) : make_float4(-INFINITY, 0.f, 0.f, 0.f);
      const int here = min(32, (records - r0 + PARTS - 1) / PARTS);
      float4 p[AT_ONCE], q[AT_ONCE];  // the first records, on their way together with the weights
      auto load = [&](int x0) {
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
          const float4* from = reinterpret_cast<const float4*>(a.partial + (size_t)__shfl_sync(0xffffffff, at, x0 + x) * PREC);
          if (x0 + x < here) p[x] = from[lane], q[x] = from[32 + lane];
        }
      };
      load(0);
      const float mn = fmaxf(m, warp_max(ml.x)), s0 = m == -INFINITY ? 0.f : exp2f(m - mn);
      const float wt = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
      l = l * s0 + warp_sum(wt * (ml.y + ml.z));  // a sum without a maximum is 0, or NaN where every score was
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] *= s0;
      m = mn;
      for (int x0 = 0; x0 < here; x0 += AT_ONCE) {
        if (x0 > 0) load(x0);
#pragma unroll
        for (int x = 0; x < AT_ONCE; ++x) {
          const float wx = __shfl_sync(0xffffffff, wt, x0 + x);
          if (x0 + x >= here || wx == 0.f) continue;
          o[0] += wx * p[x].x;
          o[1] += wx * p[x].y;
          o[2] += wx * p[x].z;
          o[3] += wx * p[x].w;
          o[4] += wx * q[x].x;
          o[5] += wx * q[x].y;
          o[6] += wx * q[x].z;
          o[7] += wx * q[x].w;
        }
      }
    }
  }
  if (PARTS > 1) {
    __shared__ float all[MERGE_WARPS][D + 2];
    float(*parts)[D + 2] = all + warp / PARTS * PARTS;
#pragma unroll
    for (int k = 0; k < 8; ++k) parts[part][(k >> 2) * 128 + lane * 4 + (k & 3)] = o[k];
    if (lane == 0) {
      parts[part][D] = m;
      parts[part][D + 1] = l;
    }
    __syncthreads();
    if (part != 0) return;
    const float mp = lane < PARTS ? parts[lane][D] : -INFINITY;
    m = warp_max(mp);
    const float wp = mp == -INFINITY ? 0.f : exp2f(mp - m);
    l = warp_sum(lane < PARTS ? wp * parts[lane][D + 1] : 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
    for (int x = 0; x < PARTS; ++x) {
      const float wx = __shfl_sync(0xffffffff, wp, x);
      if (wx == 0.f) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] += wx * parts[x][(k >> 2) * 128 + lane * 4 + (k & 3)];
    }
  }
  if (at_item != item) return;
  // A row without keys gives 0.  Any other whose sum is 0 or NaN (its scores all -inf, or one NaN) gives NaN.
  const bool empty = a.seq_lens[row] <= 0;
  const float inv = 1.f / l;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = k * 128 + lane * 4;
    float* y = o + 4 * k;
    float g[4] = {1.f, 1.f, 1.f, 1.f};
    if (a.gate != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) g[j] = sigmoidf_(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&gate[k])[j]));
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = empty ? 0.f : y[j] * inv * g[j];
    if (a.out_bf16 != nullptr)
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out_bf16) + (size_t)item * D + d) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
    if (a.out_q != nullptr) {  // a block of 32 dims is 8 lanes
      float amax = fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])));
#pragma unroll
      for (int x = 1; x < 8; x <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffff, amax, x));
      const uint8_t code = mx_scale_e8m0(amax);
      const float si = mx_inv_scale(code);
      uint32_t four = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) four |= (uint32_t)f32_to_e4m3(y[j] * si) << (8 * j);
      *reinterpret_cast<uint32_t*>(a.out_q + (size_t)item * D + d) = four;
      if ((lane & 7) == 0) {
        const int kb = h * (D / 32) + (d >> 5);
        a.out_sf[((size_t)(row >> 7) * (a.num_q_heads * D >> 7) + (kb >> 2)) * 512 + sf_atom_offset(row & 127, kb & 3)] = code;
      }
    }
  }
}

int check(const SharedAttnArgs& a) {
  if (a.num_kv_heads < 1 || a.num_q_heads % a.num_kv_heads != 0 || a.num_q_heads / a.num_kv_heads > ZS_SHARED_MAX_GROUP) return -1;
  if (a.head_dim != D || a.page_size != PAGE || a.levels < 1 || a.num_segs < 0 || a.num_segs > MAX_SEGS || a.rows < 0) return -1;
  if (a.num_pieces < 0 || a.num_pieces > MAX_PIECES) return -1;
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
  using namespace zs::sattn;
  cudaFuncSetAttribute(tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  zs_launch(tiles_kernel, CTAS, THREADS, SMEM, stream, a);
  const int items = a.rows * a.num_q_heads;
  // Warps that share the records of a (row, q head) pair: with few pairs a long prefix leaves a record
  // in every CTA, with many there are a few each and the device is full without.  The whole call in us
  // with 1, 2, 4 and 8: 64 pairs 21.7, 18.8, 17.0, 16.2; 768 pairs 61.6, 55.6, 52.4, 56.7; 1824 pairs
  // 39.6, 39.7, 43.6, 49.4; 7296 pairs 57.1, 65.3, 75.3, 96.5.
  int parts = MERGE_WARPS;
  while (parts > 1 && (long long)items * parts > 4096) parts /= 2;
  const auto merge = parts == 8 ? merge_kernel<8> : parts == 4 ? merge_kernel<4> : parts == 2 ? merge_kernel<2> : merge_kernel<1>;
  zs_launch(merge, (int)(((long long)items * parts + MERGE_WARPS - 1) / MERGE_WARPS), MERGE_WARPS * 32, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
