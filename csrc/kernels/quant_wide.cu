// Attention over the quantised K/V cache for sequences with many query slots (slot = row x head of a
// kv head's group): the rows of a verify step, chunks of prompts, wide groups.
//
// A unit is up to 128 slots of one sequence and kv head; a CTA (one an SM) takes its share of all units'
// 64-key tiles as in quant_cache.cu, and its records are joined there.  S = Q K^T (M = 128 slots, N = 64
// keys) and O += P V (N = the dims) run on tcgen05 with Q and P in TMEM, so that a tile is turned into f16
// once for all slots and shared memory is read once for it:
//  * copy warp: page ids, then one bulk copy per 16-token block into a ring of tiles;
//  * 14 converter warps, each at a block, its K and then its V: s n + z as one f16 fused multiply-add of two
//    numbers, rounded once (by up to 2^-11 of a value, an eighth of what a bf16 output is).  (w & 0x000F000F) is two
//    subnormals n 2^-24 and the factor s 2^24, so a pair costs an integer instruction, a part of a shift and the
//    multiply-add.  A power of two per token (its unit) brings its largest scale to [2^-9, 2^-8), which keeps s 2^24 and
//    every value in f16's range whatever their size (an offset is below 2^19 of its group's scale), and no token's
//    precision depends on another; K's unit goes to the token's scores and V's to its weights, in 32 bits.  V's numbers of 4 bits
//    are all taken times 16 and its scales brought to [2^-5, 2^-4), so that a group 2^12 smaller than the token's largest still has
//    a step of 2^7 times f16's smallest (two shifts more for four tokens' numbers: verify requests 112 -> 113 us).  K goes to a
//    swizzled image of keys x dims, V to one of dims x keys (as it is stored), both K-major operands;
//  * MMA warp: S of the next tile goes before O of this one;
//  * 16 softmax warps: a thread has a block of a tile for a slot.  The weights 2^(x - reference) are held
//    below 2^14 with the token's unit of V, as f16 (2^-11); the reference follows the largest score only when that
//    outgrew it by 2^8, and O in TMEM is rescaled then.
// f16 outputs, which all this would cost bits, are left to quant_cache.cu.
// A poisoned group of V (NaN) is 0 in the image; the slots that see its key note it, and their dims of the
// group become NaN in the record.  So nothing of a masked key reaches a slot: its bits are the same whatever stands there.
//
// Measured (us, 16 q heads, 2 kv heads of 256 dims, 4 bits): 128 sequences of up to 2300 keys with 4 rows 108, three
// chunks of up to 700 rows that see up to 4500 keys 211 (0.52 PFLOP/s of products).  A tile takes some 3000
// cycles with 256 dims and 1900 with 64, of which the products are 1000 and 260.  No unit is full with 256 dims (issue slots 46 %,
// tensor pipe 33 %, DRAM 18 %): a tile goes through converters, products, softmax and products again, two at a time.  The four
// softmax warps of the same 32 slots are on one scheduler, which has all of a verify step's.  With 64 dims it is the softmax's
// chain: scores 360 cycles, agreement of the four warps 190, weights 840 (64 exponentials of four warps), handing over 150.  Tried and slower or no faster: tiles taken in turn by two sets of softmax
// warps, blocks given to whichever converter is free, one barrier of all softmax warps, more registers for fewer
// converters, unrolled conversion loops (they leave the instruction cache: 224 -> 296 us).
#include "quant_cache.cuh"

namespace zs {
namespace qc {
namespace {

constexpr int SOFT = 512, CONV = 448;               // threads; then the MMA and the copy warp
constexpr int THREADS = SOFT + CONV + 64;
constexpr int MMA_WARP = (SOFT + CONV) / 32, COPY_WARP = MMA_WARP + 1;
constexpr int TBLOCKS = WIDE_KEYS / TOK;   // blocks of a tile
constexpr uint32_t TMEM_Q = 128, TMEM_O = 256, TMEM_COLS = 512;   // two S of 64 columns, Q as pairs, O
constexpr int MAX_RAW = 4;
// Tiles whose units are kept.  The raw blocks of tile i come into the place of tile i - MAX_RAW's at the earliest, whose V was
// converted once O of tile i - MAX_RAW - 2 was done: no unit is overwritten that a softmax still needs.
constexpr int UNITS = MAX_RAW + 2;

// What a unit of K is held as: a unit is at most 2^132, and scores of the largest K and q still stay below 2^116.
constexpr int K_SMALL_LOG = -33;

struct Smem {
  uint64_t raw_full[4], raw_empty[MAX_RAW];
  uint64_t k_full[2], v_full[2], k_empty[4], v_empty[4], s_full[2], p_full[2], o_full[2], q_full;
  uint32_t tmem;
  int abort;
  alignas(16) float k_unit[UNITS][WIDE_KEYS];   // a token's unit of K, times 2^K_SMALL_LOG
  float v_log[UNITS][WIDE_KEYS];         // log2 of a token's unit of V
  float v_inv[UNITS][WIDE_KEYS];         // 2^ABOVE over the same unit
  uint32_t v_bad[UNITS][TBLOCKS][2];     // poisoned (token, group) pairs: pair x is bit x / n of word x % n (n words are used)
  alignas(16) uint32_t pairs[CONV / 32][2][TOK * 4];   // of a converter's block, K and V: per group and token, scale and offset in f16
  float top[TBLOCKS][WIDE_SLOTS];
  uint4 stage[SOFT / 32][32][2];     // 8 columns of a warp's 32 slots, on their way to the record
};

template <int D_, int BITS_>
struct Wide {
  static constexpr int D = D_, BITS = BITS_, NG = D / GROUP;
  static constexpr int CODES = code_bytes(D, BITS), BLOCK = block_bytes(D, BITS);
  static constexpr int K_IMAGE = WIDE_KEYS * D * 2, V_IMAGE = D * WIDE_KEYS * 2;
  static constexpr int IMAGES = 2 * (K_IMAGE + V_IMAGE);
  static constexpr int RAW = TBLOCKS * BLOCK;
  static constexpr int RING = (227 * 1024 - IMAGES - (int)sizeof(Smem) - 1024) / RAW < MAX_RAW
                                  ? (227 * 1024 - IMAGES - (int)sizeof(Smem) - 1024) / RAW : MAX_RAW;
  static constexpr int BYTES = IMAGES + RING * RAW + (int)sizeof(Smem);
  static_assert(RING >= 2, "");
};

struct Piece {
  int chunk, head, first, n;   // tiles [first, first + n) of the unit
  int row, slot, slot0, count, len;
};

// A wait that gave up makes all later ones that would wait give up at once.
__device__ __forceinline__ bool wait_for(Smem& s, uint64_t* bar, uint32_t phase, int* err) {
  if (mbar_try_wait(bar, phase)) return true;
  for (uint32_t i = 0; i < kMbarSpinLimit; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (*reinterpret_cast<volatile int*>(&s.abort)) return false;
    if (i > 64) __nanosleep(64);
  }
  report_error(err, kErrMbarTimeout);
  *reinterpret_cast<volatile int*>(&s.abort) = 1;
  return false;
}
// Of the four warps that have the same slots.
__device__ __forceinline__ void slots_sync(int quarter) { asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory"); }
__device__ __forceinline__ bool slots_any(int quarter, bool x) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, 128, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((int)x), "r"(1 + quarter)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ float2 fma_two(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul_two(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add_two(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t sixteenth(uint32_t a) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0x2C002C00u));
  return d;
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld_x8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
__device__ __forceinline__ uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

// A in TMEM, B K-major with a 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ void mma_step(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((int)add), "n"((1024 >> 4) | (1 << 14) | (2 << 29))
      : "memory");
}
__device__ __forceinline__ uint32_t desc_lo(const void* p) { return (smem_u32(p) >> 4) | ((16 >> 4) << 16); }
constexpr uint32_t idesc_f16(uint32_t m, uint32_t n) { return 1u << 4 | (n >> 3) << 17 | (m >> 4) << 24; }


template <class W>
__global__ void __launch_bounds__(THREADS, 1) wide_kernel(const QuantAttnArgs a) {
  constexpr int D = W::D, BITS = W::BITS, NG = W::NG, BLOCK = W::BLOCK, RING = W::RING;
  extern __shared__ __align__(1024) uint8_t raw_smem[];
  uint8_t* k_image = raw_smem;
  uint8_t* v_image = raw_smem + 2 * W::K_IMAGE;
  uint8_t* ring = raw_smem + W::IMAGES;
  Smem& s = *reinterpret_cast<Smem*>(ring + RING * W::RAW);
  if ((smem_u32(raw_smem) & 1023) != 0) {   // the swizzled images need it
    report_error(a.err, kErrBadShape);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == MMA_WARP) {
    tmem_alloc(&s.tmem, TMEM_COLS);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < RING; ++i) mbar_init(&s.raw_empty[i], TBLOCKS);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s.k_full[i], TBLOCKS);
      mbar_init(&s.v_full[i], TBLOCKS);
      mbar_init(&s.s_full[i], 1);
      mbar_init(&s.p_full[i], SOFT / 32);
      mbar_init(&s.o_full[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s.raw_full[i], 1);
      mbar_init(&s.k_empty[i], 1);
      mbar_init(&s.v_empty[i], 1);
    }
    mbar_init(&s.q_full, SOFT / 32);
    s.abort = 0;
    fence_barrier_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s.tmem;
  pdl_wait();
  pdl_trigger();
  const Plan plan = plan_of(a);
  const long long total = stages_of(plan, a);
  const int B = ctas_of(total, gridDim.x, a.least), cta = blockIdx.x;
  const bool work = cta < B && total > 0;
  const int group = a.num_q_heads / a.num_kv_heads;
  // Every role walks the CTA's pieces by itself.
  long long pos = work ? total * cta / B : 0;
  const long long hi = work ? total * (cta + 1) / B : 0;
  int chunk = work ? plan.start[cta] : 0;
  auto next_piece = [&](Piece& p) {
    if (pos >= hi) return false;
    Chunk e = plan.table[chunk];
    while (e.before + (long long)e.stages * a.num_kv_heads <= pos) e = plan.table[++chunk];
    const int r = (int)(pos - e.before);
    p.chunk = chunk;
    p.head = r / e.stages;
    p.first = r % e.stages;
    p.n = (int)min((long long)(e.stages - p.first), hi - pos);
    p.row = e.row;
    p.slot = e.slot;
    p.slot0 = e.first;
    p.count = e.count;
    p.len = e.len;
    pos += p.n;
    return true;
  };
  Piece p;

  if (warp == COPY_WARP) {
    // ------------------------------------------------------------------ copies
    const int bshift = a.page_shift - 4;
    int i = 0, st = 0;
    uint32_t phase = 1;   // of raw_empty: passes at once in the first round
    bool ok = true;
    while (ok && next_piece(p)) {
      const bool known = p.slot >= 0 && p.slot < a.num_slots;
      auto page_of = [&](int t) {   // -1: a place that does not exist; raw, so that nothing waits for it here
        const int blk = (p.first + t) * TBLOCKS + lane;
        if (lane >= TBLOCKS || t >= p.n || blk * TOK >= p.len) return 0;
        return known && (blk >> bshift) < a.max_pages ? a.page_table[(size_t)p.slot * a.max_pages + (blk >> bshift)] : -1;
      };
      int page = page_of(0);
      for (int t = 0; ok && t < p.n; ++t, ++i) {
        const int after = page_of(t + 1);
        const int blk = (p.first + t) * TBLOCKS + lane, count = min(TBLOCKS, (p.len + TOK - 1) / TOK - (p.first + t) * TBLOCKS);
        if (page < 0 || page >= a.num_pages) {
          report_error(a.err, kErrBadShape);
          page = 0;
        }
        ok = __all_sync(0xffffffff, wait_for(s, &s.raw_empty[st], phase, a.err));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(&s.raw_full[i & 3], count * BLOCK);
        __syncwarp();
        if (lane < count)
          bulk_load(ring + st * W::RAW + lane * BLOCK,
                    a.data + ((((size_t)page * a.num_kv_heads + p.head) << bshift) + (blk & ((1 << bshift) - 1))) * BLOCK, BLOCK, &s.raw_full[i & 3]);
        page = after;
        if (++st == RING) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    // Copies in flight land before the CTA gives its shared memory back.
    if (lane == 0)
      for (int m = max(0, i - RING); m < i; ++m) mbar_wait(&s.raw_full[m & 3], (m >> 2) & 1, nullptr);
  } else if (warp == MMA_WARP) {
    // -------------------------------------------------------------------- MMA
    const bool leader = elect_one();
    const uint32_t idesc_s = idesc_f16(WIDE_SLOTS, WIDE_KEYS), idesc_o = idesc_f16(WIDE_SLOTS, D);
    const uint32_t k_lo = desc_lo(k_image), v_lo = desc_lo(v_image);
    int ns = 0, no = 0, nq = 0;   // issued products, queries met
    auto scores = [&](int i) {
      const int b = i & 1;
      if (!wait_for(s, &s.k_full[b], (i >> 1) & 1, a.err)) return false;
      // It takes the place of the P two tiles before.
      if (i >= 2 && !wait_for(s, &s.o_full[b], ((i >> 1) - 1) & 1, a.err)) return false;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
          mma_step(tmem + b * 64, tmem + TMEM_Q + x * 8, k_lo + (b * W::K_IMAGE + (x >> 2) * WIDE_KEYS * 128) / 16 + (x & 3) * 2, idesc_s, x > 0);
        tc_commit(&s.k_empty[i & 3]);
        tc_commit(&s.s_full[b]);
      }
      ++ns;
      return true;
    };
    auto output = [&](int i, bool fresh) {
      const int b = i & 1;
      if (!wait_for(s, &s.v_full[b], (i >> 1) & 1, a.err)) return false;
      if (!wait_for(s, &s.p_full[b], (i >> 1) & 1, a.err)) return false;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int k = 0; k < WIDE_KEYS / 16; ++k)
          mma_step(tmem + TMEM_O, tmem + b * 64 + k * 16, v_lo + b * W::V_IMAGE / 16 + k * 2, idesc_o, !fresh || k > 0);
        tc_commit(&s.v_empty[i & 3]);
        tc_commit(&s.o_full[b]);
      }
      ++no;
      return true;
    };
    int i = 0;
    bool ok = true;
    while (ok && next_piece(p)) {
      ok = __all_sync(0xffffffff, wait_for(s, &s.q_full, nq++ & 1, a.err) && scores(i));
      for (int t = 0; ok && t < p.n; ++t, ++i) {
        // S of the piece's next tile goes before O of this one; the next piece's waits for its queries.
        const bool good = (t + 1 >= p.n || scores(i + 1)) && output(i, t == 0);
        ok = __all_sync(0xffffffff, good);
      }
    }
    // The issued products end before TMEM is released.
    if (ns > 0) mbar_wait(&s.s_full[(ns - 1) & 1], ((ns - 1) >> 1) & 1, nullptr);
    if (no > 0) mbar_wait(&s.o_full[(no - 1) & 1], ((no - 1) >> 1) & 1, nullptr);
    __syncwarp();
  } else if (warp >= SOFT / 32) {
    // -------------------------------------------------------------- converters
    // The warps take the blocks of the tiles in turn, K and then V of each.
    const int w = warp - SOFT / 32, g = lane >> 2, t4 = lane & 3;
    constexpr int PAIRS = (TOK * NG + 31) / 32;
    int at = w, before = 0;   // the next block, counted over the CTA's tiles; tiles of the pieces before
    bool ok = true;
    while (ok && next_piece(p)) {
      for (; ok && at / TBLOCKS < before + p.n; at += CONV / 32) {
        const int i = at / TBLOCKS, b = i & 1, kb = at & (TBLOCKS - 1);
        const int st = i % RING, left = p.len - (p.first + i - before) * WIDE_KEYS - kb * TOK;   // keys of the block from here on
        const uint8_t* in = ring + st * W::RAW + kb * BLOCK;
        ok = __all_sync(0xffffffff, wait_for(s, &s.raw_full[i & 3], (i >> 2) & 1, a.err));
        if (!ok) break;
        // The tokens' units from their scales and offsets (a lane has one or two of the 16 NG pairs, two lanes a token where
        // there are more than one), and those as multiples of it: s 2^24 and z.  What is behind the sequence is 0 in V, as
        // poisoned groups are.  The softmax reads the units once S is there, which no K is missing from.
#pragma unroll 1
        for (int is_v = 0; is_v < 2; ++is_v) {
          // Bits below which the largest scale comes, and what its numbers are f16 subnormals of.
          const int below = BITS == 4 && is_v ? 4 : 8;
          const float number = BITS == 4 && is_v ? 0x1p20f : 0x1p24f, most_z = BITS == 4 && is_v ? 0x1p-18f : 0x1p-22f;
          const uint32_t* sz = reinterpret_cast<const uint32_t*>(in + 2 * W::CODES) + is_v * TOK * NG;
          float sf[PAIRS], zf[PAIRS], top = 0.f;
          uint32_t bad[PAIRS];
#pragma unroll
          for (int c = 0; c < PAIRS; ++c) {
            const int x = lane * PAIRS + c, token = x / NG;
            const uint32_t u = x < TOK * NG ? sz[x] : 0;
            const bool nan = (u & 0x7FFFu) > 0x7F80u, out = token >= left;
            sf[c] = scale_of(u);
            zf[c] = offset_of(u);
            bad[c] = __ballot_sync(0xffffffff, nan && !out);
            if (nan || out) {
              if (is_v) sf[c] = zf[c] = 0.f;
            } else {
              top = fmaxf(top, fmaxf(sf[c], fabsf(zf[c]) * most_z));
            }
          }
          if (NG > 1) top = fmaxf(top, __shfl_xor_sync(0xffffffff, top, 1));
          const int e = max((int)(__float_as_uint(top) >> 23) - 127, -72) + below + 1;
          const float f1 = __uint_as_float((uint32_t)(127 - (e >> 1)) << 23), f2 = __uint_as_float((uint32_t)(127 - (e - (e >> 1))) << 23);
#pragma unroll
          for (int c = 0; c < PAIRS; ++c) {
            const int x = lane * PAIRS + c;
            if (x < TOK * NG) s.pairs[w][is_v][x % NG * TOK + x / NG] = pack_f16(sf[c] * f1 * f2 * number, zf[c] * f1 * f2);
          }
          if (lane * PAIRS < TOK * NG && lane * PAIRS % NG == 0) {
            const int key = kb * TOK + lane * PAIRS / NG;
            if (is_v) {
              s.v_log[i % UNITS][key] = (float)e;
              s.v_inv[i % UNITS][key] = __uint_as_float((uint32_t)((int)ABOVE - e + 127) << 23);
            } else {
              s.k_unit[i % UNITS][key] = __uint_as_float((uint32_t)(e + K_SMALL_LOG + 127) << 23);
            }
          }
          if (is_v && lane == 0) {
            s.v_bad[i % UNITS][kb][0] = bad[0];
            s.v_bad[i % UNITS][kb][1] = PAIRS > 1 ? bad[PAIRS - 1] : 0;
          }
        }
        __syncwarp();
        // An image is free once the product of the tile two before has read it.  The warps are not in step: one may be
        // here before the product of the tile four before is done, but not that of six before, whose blocks have left the
        // ring.  A barrier for each of four tiles, here and for the blocks, then has one phase that can be meant.
        if (i >= 2) ok = __all_sync(0xffffffff, wait_for(s, &s.k_empty[(i - 2) & 3], ((i - 2) >> 2) & 1, a.err));
        if (!ok) break;
        {
          const int r0 = kb * 16 + 2 * g;
          uint8_t* out = k_image + b * W::K_IMAGE + r0 * 128;
          // Every second row the other way round: the lanes of a phase then touch 32 banks.
          const int flip = g & 1, at0 = ((t4 * 2 + flip) ^ (r0 & 7)) << 4, at1 = at0 ^ 16;
#pragma unroll 1
          for (int gi = 0; gi < NG; ++gi) {
            const uint2 sz = *reinterpret_cast<const uint2*>(&s.pairs[w][0][gi * TOK + 2 * g]);
#pragma unroll
            for (int tk = 0; tk < 2; ++tk) {
              const uint32_t pair = tk ? sz.y : sz.x, S = __byte_perm(pair, pair, 0x1010), Z = __byte_perm(pair, pair, 0x3232);
              uint8_t* row = out + gi * (WIDE_KEYS * 128) + tk * 128;   // an odd row: pieces and their neighbours change places
              if constexpr (BITS == 4) {
                const uint2 u = *reinterpret_cast<const uint2*>(in + gi * 512 + lane * 16 + tk * 8);
                const uint32_t n0 = flip ? u.y : u.x, n1 = flip ? u.x : u.y, m0 = n0 >> 8, m1 = n1 >> 8, T = sixteenth(S);
                *reinterpret_cast<uint4*>(row + (at0 ^ (tk * 16))) =
                    make_uint4(fma2(n0 & 0x000F000Fu, S, Z), fma2(n0 & 0x00F000F0u, T, Z), fma2(m0 & 0x000F000Fu, S, Z), fma2(m0 & 0x00F000F0u, T, Z));
                *reinterpret_cast<uint4*>(row + (at1 ^ (tk * 16))) =
                    make_uint4(fma2(n1 & 0x000F000Fu, S, Z), fma2(n1 & 0x00F000F0u, T, Z), fma2(m1 & 0x000F000Fu, S, Z), fma2(m1 & 0x00F000F0u, T, Z));
              } else {
                const uint4 u = lds128(in + gi * 1024 + tk * 512 + lane * 16);
                const uint32_t n0 = flip ? u.z : u.x, m0 = flip ? u.w : u.y, n1 = flip ? u.x : u.z, m1 = flip ? u.y : u.w;
                *reinterpret_cast<uint4*>(row + (at0 ^ (tk * 16))) =
                    make_uint4(fma2(n0 & 0x00FF00FFu, S, Z), fma2((n0 >> 8) & 0x00FF00FFu, S, Z), fma2(m0 & 0x00FF00FFu, S, Z), fma2((m0 >> 8) & 0x00FF00FFu, S, Z));
                *reinterpret_cast<uint4*>(row + (at1 ^ (tk * 16))) =
                    make_uint4(fma2(n1 & 0x00FF00FFu, S, Z), fma2((n1 >> 8) & 0x00FF00FFu, S, Z), fma2(m1 & 0x00FF00FFu, S, Z), fma2((m1 >> 8) & 0x00FF00FFu, S, Z));
              }
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.k_full[b]);
        if (i >= 2) ok = __all_sync(0xffffffff, wait_for(s, &s.v_empty[(i - 2) & 3], ((i - 2) >> 2) & 1, a.err));
        if (!ok) break;
        {
          const int perm = (2 * g + (g >> 2)) & 7;
          uint8_t* out = v_image + b * W::V_IMAGE + perm * 128 + (((kb * 2 + (t4 >> 1)) ^ perm) << 4) + (t4 & 1) * 8;
#pragma unroll 1
          for (int gi = 0; gi < NG; ++gi, out += 64 * 128) {
            const uint4 sz = *reinterpret_cast<const uint4*>(&s.pairs[w][1][gi * TOK + t4 * 4]);
            const uint32_t S0 = __byte_perm(sz.x, sz.z, 0x5410), Z0 = __byte_perm(sz.x, sz.z, 0x7632);
            const uint32_t S1 = __byte_perm(sz.y, sz.w, 0x5410), Z1 = __byte_perm(sz.y, sz.w, 0x7632);
#pragma unroll
            for (int h = 0; h < BITS / 4; ++h) {
              const uint4 u = lds128(in + W::CODES + gi * (BITS * 128) + h * 512 + lane * 16);
              const uint32_t n[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) {   // 4 bits: dims 2k and 2k + 1; 8 bits: dim 4h + k
                const uint32_t x = n[k];
                if constexpr (BITS == 4) {
                  *reinterpret_cast<uint2*>(out + 2 * k * 1024) = make_uint2(fma2((x << 4) & 0x00F000F0u, S0, Z0), fma2((x >> 4) & 0x00F000F0u, S1, Z1));
                  *reinterpret_cast<uint2*>(out + (2 * k + 1) * 1024) = make_uint2(fma2(x & 0x00F000F0u, S0, Z0), fma2((x >> 8) & 0x00F000F0u, S1, Z1));
                } else {
                  *reinterpret_cast<uint2*>(out + (4 * h + k) * 1024) = make_uint2(fma2(x & 0x00FF00FFu, S0, Z0), fma2((x >> 8) & 0x00FF00FFu, S1, Z1));
                }
              }
            }
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s.raw_empty[st]);
          mbar_arrive(&s.v_full[b]);
        }
      }
      before += p.n;
    }
  } else {
    // ---------------------------------------------------------------- softmax
    // After a wait that gave up these warps go on to their last piece's end (every later wait gives up at
    // once), so that their barriers meet.
    const int part = warp >> 2, quarter = warp & 3, slot = quarter * 32 + lane;   // the block of a tile, and the quarter of O's columns
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const auto row_of = [&](const Piece& x) { return x.row + (x.slot0 + min(slot, x.count - 1)) / group; };
    const auto query_of = [&](const Piece& x) {
      const int id = x.slot0 + min(slot, x.count - 1);
      return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (size_t)(x.row + id / group) * a.q_row +
                                            (size_t)(x.head * group + id % group) * a.q_head + part * (D / 4));
    };
    int i = 0;
    bool more = next_piece(p);
    int limit = more ? plan.lens[row_of(p)] : 0;
    while (more) {
      const bool used = slot < p.count, busy = quarter * 32 < p.count;
      float fac;
      {
        // The slot's quarter of the query, brought to [2^13, 2^14) by a power of two, as pairs in the order in which
        // the converters leave K's dims: 0 4 1 5 2 6 3 7, or 0 2 1 3 4 6 5 7.
        const uint4* from = query_of(p);
        uint4 u[D / 32];
#pragma unroll
        for (int j = 0; j < D / 32; ++j) u[j] = busy ? from[j] : make_uint4(0, 0, 0, 0);
        uint32_t bits = 0;   // of the largest magnitudes, which grow with them, infinities and NaN last
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) bits = __vmaxu2(bits, w[k] & 0x7FFF7FFFu);
        }
        s.top[part][slot] = __uint_as_float(max(bits << 16, bits & 0xFFFF0000u));
        slots_sync(quarter);
        bits = 0;
#pragma unroll
        for (int j = 0; j < TBLOCKS; ++j) bits = max(bits, __float_as_uint(s.top[j][slot]));
        const float big = __uint_as_float(bits);
        slots_sync(quarter);
        const int e = 13 - min(max((int)(bits >> 23) - 127, -100), 100);
        const float size = a.sm_scale == 0.f ? 0.f : copysignf(__uint_as_float((uint32_t)(e + 127) << 23), a.sm_scale);
        const float up = big < MAX_QUERY ? size : NAN;
        fac = fabsf(a.sm_scale) * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - K_SMALL_LOG - e) << 23);
        fac = fminf(fmaxf(fac, 0x1p-126f), 0x1p126f);   // its product with the distance to no reference is infinite
        if (busy) {
#pragma unroll
          for (int c = 0; c < D / 32; c += 2) {
            uint32_t y[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t w[4] = {u[c + j].x, u[c + j].y, u[c + j].z, u[c + j].w};
              float x[8];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float2 f = two_floats(w[k], false);
                x[2 * k] = f.x * up;
                x[2 * k + 1] = f.y * up;
              }
#pragma unroll
              for (int k = 0; k < 4; ++k)
                y[4 * j + k] = BITS == 4 ? pack_f16(x[k], x[k + 4]) : pack_f16(x[(k >> 1) * 4 + (k & 1)], x[(k >> 1) * 4 + (k & 1) + 2]);
            }
            tmem_st_x8(lanes + TMEM_Q + part * (D / 8) + c * 4, y);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.q_full);
      }
      // The next piece is looked up, and its queries are brought into L2, while this one's tiles are on their way.
      Piece next;
      more = next_piece(next);
      int next_limit = 0;
      if (more) {
        next_limit = plan.lens[row_of(next)];
        asm volatile("prefetch.global.L2 [%0];" ::"l"(query_of(next)));
      }
      // The reference's score is kept as it stands before `fac`, so that the largest one's difference to it is exactly 0.
      float ref = -INFINITY, rest = 0.f, l = 0.f;
      uint32_t bad = 0;
      for (int t = 0; t < p.n; ++t, ++i) {
        const int b = i & 1, valid = limit - (p.first + t) * WIDE_KEYS - part * TOK;
        wait_for(s, &s.s_full[b], (i >> 1) & 1, a.err);
        tc_fence_after();
        const float4* k_unit = reinterpret_cast<const float4*>(s.k_unit[i % UNITS] + part * TOK);
        const float4* v_log = reinterpret_cast<const float4*>(s.v_log[i % UNITS] + part * TOK);
        const float4* v_inv = reinterpret_cast<const float4*>(s.v_inv[i % UNITS] + part * TOK);
        uint32_t r[16];
        if (busy) {
          // A reference that has to move takes the largest score first, then what V's units add to the scores against it.  It is
          // set at a piece's first tile and looked at again at each other: two turns there where one has to move.
          bool raise = t == 0, grow = used && raise;
          for (;;) {
            const auto key_scores = [&]() {
              tmem_ld_32x32b_x16(lanes + b * 64 + part * 16, r);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const float4 k = k_unit[j / 4];
                const float2 lo = mul_two(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), make_float2(k.x, k.y));
                const float2 hi = mul_two(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])), make_float2(k.z, k.w));
                r[j] = __float_as_uint(lo.x);
                r[j + 1] = __float_as_uint(lo.y);
                r[j + 2] = __float_as_uint(hi.x);
                r[j + 3] = __float_as_uint(hi.y);
              }
            };
            const auto largest = [&]() {   // of the keys that the slot sees
              if (__any_sync(0xffffffff, valid < 16)) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  if (j >= valid) r[j] = 0xFF800000u;
              }
              float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int j = 0; j < 16; ++j) x[j & 1] = fmaxf(x[j & 1], __uint_as_float(r[j]));
              return fmaxf(x[0], x[1]);
            };
            const auto of_all = [&](float x) {   // the largest of the four blocks'
              s.top[part][slot] = x;
              slots_sync(quarter);
              x = fmaxf(fmaxf(s.top[0][slot], s.top[1][slot]), fmaxf(s.top[2][slot], s.top[3][slot]));
              slots_sync(quarter);
              return x;
            };
            const float was = rest;
            float moved = 0.f;
            if (raise) {
              key_scores();
              const float score = of_all(largest());
              if (grow && score > ref) {   // the same reference from another score
                moved = (score - ref) * fac;
                ref = score;
              }
            }
            key_scores();
            const float2 fac2 = make_float2(fac, fac), from = make_float2(-ref, -ref);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float4 v = v_log[j / 4];
              const float2 x = fma_two(add_two(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), from), fac2,
                                       j & 2 ? make_float2(v.z, v.w) : make_float2(v.x, v.y));
              r[j] = __float_as_uint(x.x);
              r[j + 1] = __float_as_uint(x.y);
            }
            float most = largest();
            if (!raise) {
              if (!slots_any(quarter, used && most > rest + SLACK)) break;
              most = of_all(most);   // by every thread: it has barriers
              grow = used && most > rest + SLACK;
              raise = true;
              continue;
            }
            most = of_all(most);
            float shrink = 1.f;
            if (grow) {
              rest = fmaxf(was - moved, most);
              shrink = ex2((was - moved) - rest);
              l *= shrink;
            }
            if (t > 0 && __any_sync(0xffffffff, grow)) {
              wait_for(s, &s.o_full[b ^ 1], ((i - 1) >> 1) & 1, a.err);   // O holds every tile before this one
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 4; c += 8) {
                uint32_t o[8];
                const uint32_t at = lanes + TMEM_O + part * (D / 4) + c;
                tmem_ld_x8(at, o);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                tmem_st_x8(at, o);
              }
              tmem_st_wait();
            }
            break;
          }
          const float off = LIFT - rest;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            float2 w = add_two(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), make_float2(off, off));
            w.x = ex2(w.x);
            w.y = ex2(w.y);
            r[j] = __float_as_uint(w.x);
            r[j + 1] = __float_as_uint(w.y);
            const float4 inv = v_inv[j / 4];
            sum = fma_two(w, j & 2 ? make_float2(inv.z, inv.w) : make_float2(inv.x, inv.y), sum);
          }
          l += sum.x + sum.y;
          // Tokens of a four lie in the order 0 2 1 3 in V's image; the weights take the place of their own scores.
          uint32_t pk[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int k = (j >> 1) * 4 + (j & 1);
            pk[j] = pack_f16(__uint_as_float(r[k]), __uint_as_float(r[k + 2]));
          }
          tmem_st_x8(lanes + b * 64 + part * 16, pk);
          tmem_st_wait();
          const uint32_t* poison = s.v_bad[i % UNITS][part];
          if (poison[0] | poison[1]) {
            constexpr int PAIRS = (TOK * NG + 31) / 32;
            for (int j = 0; j < min(valid, TOK); ++j)
              for (int gi = 0; gi < NG; ++gi) {
                const int x = j * NG + gi;
                bad |= (poison[x % PAIRS] >> (x / PAIRS) & 1) << gi;
              }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s.p_full[b]);
      }
      // ---- the slots' records
      s.top[part][slot] = l;
      slots_sync(quarter);
      l = (s.top[0][slot] + s.top[1][slot]) + (s.top[2][slot] + s.top[3][slot]);
      slots_sync(quarter);
      s.top[part][slot] = __uint_as_float(bad);
      slots_sync(quarter);
      bad = (__float_as_uint(s.top[0][slot]) | __float_as_uint(s.top[1][slot])) | (__float_as_uint(s.top[2][slot]) | __float_as_uint(s.top[3][slot]));
      wait_for(s, &s.o_full[(i - 1) & 1], ((i - 1) >> 1) & 1, a.err);
      tc_fence_after();
      const size_t rec = (size_t)p.chunk * a.num_kv_heads + p.head + cta;
      float* to = a.partial + rec * WIDE_SLOTS * (D + RECORD_REST);
      if (busy) {
        // Column gi 64 + 8 j + perm(g) is dim gi 64 + 8 g + j; the join puts them in order.  8 columns at a time go
        // through shared memory, so that an instruction stores whole sectors.
        float* mine = to + (size_t)(quarter * 32 + (lane >> 1)) * D + part * (D / 4) + (lane & 1) * 4;
        const int left = p.count - quarter * 32 - (lane >> 1);
#pragma unroll 1
        for (int c = 0; c < D / 4; c += 8) {
          uint32_t o[8];
          tmem_ld_x8(lanes + TMEM_O + part * (D / 4) + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * (1.f / BELOW));
          const bool nan = bad >> ((part * (D / 4) + c) >> 6) & 1;
          uint4* st = s.stage[warp][lane];   // its halves change places in every second four of slots
          const int turn = lane >> 2 & 1;
          st[turn] = nan ? make_uint4(0x7FC00000u, 0x7FC00000u, 0x7FC00000u, 0x7FC00000u) : make_uint4(o[0], o[1], o[2], o[3]);
          st[turn ^ 1] = nan ? make_uint4(0x7FC00000u, 0x7FC00000u, 0x7FC00000u, 0x7FC00000u) : make_uint4(o[4], o[5], o[6], o[7]);
          __syncwarp();
          const uint4 x0 = s.stage[warp][lane >> 1][(lane ^ lane >> 3) & 1];
          const uint4 x1 = s.stage[warp][16 + (lane >> 1)][(lane ^ lane >> 3) & 1];
          if (left > 0) *reinterpret_cast<uint4*>(mine + c) = x0;
          if (left > 16) *reinterpret_cast<uint4*>(mine + 16 * D + c) = x1;
          __syncwarp();
        }
        if (used && part == 0)
          *reinterpret_cast<float4*>(to + (size_t)WIDE_SLOTS * D + RECORD_REST * slot) =
              make_float4(ref * fac, rest, l, 0.f);
      }
      slots_sync(quarter);   // the poisoned groups have been read
      tc_fence_before();
      p = next;
      limit = next_limit;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

template <int D, int BITS>
int launch(const QuantAttnArgs& a, cudaStream_t stream) {
  using W = Wide<D, BITS>;
  const auto kernel = wide_kernel<W>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, W::BYTES);
  zs_launch(kernel, a.grid, THREADS, W::BYTES, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

}  // namespace

int launch_wide(QuantAttnArgs a, cudaStream_t stream) {
  if (a.chunk != WIDE_SLOTS || a.stage != WIDE_KEYS || a.grid > 148 || a.half) return -1;
  if (a.head_dim == 64) return a.bits == 4 ? launch<64, 4>(a, stream) : launch<64, 8>(a, stream);
  if (a.head_dim == 128) return a.bits == 4 ? launch<128, 4>(a, stream) : launch<128, 8>(a, stream);
  return a.bits == 4 ? launch<256, 4>(a, stream) : launch<256, 8>(a, stream);
}

}  // namespace qc
}  // namespace zs
