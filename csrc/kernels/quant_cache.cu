// K/V cache held in 4 or 8 bits: rows quantised into it, read back, and attention over it.
//
// Numbers.  A group is 64 consecutive dims of one token and head, of K or of V.  With N = 15 or
// 255 it is held as whole numbers n in 0..N, a scale s and an offset z in bf16:
//     z = min(x) rounded down,  s = (max(x) - z) / N rounded up,  n = (x - z) / s to the nearest,
// ties to even, all in 32 bits, and stands for s n + z.  z is rounded down and s up so that no x
// falls outside 0..N.  A group with a NaN, an infinity or a value beyond 2^126 is poisoned (s and z
// are NaN) and reads back as NaN.
//
// Storage.  16 tokens of one kv head are one block: the numbers of K, those of V, then a 32-bit
// (s | z << 16) per token and group, of K and of V.  The order of the numbers is the one in which
// the attention's matrix fragments want them (k_offset, v_offset): a lane reads 16 bytes that are
// its own, the eight lanes of a phase touch 32 different banks, and a block is one bulk copy.
//
// Attention.  With q . K_j = sum over groups of s (q . n) + z (sum of q), and the same for
// sum_j p_j V_j = sum_j (p_j s) n_j + p_j z, the whole numbers themselves are the matrix operand:
// (w & 0x000F000F) of a 32-bit word of eight numbers is two f16 subnormals n 2^-24, exact, and
// (w & 0x00F000F0) the next two times 16.  So a pair costs one or two integer instructions and no
// multiplication; scales go to the 32-bit scores and to the weights.  The scaled weights are
// rounded to f16 (2^-11): the running reference of a row is the maximum of score + log2(scale), so
// that they stay below 2^15 whatever the size of V.
#include <cuda_fp16.h>

#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace qc {

constexpr int TOK = 16;      // tokens of a block
constexpr int GROUP = 64;    // dims that share a scale and an offset
constexpr uint32_t POISON = 0x7FFFFFFFu;  // z = NaN, s = NaN with its sign set (a negative 16-bit number)

// Bytes of the block of 16 tokens of one kv head.
__host__ __device__ constexpr int code_bytes(int d, int bits) { return TOK * d * bits / 8; }
__host__ __device__ constexpr int block_bytes(int d, int bits) { return 2 * code_bytes(d, bits) + 2 * TOK * (d / GROUP) * 4; }

// Where the 8 numbers of dims d..d+7 (d a multiple of 8) of K's token t are in the block: bits bytes.
__device__ __forceinline__ int k_offset(int dim, int bits, int t, int d) {
  const int lane = (d & 63) >> 4, half = (d >> 3) & 1;   // of the four lanes of a row, 16 dims each
  if (bits == 8) return (d >> 6) * 1024 + t * 64 + lane * 16 + half * 8;
  if (dim == 64) return t * 32 + lane * 8 + half * 4;
  return (d >> 7) * 1024 + t * 64 + lane * 16 + ((d >> 6) & 1) * 8 + half * 4;
}

// The same of V's: eight lanes have 8 dims of a group each, for all 16 tokens.  The two halves of the
// tokens are exchanged in every second of them, which spreads a phase over all banks.
__device__ __forceinline__ int v_offset(int dim, int bits, int t, int d) {
  const int lane = (d & 63) >> 3;
  if (bits == 4 && dim == 64) return lane * 64 + ((t >> 3) ^ ((lane >> 1) & 1)) * 32 + (t & 7) * 4;
  const int at = lane * 128 + ((t >> 3) ^ (lane & 1)) * 64 + (t & 7) * 8;
  return bits == 8 ? (d >> 6) * 1024 + at : (d >> 7) * 1024 + at + ((d >> 6) & 1) * 4;
}

__device__ __forceinline__ float bf16_up(float x) {   // x >= 0
  return __uint_as_float((__float_as_uint(x) + 0xFFFFu) & 0xFFFF0000u);
}
__device__ __forceinline__ float bf16_down(float x) {
  const uint32_t u = __float_as_uint(x);
  return __uint_as_float((u >> 31 ? u + 0xFFFFu : u) & 0xFFFF0000u);
}
__device__ __forceinline__ float scale_of(uint32_t sz) { return __uint_as_float(sz << 16); }
__device__ __forceinline__ float offset_of(uint32_t sz) { return __uint_as_float(sz & 0xFFFF0000u); }

__device__ __forceinline__ float2 two_floats(uint32_t u, bool half) {
  return half ? __half22float2(*reinterpret_cast<const __half2*>(&u)) : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
__device__ __forceinline__ uint32_t two_halves(float a, float b, bool half) {
  if (half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The block of (slot, position) for kv head 0, or null where there is none.  Heads are `stride` bytes apart.
__device__ __forceinline__ uint8_t* block_at(const QuantRowsArgs& a, int row, int* token) {
  const int pos = a.positions[row], slot = a.slots[row];
  if (pos < 0) return nullptr;
  if (slot < 0 || slot >= a.num_slots || (pos >> a.page_shift) >= a.max_pages) {
    report_error(a.err, kErrBadShape);
    return nullptr;
  }
  const int page = a.page_table[(size_t)slot * a.max_pages + (pos >> a.page_shift)];
  if (page < 0 || page >= a.num_pages) {
    report_error(a.err, kErrBadShape);
    return nullptr;
  }
  *token = pos & (TOK - 1);
  const int sub = (pos & ((1 << a.page_shift) - 1)) / TOK;
  return a.data + (((size_t)page * a.num_kv_heads << (a.page_shift - 4)) + sub) * block_bytes(a.head_dim, a.bits);
}

// Eight dims a thread, eight threads a group.
constexpr int ROW_THREADS = 256;

__global__ void __launch_bounds__(ROW_THREADS) store_kernel(const QuantRowsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int octets = a.head_dim / 8;
  const long long item = (long long)blockIdx.x * ROW_THREADS + threadIdx.x;
  const int d = (int)(item % octets) * 8;
  const long long rest = item / octets;
  const int head = (int)(rest % a.num_kv_heads);
  const bool is_v = (rest / a.num_kv_heads) & 1;
  const long long row = rest / a.num_kv_heads / 2;
  if (row >= a.rows) return;   // whole groups of eight threads
  const unsigned mates = 0xFFu << (threadIdx.x & 24);
  const long long from = is_v ? row * a.v_row + head * a.v_head : row * a.k_row + head * a.k_head;
  const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(is_v ? a.v : a.k) + from + d);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float x[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = two_floats(w[j], a.half);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
  float lo = x[0], hi = x[0];
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
    fine = fine && fabsf(x[j]) <= 0x1p126f;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(mates, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(mates, hi, o));
  }
  fine = (__ballot_sync(mates, fine) & mates) == mates;
  const int top = (1 << a.bits) - 1;
  const float z = bf16_down(lo);
  const float s = bf16_up(__fdiv_rn(hi - z, (float)top));
  uint32_t n[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float q = s > 0.f ? rintf(__fdiv_rn(x[j] - z, s)) : 0.f;
    q = fine ? fminf(fmaxf(q, 0.f), (float)top) : 0.f;
    if (a.bits == 4) n[0] |= (uint32_t)q << (4 * j);
    else n[j >> 2] |= (uint32_t)q << (8 * (j & 3));
  }
  int t = 0;
  uint8_t* block = block_at(a, (int)row, &t);
  if (block == nullptr) return;
  block += ((size_t)head << (a.page_shift - 4)) * block_bytes(a.head_dim, a.bits);
  const int codes = code_bytes(a.head_dim, a.bits), groups = a.head_dim / GROUP;
  uint8_t* to = is_v ? block + codes + v_offset(a.head_dim, a.bits, t, d) : block + k_offset(a.head_dim, a.bits, t, d);
  if (a.bits == 4) *reinterpret_cast<uint32_t*>(to) = n[0];
  else *reinterpret_cast<uint2*>(to) = make_uint2(n[0], n[1]);
  if ((d & 63) == 0) {
    uint32_t* sz = reinterpret_cast<uint32_t*>(block + 2 * codes) + (is_v ? TOK * groups : 0) + t * groups + d / GROUP;
    *sz = fine ? __float_as_uint(s) >> 16 | __float_as_uint(z) : POISON;
  }
}

__global__ void __launch_bounds__(ROW_THREADS) load_kernel(const QuantRowsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int octets = a.head_dim / 8;
  const long long item = (long long)blockIdx.x * ROW_THREADS + threadIdx.x;
  const int d = (int)(item % octets) * 8;
  const long long rest = item / octets;
  const int head = (int)(rest % a.num_kv_heads);
  const bool is_v = (rest / a.num_kv_heads) & 1;
  const long long row = rest / a.num_kv_heads / 2;
  if (row >= a.rows) return;
  int t = 0;
  const uint8_t* block = block_at(a, (int)row, &t);
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = 0.f;
  if (block != nullptr) {
    block += ((size_t)head << (a.page_shift - 4)) * block_bytes(a.head_dim, a.bits);
    const int codes = code_bytes(a.head_dim, a.bits), groups = a.head_dim / GROUP;
    const uint8_t* from = is_v ? block + codes + v_offset(a.head_dim, a.bits, t, d) : block + k_offset(a.head_dim, a.bits, t, d);
    const uint32_t sz = *(reinterpret_cast<const uint32_t*>(block + 2 * codes) + (is_v ? TOK * groups : 0) + t * groups + d / GROUP);
    const float s = scale_of(sz), z = offset_of(sz);
    if (a.bits == 4) {
      const uint32_t n = *reinterpret_cast<const uint32_t*>(from);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf((float)(n >> (4 * j) & 15), s, z);
    } else {
      const uint2 n = *reinterpret_cast<const uint2*>(from);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf((float)((j < 4 ? n.x : n.y) >> (8 * (j & 3)) & 255), s, z);
    }
  }
  const long long to = is_v ? row * a.v_row + head * a.v_head : row * a.k_row + head * a.k_head;
  void* out = const_cast<void*>(is_v ? a.v : a.k);
  if (a.f32) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + to + d);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + to + d) =
        make_uint4(two_halves(x[0], x[1], a.half), two_halves(x[2], x[3], a.half), two_halves(x[4], x[5], a.half), two_halves(x[6], x[7], a.half));
  }
}

// ------------------------------------------------------------------------------------ plan
// A query slot is one (row, q head of the kv head's group) of a sequence; up to `a.chunk` slots of one
// sequence and kv head are a unit, and its keys are walked in stages of 32.  The chunks (units of all
// kv heads at once) stand in a table with the number of stages before them; CTA b of the attention
// takes the stages [b T / B, (b + 1) T / B) of all T, so that every CTA has the same work whatever the
// lengths.  One CTA of 1024 threads plans; a step's layers share the plan.
constexpr int PLAN_THREADS = 1024;
constexpr int STAGE = 32;   // keys

struct Chunk {          // 32 bytes
  long long before;     // stages of the chunks before, all kv heads
  int row, slot;        // first row of the sequence, its page-table row
  int first, count;     // slots [first, first + count) of the sequence
  int len, stages;      // keys of the longest row among them, stages of one kv head
};

struct Plan {           // the workspace's integers
  long long* total;     // stages of all chunks, all kv heads
  int* chunks;          // number of chunks
  Chunk* table;         // [max_chunks]
  int2* rows;           // [max_rows] first chunk and first row of the row's sequence (-1: none)
  int* lens;            // [max_rows] keys of the row
  int* offset;          // [max_seqs] chunks before the sequence
};

__host__ __device__ inline Plan plan_of(const QuantAttnArgs& a) {
  Plan p;
  uint8_t* w = reinterpret_cast<uint8_t*>(a.work);
  p.total = reinterpret_cast<long long*>(w);
  p.chunks = reinterpret_cast<int*>(w + 8);
  p.table = reinterpret_cast<Chunk*>(w + 32);
  p.rows = reinterpret_cast<int2*>(p.table + a.max_chunks);
  p.lens = reinterpret_cast<int*>(p.rows + a.max_rows);
  p.offset = p.lens + a.max_rows;
  return p;
}

// Exclusive sum over the CTA's threads; *all gets the sum of all.
__device__ __forceinline__ long long block_scan(long long x, long long* warps, long long* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long run = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffff, run, o);
    if (lane >= o) run += y;
  }
  __syncthreads();   // the last call's sums have been read
  if (lane == 31) warps[warp] = run;
  __syncthreads();
  if (warp == 0) {
    long long s = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffff, s, o);
      if (lane >= o) s += y;
    }
    warps[lane] = s;
  }
  __syncthreads();
  *all = warps[31];
  return run - x + (warp > 0 ? warps[warp - 1] : 0);
}

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const QuantAttnArgs a) {
  __shared__ long long warps[32];
  pdl_wait();
  pdl_trigger();
  const Plan p = plan_of(a);
  const int group = a.num_q_heads / a.num_kv_heads;
  // Rows of no sequence have no chunk.
  for (int r = threadIdx.x; r < a.rows; r += PLAN_THREADS) {
    p.rows[r] = make_int2(-1, 0);
    p.lens[r] = max(a.seq_lens[r], 0);
  }
  long long base = 0, all = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += PLAN_THREADS) {
    const int s = s0 + threadIdx.x;
    int n = 0;
    if (s < a.num_seqs) {
      int lo = s, hi = s + 1;
      if (a.seq_start != nullptr) {
        lo = a.seq_start[s];
        hi = a.seq_start[s + 1];
      }
      if (lo < 0 || hi < lo || hi > a.rows || hi - lo > a.max_seq_rows) {
        report_error(a.err, kErrBadShape);
        lo = hi = 0;
      }
      n = ((hi - lo) * group + a.chunk - 1) / a.chunk;
    }
    const long long at = base + block_scan(n, warps, &all);
    if (s < a.num_seqs) p.offset[s] = (int)at;
    base += all;
  }
  // The table is sized for sequences that follow one another; boundaries that go back do not fit.
  const int chunks = base <= a.max_chunks ? (int)base : 0;
  if (chunks < base && threadIdx.x == 0) report_error(a.err, kErrBadShape);
  __syncthreads();
  base = 0;
  for (int c0 = 0; c0 < chunks; c0 += PLAN_THREADS) {
    const int c = c0 + threadIdx.x;
    Chunk e = {};
    if (c < chunks) {
      int lo = 0, hi = a.num_seqs;   // the last sequence with offset <= c that has chunks: offsets of empty ones repeat
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.offset[mid] <= c) lo = mid;
        else hi = mid;
      }
      const int r0 = a.seq_start != nullptr ? a.seq_start[lo] : lo;
      const int r1 = a.seq_start != nullptr ? a.seq_start[lo + 1] : lo + 1;
      e.row = r0;
      e.slot = a.slots[r0];
      e.first = (c - p.offset[lo]) * a.chunk;
      e.count = min(a.chunk, (r1 - r0) * group - e.first);
      const int from = r0 + e.first / group, to = r0 + (e.first + e.count - 1) / group;
      for (int r = from; r <= to; ++r) {
        e.len = max(e.len, a.seq_lens[r]);
        // A row whose slots are in two chunks is entered by both, with the same numbers.
        p.rows[r] = make_int2(p.offset[lo], r0);
      }
      e.stages = (e.len + STAGE - 1) / STAGE;
    }
    const long long cost = (long long)e.stages * a.num_kv_heads;
    e.before = base + block_scan(cost, warps, &all);
    if (c < chunks) p.table[c] = e;
    base += all;
  }
  if (threadIdx.x == 0) {
    *p.total = base;
    *p.chunks = chunks;
  }
}

// Number of CTAs that share T stages.
__device__ __forceinline__ int ctas_of(long long total, int grid, int least) {
  return (int)max(1ll, min((long long)grid, total / least));
}

// ------------------------------------------------------------------------------- attention
constexpr int WARPS = 8;
constexpr int MAX_RING = 8;
constexpr float LIFT = 11.f;    // log2 of what a weight times its scale is held at: below 2^(11 + 1 + SLACK)
constexpr float SLACK = 3.f;    // the reference moves when a score goes this far above it

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {   // 2^x, results below 2^-126 as 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int N>
__device__ __forceinline__ void lds(uint32_t (&r)[N], const uint8_t* p) {
  static_assert(N == 1 || N == 2 || N % 4 == 0, "");
  if constexpr (N == 1) {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r[0] = u.x;
    r[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      r[4 * i] = u.x;
      r[4 * i + 1] = u.y;
      r[4 * i + 2] = u.z;
      r[4 * i + 3] = u.w;
    }
  }
}

// Shared memory of a CTA with `lanes` key lanes (KW) of `sw` warps.
template <int D, int BITS, int NT>
struct Shape {
  static constexpr int KS = D / 16;                 // k16 steps of a score
  static constexpr int NG = D / GROUP;
  static constexpr int CODES = code_bytes(D, BITS);
  static constexpr int BLOCK = block_bytes(D, BITS);
  static constexpr int STAGE_BYTES = 2 * BLOCK;
  static constexpr int MERGE_REGS = KS * NT * 4 + NG * NT * 2 + 4 * NT;   // O, its offset part, l and reference
  static constexpr int MERGE = WARPS / 2 * MERGE_REGS * 128;
  static constexpr int HEAD = 2 * WARPS * MAX_RING * 8;
  __host__ __device__ static constexpr int slots(int sw) { return 8 * NT * sw; }
  __host__ __device__ static constexpr int fixed(int sw) {
    return HEAD + slots(sw) * (NG + 2) * 4 + KS * NT * sw * 256 + (sw < WARPS ? MERGE : 0);
  }
};

struct Piece {
  int chunk, head, first, n;   // stages [first, first + n) of the unit
  int row, slot, slot0, count, len;
};

template <int D, int BITS, int NT, int MIN_CTAS>
__global__ void __launch_bounds__(WARPS * 32, MIN_CTAS) attend_kernel(const QuantAttnArgs a) {
  using S = Shape<D, BITS, NT>;
  constexpr int KS = S::KS, NG = S::NG, BLOCK = S::BLOCK;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_trigger();
  const Plan plan = plan_of(a);
  const long long total = *plan.total;
  const int sw_n = a.slot_warps, kw = WARPS / sw_n, ring = a.ring;
  const int B = ctas_of(total, gridDim.x, kw);
  const int b = blockIdx.x;
  if (b >= B || total == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kl = warp / sw_n, sw = warp % sw_n;   // key lane, slot part
  const int g = lane >> 2, t = lane & 3;
  const int slots = S::slots(sw_n);
  const int group = a.num_q_heads / a.num_kv_heads;

  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + kl * ring;
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem) + WARPS * MAX_RING + kl * ring;
  float* qsum = reinterpret_cast<float*>(smem + S::HEAD);         // [NG][slots]
  float* qfac = qsum + NG * slots;                                // [slots]
  int* qlen = reinterpret_cast<int*>(qfac + slots);               // [slots]
  uint8_t* qfrag = reinterpret_cast<uint8_t*>(qlen + slots);      // [KS][NT sw][32 lanes][8 bytes]
  float* merge = reinterpret_cast<float*>(qfrag + KS * NT * sw_n * 256);
  uint8_t* stage0 = smem + a.ring_offset + (size_t)kl * ring * S::STAGE_BYTES;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kw; ++i)
      for (int j = 0; j < ring; ++j) {
        mbar_init(reinterpret_cast<uint64_t*>(smem) + i * ring + j, 1);
        mbar_init(reinterpret_cast<uint64_t*>(smem) + WARPS * MAX_RING + i * ring + j, sw_n);
      }
    fence_barrier_init();
  }

  // This CTA's stages, and the chunk that the first is in.
  const long long lo = total * b / B, hi = total * (b + 1) / B;
  const int chunks = *plan.chunks;
  int c = 0;
  {
    int n = chunks;   // the last chunk with before <= lo, 32 candidates at a time
    while (n > 1) {
      const int step = (n + 31) / 32;
      const int at = c + lane * step;
      const bool below = lane * step < n && plan.table[at].before <= lo;
      const int k = 31 - __clz(__ballot_sync(0xffffffff, below));   // lane 0 is always below
      c += k * step;
      n = min(step, n - k * step);
    }
  }
  __syncthreads();

  auto piece_at = [&](long long pos) {   // c: a chunk at or before pos
    Chunk e = plan.table[c];
    while (e.before + (long long)e.stages * a.num_kv_heads <= pos) e = plan.table[++c];
    const int r = (int)(pos - e.before);
    Piece p;
    p.chunk = c;
    p.head = r / e.stages;
    p.first = r % e.stages;
    p.n = (int)min((long long)(e.stages - p.first), hi - pos);
    p.row = e.row;
    p.slot = e.slot;
    p.slot0 = e.first;
    p.count = e.count;
    p.len = e.len;
    return p;
  };

  // The producer of a key lane: its first warp.  Lane j of it holds the page of block j % 2 of stage j / 2 of 16.
  int ids = 0, ids_next = 0, issued = 0, fill = 0, fill_phase = 1;   // stages of the piece issued; ring place
  Piece src = {};      // the piece that is being loaded
  int src_n = 0;
  const int bshift = a.page_shift - 4;
  auto page_ids = [&](int i0) {
    const int stage = src.first + kl + (i0 + (lane >> 1)) * kw;
    const int blk = stage * 2 + (lane & 1);
    int page = 0;
    if (i0 + (lane >> 1) < src_n && blk * TOK < src.len) {
      const int index = blk >> bshift;
      const bool ok = src.slot >= 0 && src.slot < a.num_slots && index < a.max_pages;
      page = ok ? a.page_table[(size_t)src.slot * a.max_pages + index] : -1;
      if (page < 0 || page >= a.num_pages) {
        report_error(a.err, kErrBadShape);
        page = 0;
      }
    }
    return page;
  };
  auto start_loads = [&](const Piece& p) {
    src = p;
    src_n = (p.n - kl + kw - 1) / kw;
    if (p.n <= kl) src_n = 0;
    issued = 0;
    ids = page_ids(0);
    ids_next = page_ids(16);
  };
  auto issue = [&]() {   // the next stage of the source piece into the ring
    if (issued >= src_n) return;
    mbar_wait(&empty[fill], fill_phase, a.err);
    const int stage = src.first + kl + issued * kw;
    const int k = issued & 15;
    const int p0 = __shfl_sync(0xffffffff, ids, 2 * k), p1 = __shfl_sync(0xffffffff, ids, 2 * k + 1);
    if (lane == 0) {
      uint8_t* to = stage0 + (size_t)fill * S::STAGE_BYTES;
      const int blk = stage * 2, mask = (1 << bshift) - 1;
      const bool two = (blk + 1) * TOK < src.len;
      mbar_expect_tx(&full[fill], two ? 2 * BLOCK : BLOCK);
      bulk_load(to, a.data + (((((size_t)p0 * a.num_kv_heads + src.head) << bshift) + (blk & mask)) * BLOCK), BLOCK, &full[fill]);
      if (two)
        bulk_load(to + BLOCK, a.data + (((((size_t)p1 * a.num_kv_heads + src.head) << bshift) + ((blk + 1) & mask)) * BLOCK), BLOCK, &full[fill]);
    }
    if (++fill == ring) {
      fill = 0;
      fill_phase ^= 1;
    }
    if ((++issued & 15) == 0) {
      ids = ids_next;
      ids_next = page_ids(issued + 16);
    }
  };

  int use = 0, use_phase = 0;   // the ring's place to be read
  long long pos = lo;
  Piece cur = piece_at(pos);
  if (sw == 0) {
    start_loads(cur);
    for (int i = 0; i < ring; ++i) issue();
  }
  while (true) {
    // Queries: a warp a slot.  A slot's numbers are brought to [2^13, 2^14) by a power of two, where f16
    // holds a bf16 or f16 exactly down to 2^-27 of the largest; the numbers that meet w & 0x00F000F0 are
    // divided by 16.
    const int slot_end = min(slots, (cur.count + 7) / 8 * 8);
    for (int s = warp; s < slot_end; s += WARPS) {
      constexpr int PER = D / 32;
      float x[PER];
      const int id = cur.slot0 + s;
      const int row = cur.row + id / group;
      const bool real = s < cur.count;
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = 0.f;
      if (real) {
        const uint16_t* from = static_cast<const uint16_t*>(a.q) + (size_t)row * a.q_row + (size_t)(cur.head * group + id % group) * a.q_head + lane * PER;
        uint32_t w[PER / 2];
        if constexpr (PER == 2) w[0] = *reinterpret_cast<const uint32_t*>(from);
        if constexpr (PER == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(from);
          w[0] = u.x; w[1] = u.y;
        }
        if constexpr (PER == 8) {
          const uint4 u = *reinterpret_cast<const uint4*>(from);
          w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
        }
#pragma unroll
        for (int j = 0; j < PER / 2; ++j) {
          const float2 f = two_floats(w[j], a.half);
          x[2 * j] = f.x;
          x[2 * j + 1] = f.y;
        }
      }
      float big = 0.f;
      bool fine = true;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        big = fmaxf(big, fabsf(x[j]));
        fine = fine && fabsf(x[j]) < INFINITY;
      }
      big = warp_max(big);
      fine = __all_sync(0xffffffff, fine);
      const int e = 13 - min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 100);
      const float up = __uint_as_float((uint32_t)(e + 127) << 23);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        x[j] = fine ? x[j] * up : NAN;
        sum += x[j];
      }
#pragma unroll
      for (int o = 1; o < GROUP / PER; o <<= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
      if (lane % (GROUP / PER) == 0) qsum[lane / (GROUP / PER) * slots + s] = sum * 0x1p-24f;
      if (lane == 0) {
        qfac[s] = a.sm_scale * 1.4426950408889634f * __uint_as_float((uint32_t)(24 - e + 127) << 23);
        qlen[s] = real ? plan.lens[row] : cur.len;
      }
      __half* q16 = reinterpret_cast<__half*>(qfrag);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int d = lane * PER + j, in = d & 15;
        int ks, reg, part;
        if (BITS == 4) {
          ks = (d >> 6) * 4 + (in >> 3) * 2 + ((in >> 1) & 1);
          reg = in & 1;
          part = (in >> 2) & 1;
          if (reg) x[j] *= 0.0625f;
        } else {
          ks = (d >> 6) * 4 + (in >> 2);
          reg = in & 1;
          part = (in >> 1) & 1;
        }
        const int ln = (s & 7) * 4 + ((d & 63) >> 4);
        q16[(((ks * NT * sw_n + (s >> 3)) * 32 + ln) * 2 + reg) * 2 + part] = __float2half_rn(x[j]);
      }
    }
    __syncthreads();

    // A part of the slots that the chunk does not reach has nothing to do (but it releases the stages).
    const bool busy = sw * NT * 8 < slot_end;
    float o[KS][NT][4], oz[NG][NT][2], l[NT][2], ref[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][n][j] = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < NG; ++i) oz[i][n][j] = 0.f;
        l[n][j] = 0.f;
        ref[n][j] = -INFINITY;
      }
    }
    int lens[NT][2], shortest = INT_MAX;
    float fac[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s = (sw * NT + n) * 8 + 2 * t + j;
        const bool there = s < slot_end;
        lens[n][j] = there ? qlen[s] : cur.len;
        fac[n][j] = there ? qfac[s] : 0.f;
        shortest = min(shortest, lens[n][j]);
      }
    shortest = __reduce_min_sync(0xffffffff, shortest);

    const int n_mine = cur.n > kl ? (cur.n - kl + kw - 1) / kw : 0;
    for (int it = 0; it < n_mine; ++it) {
      mbar_wait(&full[use], use_phase, a.err);
      if (busy) {
        const uint8_t* st = stage0 + (size_t)use * S::STAGE_BYTES;
        const int key0 = (cur.first + kl + it * kw) * STAGE;
        // Scores.
        float sc[2][NT][4];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[kb][n][j] = 0.f;
        uint32_t ksz[2][2][NG];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 2; ++r) lds(ksz[kb][r], st + kb * BLOCK + 2 * S::CODES + (g + 8 * r) * NG * 4);
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) {
          constexpr int WG = BITS / 2;   // words of a lane in a group
          uint32_t w[2][2][WG];
          constexpr bool SMALL = BITS == 4 && D == 64;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int row = g + 8 * r;
              const uint8_t* p = st + kb * BLOCK +
                                 (SMALL ? row * 32 + t * 8 : BITS == 8 ? gi * 1024 + row * 64 + t * 16 : (gi >> 1) * 1024 + row * 64 + t * 16 + (gi & 1) * 8);
              lds(w[kb][r], p);
            }
          float acc[2][NT][4];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[kb][n][j] = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t bq[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
              lds(bq[n], qfrag + (((gi * 4 + k) * NT * sw_n + sw * NT + n) * 32 + lane) * 8);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              uint32_t f[2][2];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                if (BITS == 4) {
                  const uint32_t x = w[kb][r][k >> 1] >> (8 * (k & 1));
                  f[r][0] = x & 0x000F000Fu;
                  f[r][1] = x & 0x00F000F0u;
                } else {
                  f[r][0] = w[kb][r][k % WG] & 0x00FF00FFu;
                  f[r][1] = (w[kb][r][k % WG] >> 8) & 0x00FF00FFu;
                }
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16816(acc[kb][n], f[0][0], f[1][0], f[0][1], f[1][1], bq[n][0], bq[n][1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 qs = *reinterpret_cast<const float2*>(qsum + gi * slots + (sw * NT + n) * 8 + 2 * t);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t sz = ksz[kb][j >> 1][gi];
                sc[kb][n][j] = fmaf(scale_of(sz), acc[kb][n][j], fmaf(offset_of(sz), j & 1 ? qs.y : qs.x, sc[kb][n][j]));
              }
          }
        }
        // Weights.
        const bool whole = key0 + STAGE <= shortest;
        uint32_t vsz[2][2][NG];
        float most[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) most[n][0] = most[n][1] = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            lds(vsz[kb][r], st + kb * BLOCK + 2 * S::CODES + TOK * NG * 4 + (g + 8 * r) * NG * 4);
            int top = 0x1F80;   // at least 2^-64; a poisoned scale is negative
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) top = max(top, (int)(short)(vsz[kb][r][gi] & 0xFFFFu));
            const float ex = __uint_as_float(0x4B000000u | (uint32_t)(top >> 7)) - (8388608.f + 127.f);
            const int key = key0 + kb * 16 + r * 8 + g;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float x = sc[kb][n][2 * r + j] * fac[n][j];
                if (!whole && key >= lens[n][j]) x = -INFINITY;
                sc[kb][n][2 * r + j] = x;
                most[n][j] = fmaxf(most[n][j], x + ex);
              }
          }
        bool move = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) move = move || most[n][0] > ref[n][0] + SLACK || most[n][1] > ref[n][1] + SLACK;
        if (__any_sync(0xffffffff, move)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float m = most[n][j];
#pragma unroll
              for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffff, m, x));
              m = fmaxf(m, ref[n][j]);
              const float f = m == ref[n][j] ? 1.f : ex2(ref[n][j] - m);
              ref[n][j] = m;
              l[n][j] *= f;
#pragma unroll
              for (int gi = 0; gi < NG; ++gi) oz[gi][n][j] *= f;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                o[i][n][j] *= f;
                o[i][n][2 + j] *= f;
              }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          bool seen[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              seen[n][j] = whole || key0 + kb * 16 + (j >> 1) * 8 + g < lens[n][j & 1];
              const float p = seen[n][j] ? ex2(sc[kb][n][j] - ref[n][j & 1] + LIFT) : 0.f;
              sc[kb][n][j] = p;
              l[n][j & 1] += p;
            }
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            uint32_t bp[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float ps[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t sz = vsz[kb][j >> 1][gi];
                ps[j] = sc[kb][n][j] * scale_of(sz);
                float pz = sc[kb][n][j] * offset_of(sz);
                if (!seen[n][j]) ps[j] = pz = 0.f;   // nothing of a masked key, NaN among it, is taken
                oz[gi][n][j & 1] += pz;
              }
              bp[n][0] = transpose8x8(pack_f16(ps[0], ps[1]));
              bp[n][1] = transpose8x8(pack_f16(ps[2], ps[3]));
            }
            // V's numbers of tokens 2t, 2t + 1 and 2t + 8, 2t + 9 for this lane's 8 dims of the group.
            constexpr int WV = BITS / 4;   // words of 8 dims
            uint32_t va[2][2][WV];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint8_t* vp = st + kb * BLOCK + S::CODES;
              if constexpr (BITS == 4 && D == 64) {
                uint32_t u[2];
                lds(u, vp + g * 64 + (h ^ ((g >> 1) & 1)) * 32 + t * 8);
                va[h][0][0] = u[0];
                va[h][1][0] = u[1];
              } else {
                uint32_t u[4];
                lds(u, vp + (BITS == 8 ? gi : gi >> 1) * 1024 + g * 128 + (h ^ (g & 1)) * 64 + t * 16);
                if constexpr (BITS == 4) {
                  va[h][0][0] = u[gi & 1];
                  va[h][1][0] = u[2 + (gi & 1)];
                } else {
                  va[h][0][0] = u[0];
                  va[h][0][WV - 1] = u[1];
                  va[h][1][0] = u[2];
                  va[h][1][WV - 1] = u[3];
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t f[2][2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (BITS == 4) {
                  const uint32_t x = __byte_perm(va[h][0][0], va[h][1][0], i < 2 ? 0x5410 : 0x7632) >> (8 * (i & 1));
                  f[h][0] = x & 0x000F000Fu;
                  f[h][1] = x & 0x00F000F0u;
                } else {
                  const uint32_t x = __byte_perm(va[h][0][(i >> 1) % WV], va[h][1][(i >> 1) % WV], i & 1 ? 0x7632 : 0x5410);
                  f[h][0] = x & 0x00FF00FFu;
                  f[h][1] = (x >> 8) & 0x00FF00FFu;
                }
              }
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16816(o[gi * 4 + i][n], f[0][0], f[0][1], f[1][0], f[1][1], bp[n][0], bp[n][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[use]);
      if (++use == ring) {
        use = 0;
        use_phase ^= 1;
      }
      if (sw == 0) issue();
    }

    // The next piece's first stages are on their way while this one's warps are joined.
    const Piece done = cur;
    pos += cur.n;
    const bool more = pos < hi;
    if (more) {
      cur = piece_at(pos);
      if (sw == 0) {
        start_loads(cur);
        for (int i = 0; i < ring; ++i) issue();
      }
    }
    // Key lanes are joined in halves: those of the upper half leave their sums, register by register.
    for (int half = kw / 2; half >= 1; half /= 2) {
      float* place = merge + ((size_t)((kl % half) * sw_n + sw) * S::MERGE_REGS * 32) + lane;
      if (kl >= half && kl < 2 * half) {
        int r = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            place[32 * r++] = ref[n][j];
            place[32 * r++] = l[n][j];
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) place[32 * r++] = oz[gi][n][j];
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              place[32 * r++] = o[i][n][j];
              place[32 * r++] = o[i][n][2 + j];
            }
          }
        }
      }
      __syncthreads();
      if (kl < half) {
        int r = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float other = place[32 * r++];
            const float m = fmaxf(ref[n][j], other);
            const float f0 = ref[n][j] == m ? 1.f : ex2(ref[n][j] - m), f1 = other == m ? 1.f : ex2(other - m);
            ref[n][j] = m;
            l[n][j] = l[n][j] * f0 + place[32 * r++] * f1;
#pragma unroll
            for (int gi = 0; gi < NG; ++gi) oz[gi][n][j] = oz[gi][n][j] * f0 + place[32 * r++] * f1;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              o[i][n][j] = o[i][n][j] * f0 + place[32 * r++] * f1;
              o[i][n][2 + j] = o[i][n][2 + j] * f0 + place[32 * r++] * f1;
            }
          }
        }
      }
      __syncthreads();
    }
    if (kw == 1) __syncthreads();   // the queries are read no more
    if (kl == 0 && busy) {
      // Record: per slot D sums, then reference and l of all slots.
      const size_t rec = (size_t)done.chunk * a.num_kv_heads + done.head + b;
      float* to = a.partial + rec * slots * (D + 2);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int s = (sw * NT + n) * 8 + 2 * t + j;
          float sum = l[n][j];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffff, sum, x);
          if (g == 0 && s < done.count) *reinterpret_cast<float2*>(to + slots * D + 2 * s) = make_float2(ref[n][j], sum);
#pragma unroll
          for (int gi = 0; gi < NG; ++gi) {
            float zz = oz[gi][n][j];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) zz += __shfl_xor_sync(0xffffffff, zz, x);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[2 * i] = fmaf(o[gi * 4 + i][n][j], 0x1p24f, zz);
              v[2 * i + 1] = fmaf(o[gi * 4 + i][n][2 + j], BITS == 4 ? 0x1p20f : 0x1p24f, zz);
            }
            if (s < done.count) {
              float4* to4 = reinterpret_cast<float4*>(to + s * D + gi * GROUP + g * 8);
              to4[0] = make_float4(v[0], v[1], v[2], v[3]);
              to4[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
        }
    }
    if (!more) break;
  }
}

// Joins the records of a (row, kv head): a CTA of 8 warps.  With few records a warp takes a head; with
// many the warps share a head's records.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const QuantAttnArgs a) {
  constexpr int PER = D / 32;
  __shared__ float part[8][D + 2];
  pdl_wait();
  pdl_trigger();
  const Plan plan = plan_of(a);
  const int row = blockIdx.x, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.num_q_heads / a.num_kv_heads;
  const long long total = *plan.total;
  const int B = ctas_of(total, a.grid, 8 / a.slot_warps);
  const int2 where = plan.rows[row];
  const int len = plan.lens[row];
  for (int h0 = 0; h0 < group; ++h0) {
    const int s = (row - where.y) * group + h0;
    Chunk e = {};
    int chunk = 0, n = 0, first = 0;
    if (where.x >= 0) {
      chunk = where.x + s / a.chunk;
      e = plan.table[chunk];
      if (e.stages > 0) {
        const long long p0 = e.before + (long long)kvh * e.stages, p1 = p0 + e.stages - 1;
        first = (int)(((p0 + 1) * B - 1) / total);
        n = (int)(((p1 + 1) * B - 1) / total) - first + 1;
      }
    }
    const bool shared = n > 4;   // the same in all warps
    if (!shared && warp != (h0 & 7)) continue;
    const int at = s % a.chunk;
    const float* rec = a.partial + ((size_t)chunk * a.num_kv_heads + kvh + first) * a.chunk * (D + 2);
    float m = -INFINITY, l = 0.f, o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = 0.f;
    for (int i = shared ? warp : 0; i < n; i += shared ? 8 : 1) {
      const float* from = rec + (size_t)i * a.chunk * (D + 2);
      const float2 ml = *reinterpret_cast<const float2*>(from + a.chunk * D + 2 * at);
      const float mm = fmaxf(m, ml.x);
      const float f0 = m == mm ? 1.f : ex2(m - mm), f1 = ml.x == mm ? 1.f : ex2(ml.x - mm);
      m = mm;
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        const float2 x = *reinterpret_cast<const float2*>(from + at * D + lane * PER + j);
        o[j] = o[j] * f0 + x.x * f1;
        o[j + 1] = o[j + 1] * f0 + x.y * f1;
      }
    }
    if (shared) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < PER; ++j) part[warp][lane * PER + j] = o[j];
      if (lane == 0) {
        part[warp][D] = m;
        part[warp][D + 1] = l;
      }
      __syncthreads();
      if (warp != (h0 & 7)) continue;
      m = -INFINITY;
      for (int i = 0; i < 8; ++i) m = fmaxf(m, part[i][D]);
      l = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] = 0.f;
      for (int i = 0; i < 8; ++i) {
        const float f = part[i][D] == m ? 1.f : ex2(part[i][D] - m);
        l += part[i][D + 1] * f;
#pragma unroll
        for (int j = 0; j < PER; ++j) o[j] += part[i][lane * PER + j] * f;
      }
    }
    // A row without keys gives 0; one whose weights are all 0 (scores of -inf) or NaN gives NaN.
    const int head = kvh * group + h0;
    const float inv = 1.f / l;
    float y[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) y[j] = len > 0 && where.x >= 0 ? o[j] * inv : 0.f;
    if (a.gate != nullptr) {
      const uint16_t* gp = static_cast<const uint16_t*>(a.gate) + (size_t)row * a.gate_row + (size_t)head * a.gate_head + lane * PER;
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        const float2 f = two_floats(*reinterpret_cast<const uint32_t*>(gp + j), a.half);
        y[j] *= sigmoidf_(f.x);
        y[j + 1] *= sigmoidf_(f.y);
      }
    }
    const size_t item = (size_t)row * a.num_q_heads + head;
    if (a.out != nullptr) {
      uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + item * D + lane * PER);
#pragma unroll
      for (int j = 0; j < PER; j += 2) to[j / 2] = two_halves(y[j], y[j + 1], a.half);
    }
    if (a.out_q != nullptr) {
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) big = fmaxf(big, fabsf(y[j]));
#pragma unroll
      for (int x = 1; x < 32 / PER; x <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffff, big, x));
      const uint8_t code = mx_scale_e8m0(big);
      const float si = mx_inv_scale(code);
#pragma unroll
      for (int j = 0; j < PER; ++j) a.out_q[item * D + lane * PER + j] = f32_to_e4m3(y[j] * si);
      if (lane % (32 / PER) == 0) {
        const int kb = (head * D + lane * PER) >> 5;
        a.out_sf[((size_t)(row >> 7) * (a.num_q_heads * D >> 7) + (kb >> 2)) * 512 + sf_atom_offset(row & 127, kb & 3)] = code;
      }
    }
  }
}

int check_rows(const QuantRowsArgs& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return -1;
  if ((a.bits != 4 && a.bits != 8) || a.page_shift < 4 || a.page_shift > 8) return -1;
  if (a.rows < 0 || a.num_kv_heads < 1 || a.num_pages < 1 || a.num_slots < 1 || a.max_pages < 1) return -1;
  return 0;
}

int row_blocks(const QuantRowsArgs& a) {
  const long long items = (long long)a.rows * a.num_kv_heads * 2 * (a.head_dim / 8);
  return (int)((items + ROW_THREADS - 1) / ROW_THREADS);
}

template <int D, int BITS, int NT, int MIN_CTAS>
int launch_attend(QuantAttnArgs a, cudaStream_t stream) {
  using S = Shape<D, BITS, NT>;
  const int kw = WARPS / a.slot_warps;
  const int room = (227 * 1024 / MIN_CTAS - 1024 * (MIN_CTAS > 1)) & ~127;
  a.ring_offset = (S::fixed(a.slot_warps) + 127) & ~127;
  a.ring = (room - a.ring_offset) / (kw * S::STAGE_BYTES);
  if (a.ring > MAX_RING) a.ring = MAX_RING;
  if (a.ring < 1 || a.chunk != S::slots(a.slot_warps)) return -1;
  const int bytes = a.ring_offset + kw * a.ring * S::STAGE_BYTES;
  a.grid = 148 * MIN_CTAS;
  if (a.grid > ZS_QUANT_CTAS) return -1;
  const auto kernel = attend_kernel<D, BITS, NT, MIN_CTAS>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  zs_launch(kernel, a.grid, WARPS * 32, bytes, stream, a);
  zs_launch(join_kernel<D>, dim3(a.rows, a.num_kv_heads), 256, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

int check_attn(const QuantAttnArgs& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return -1;
  if ((a.bits != 4 && a.bits != 8) || a.num_kv_heads < 1 || a.num_q_heads % a.num_kv_heads != 0) return -1;
  if (a.rows < 0 || a.rows > a.max_rows || a.num_seqs < 0 || a.max_seq_rows < 1 || a.work == nullptr) return -1;
  if (a.slot_warps != 1 && a.slot_warps != 2 && a.slot_warps != 4 && a.slot_warps != 8) return -1;
  return 0;
}

}  // namespace qc
}  // namespace zs

extern "C" int zs_quant_block_bytes(int head_dim, int bits) { return zs::qc::block_bytes(head_dim, bits); }

extern "C" int zs_quant_store(const QuantRowsArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_rows(*args)) return e;
  if (args->rows == 0) return 0;
  zs_launch(zs::qc::store_kernel, zs::qc::row_blocks(*args), zs::qc::ROW_THREADS, 0, stream, *args);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_quant_load(const QuantRowsArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_rows(*args)) return e;
  if (args->rows == 0) return 0;
  zs_launch(zs::qc::load_kernel, zs::qc::row_blocks(*args), zs::qc::ROW_THREADS, 0, stream, *args);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// Tiles of 8 slots a warp holds (its sums are D / 4 registers a tile), and the warps that share a key lane.
extern "C" void zs_quant_attn_shape(int head_dim, int slots, int* tiles, int* slot_warps) {
  const int most = head_dim == 256 ? 2 : 4;
  *tiles = 1;
  while (*tiles < most && 8 * *tiles < slots) *tiles *= 2;
  *slot_warps = 1;
  while (*slot_warps < zs::qc::WARPS && 8 * *tiles * *slot_warps < slots) *slot_warps *= 2;
}

extern "C" long long zs_quant_attn_work(int max_chunks, int max_rows, int max_seqs) {
  return 32 + (long long)max_chunks * 32 + (long long)max_rows * 12 + (long long)max_seqs * 4;
}

extern "C" int zs_quant_attn_plan(const QuantAttnArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_attn(*args)) return e;
  zs_launch(zs::qc::plan_kernel, 1, zs::qc::PLAN_THREADS, 0, stream, *args);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_quant_attn(const QuantAttnArgs* args, cudaStream_t stream) {
  using namespace zs::qc;
  const QuantAttnArgs& a = *args;
  if (int e = check_attn(a)) return e;
  if (a.num_pages < 1 || a.num_slots < 1 || a.max_pages < 1 || a.page_shift < 4 || a.page_shift > 8 || a.partial == nullptr) return -1;
  if (a.rows == 0) return 0;
#define ZS_QUANT_CASE(d, bits_, nt, ctas) \
  if (a.head_dim == d && a.bits == bits_ && a.tiles == nt) return launch_attend<d, bits_, nt, ctas>(a, stream);
  ZS_QUANT_CASE(64, 4, 1, 2)
  ZS_QUANT_CASE(64, 4, 2, 2)
  ZS_QUANT_CASE(64, 4, 4, 1)
  ZS_QUANT_CASE(64, 8, 1, 2)
  ZS_QUANT_CASE(64, 8, 2, 2)
  ZS_QUANT_CASE(64, 8, 4, 1)
  ZS_QUANT_CASE(128, 4, 1, 2)
  ZS_QUANT_CASE(128, 4, 2, 1)
  ZS_QUANT_CASE(128, 4, 4, 1)
  ZS_QUANT_CASE(128, 8, 1, 2)
  ZS_QUANT_CASE(128, 8, 2, 1)
  ZS_QUANT_CASE(128, 8, 4, 1)
  ZS_QUANT_CASE(256, 4, 1, 1)
  ZS_QUANT_CASE(256, 4, 2, 1)
  ZS_QUANT_CASE(256, 8, 1, 1)
  ZS_QUANT_CASE(256, 8, 2, 1)
#undef ZS_QUANT_CASE
  return -1;
}
