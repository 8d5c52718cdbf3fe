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
// its own, a warp 512 in a row, and a block is one bulk copy.
//
// Attention.  With q . K_j = sum over groups of s (q . n) + z (sum of q), and the same for
// sum_j p_j V_j = sum_j (p_j s) n_j + p_j z, the whole numbers themselves are the matrix operand:
// (w & 0x000F000F) of a word of eight is two f16 subnormals n 2^-24, exact, and (w & 0x00F000F0) the next two
// times 16.  A pair costs one integer instruction and a part of a shift, and no multiplication; scales go to the
// 32-bit scores and to the weights.  The scaled weights are rounded to f16 (2^-11; for f16 outputs a second
// product takes what that cuts off): the running reference of a row bounds score + log2(scale), so that
// they stay below 2^15 whatever the size of V.
#include <type_traits>

#include "quant_cache.cuh"

namespace zs {
namespace qc {

// Where the 8 numbers of dims d..d+7 (d a multiple of 8) of K's token t are in the block: `bits` bytes.  Rows
// g and g + 8 of a fragment are the tokens 2g and 2g + 1, and four lanes have 16 dims of a group each.
__device__ __forceinline__ int k_offset(int bits, int t, int d) {
  const int lane = (d & 63) >> 4, half = (d >> 3) & 1;
  if (bits == 8) return (d >> 6) * 1024 + (t & 1) * 512 + (t >> 1) * 64 + lane * 16 + half * 8;
  return (d >> 6) * 512 + (t >> 1) * 64 + lane * 16 + (t & 1) * 8 + half * 4;
}
// V is held by fours of tokens: byte t & 3 of a word is token t's.  With 4 bits the 8 dims d..d+7 are a byte
// each two in 4 words in a row, with 8 bits a byte each in 4 words and 4 more 512 bytes on.
__device__ __forceinline__ int v_offset(int bits, int t, int d) {
  return (d >> 6) * (bits * 128) + ((d & 63) >> 3) * 64 + (t >> 2) * 16;
}

__device__ __forceinline__ float bf16_up(float x) {   // x >= 0
  return __uint_as_float((__float_as_uint(x) + 0xFFFFu) & 0xFFFF0000u);
}
__device__ __forceinline__ float bf16_down(float x) {
  const uint32_t u = __float_as_uint(x);
  return __uint_as_float((u >> 31 ? u + 0xFFFFu : u) & 0xFFFF0000u);
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

// Rows go by fours: a warp has one group of 64 dims of four rows, eight dims a lane, and walks every `a.step`-th
// head of K and V.  Eight lanes agree on a group's range by shuffles; four tokens in a row of V leave as words.
// Measured: 6122 rows of 2 heads of 256 dims to 4 bits 10.7 us (1.5 TB/s; three loads in a row before the first
// number, then some 330 instructions for 512 numbers), 24 rows 3.4 us; back to bf16 7.8 us, 100 200 rows of 4 heads of
// 128 dims 65 us (4.0 TB/s).  A warp that takes a range of all rows, groups and heads, with the next places on their
// way, stores no faster (11.8) and loads slower (107), since neighbouring warps then read pages far apart.
constexpr int ROW_WARPS = 8;

struct RowLane {
  int row;         // of the lane
  int gi, first;   // group, first head
};
__device__ __forceinline__ bool row_lane(const QuantRowsArgs& a, int groups, RowLane* r) {
  const int w = blockIdx.x * ROW_WARPS + (threadIdx.x >> 5), share = a.step * groups;
  const int quad = w / share, in = w - quad * share;
  r->first = in / groups;
  r->gi = in - r->first * groups;
  r->row = quad * 4 + ((threadIdx.x & 31) >> 3);
  return quad * 4 < a.rows;
}

template <int BITS>
__global__ void __launch_bounds__(ROW_WARPS * 32) store_kernel(const QuantRowsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, octet = lane & 7, mine = lane >> 3;
  const int groups = a.head_dim / GROUP, heads = a.num_kv_heads;
  RowLane r;
  if (!row_lane(a, groups, &r)) return;
  const int codes = code_bytes(a.head_dim, BITS), head_bytes = block_bytes(a.head_dim, BITS) << (a.page_shift - 4);
  const int d = r.gi * GROUP + octet * 8;
  constexpr float TOP = (1 << BITS) - 1;
  // The first head's numbers are on their way while the rows' places are looked up.
  const uint16_t* k_from = static_cast<const uint16_t*>(a.k) + r.row * a.k_row + d;
  const uint16_t* v_from = static_cast<const uint16_t*>(a.v) + r.row * a.v_row + d;
  auto load = [&](const uint16_t* from, long long stride, int h) {
    return h < heads && r.row < a.rows ? *reinterpret_cast<const uint4*>(from + h * stride) : make_uint4(0, 0, 0, 0);
  };
  uint4 k_next = load(k_from, a.k_head, r.first), v_next = load(v_from, a.v_head, r.first);
  int my_token = 0;
  uint8_t* my_block = r.row < a.rows ? block_at(a, r.row, &my_token) : nullptr;
  const bool there = my_block != nullptr;
  // Four rows that are the four tokens of one word of V's are written as words.
  const long long first = __shfl_sync(0xffffffff, (long long)my_block, 0);
  const int token = __shfl_sync(0xffffffff, my_token, 0);
  const bool whole = __all_sync(0xffffffff, there && (long long)my_block == first && (token & 3) == 0 && my_token == token + mine);
  auto put = [&](auto is_v, const uint4& u, int h) {
    constexpr bool V = decltype(is_v)::value;
    uint8_t* block = my_block + (V ? codes + v_offset(BITS, my_token, d) : k_offset(BITS, my_token, d));
    uint8_t* scales = my_block + 2 * codes + (V ? TOK * groups * 4 : 0) + (my_token * groups + r.gi) * 4;
    const uint32_t word[4] = {u.x, u.y, u.z, u.w};
    float x[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = two_floats(word[j], a.half);
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
    float lo = x[0], hi = x[0], nan = 0.f;   // NaN once a NaN or an infinity has come
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
      nan = fmaf(x[j], 0.f, nan);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffff, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffff, hi, o));
      nan += __shfl_xor_sync(0xffffffff, nan, o);
    }
    const bool fine = nan == 0.f && fmaxf(fabsf(lo), fabsf(hi)) <= 0x1p126f;
    const float z = bf16_down(lo);
    const float s = bf16_up(__fdiv_rn(hi - z, TOP));
    // (x - z) / s rounded as a division rounds, by Markstein's correction of x' times the rounded 1 / s; a power
    // of two keeps 1 / s and the remainder in range.  The sum with 1.5 2^23 rounds it to a whole number, ties to
    // even.  Horner's scheme puts numbers together while they are floats (exact below 2^24).
    const float up = s < 0x1p-64f ? 0x1p100f : 1.f;
    const float su = s * up, inv = s > 0.f ? __frcp_rn(su) : 0.f;
    constexpr int PER = 16 / BITS;   // numbers of 16 bits
    uint32_t n[BITS / 4] = {};
#pragma unroll
    for (int c = 0; c < 8 / PER; ++c) {
      float both = 0.f;
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        const float y = (x[c * PER + j] - z) * up, q0 = y * inv;
        const float q = fminf(fmaf(fmaf(-q0, su, y), inv, q0), TOP);
        both = fmaf(both, TOP + 1.f, (q + 12582912.f) - 12582912.f);
      }
      n[c / 2] |= (__float_as_uint(both + 12582912.f) & 0xFFFFu) << (16 * (c & 1));
    }
    if (!fine) {
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) n[i] = 0;
    }
    const long long at = (long long)h * head_bytes;
    if (!V) {
      if (there) {
        if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(block + at) = n[0];
        else *reinterpret_cast<uint2*>(block + at) = make_uint2(n[0], n[1]);
      }
    } else if (whole) {
      // A four by four exchange of bytes: lane `mine` of a four gets byte `mine` of all four rows.
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) {
        const uint32_t x1 = __shfl_xor_sync(0xffffffff, n[i], 8);
        const uint32_t y = mine & 1 ? __byte_perm(x1, n[i], 0x7351) : __byte_perm(n[i], x1, 0x6240);   // bytes b, b + 2 of two rows
        const uint32_t x2 = __shfl_xor_sync(0xffffffff, y, 16);
        const uint32_t all = mine & 2 ? __byte_perm(x2, y, 0x7632) : __byte_perm(y, x2, 0x5410);
        *reinterpret_cast<uint32_t*>(block + at + i * 512 + mine * 4) = all;
      }
    } else if (there) {
      uint8_t* to = block + at + (my_token & 3);
#pragma unroll
      for (int j = 0; j < BITS; ++j) to[(j >> 2) * 512 + (j & 3) * 4] = (uint8_t)(n[j >> 2] >> (8 * (j & 3)));
    }
    // A constant group (s = 0) is z whatever its scale: with |z| 2^-17 no scale is below 2^-19 of its offset, and the
    // attention sees from the scales alone how large V is.
    const float held = s > 0.f ? s : fabsf(z) * 0x1p-17f;
    if (octet == 0 && there) *reinterpret_cast<uint32_t*>(scales + at) = fine ? __float_as_uint(held) >> 16 | __float_as_uint(z) : POISON;
  };
  for (int h = r.first; h < heads; h += a.step) {
    const uint4 k = k_next, v = v_next;
    k_next = load(k_from, a.k_head, h + a.step);
    v_next = load(v_from, a.v_head, h + a.step);
    put(std::false_type(), k, h);
    put(std::true_type(), v, h);
  }
}

template <int BITS>
__global__ void __launch_bounds__(ROW_WARPS * 32) load_kernel(const QuantRowsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, octet = lane & 7;
  const int groups = a.head_dim / GROUP, heads = a.num_kv_heads;
  RowLane r;
  if (!row_lane(a, groups, &r)) return;
  if (r.row >= a.rows) return;
  const int codes = code_bytes(a.head_dim, BITS), head_bytes = block_bytes(a.head_dim, BITS) << (a.page_shift - 4);
  const int d = r.gi * GROUP + octet * 8;
  int token = 0;
  const uint8_t* block = block_at(a, r.row, &token);
  const bool there = block != nullptr;
  const uint32_t pick = (token & 3) * 0x11 + 0x40;   // this token's byte of two words
  const uint8_t* k_from = block + k_offset(BITS, token, d);
  const uint8_t* v_from = block + codes + v_offset(BITS, token, d);
  const uint8_t* scales = block + 2 * codes + (token * groups + r.gi) * 4;
  const long long k_to = r.row * a.k_row + d, v_to = r.row * a.v_row + d;
  auto put = [&](void* out, long long to, const uint32_t (&n)[BITS / 4], uint32_t sz) {
    const float s = scale_of(sz), z = offset_of(sz);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // a byte below 0x4B0000 is 2^23 + n
      const uint32_t bytes = BITS == 8 ? n[(j >> 2) % (BITS / 4)] : j & 1 ? (n[0] >> 4) & 0x0F0F0F0Fu : n[0] & 0x0F0F0F0Fu;
      const int at = BITS == 8 ? j & 3 : j >> 1;
      x[j] = fmaf(__uint_as_float(__byte_perm(bytes, 0x4B000000u, 0x7440 + at)) - 8388608.f, s, z);
    }
    if (a.f32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + to);
      o[0] = make_float4(x[0], x[1], x[2], x[3]);
      o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + to) =
          make_uint4(two_halves(x[0], x[1], a.half), two_halves(x[2], x[3], a.half), two_halves(x[4], x[5], a.half), two_halves(x[6], x[7], a.half));
    }
  };
  constexpr int AT_ONCE = 4;   // heads whose loads are on their way together
  for (int h0 = r.first; h0 < heads; h0 += AT_ONCE * a.step) {
    uint32_t n[AT_ONCE][BITS / 4] = {}, k_sz[AT_ONCE] = {}, v_sz[AT_ONCE] = {};
    uint4 u[AT_ONCE][BITS / 4] = {};
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int h = h0 + i * a.step;
      if (h >= heads || !there) continue;
      const long long at = (long long)h * head_bytes;
      k_sz[i] = *reinterpret_cast<const uint32_t*>(scales + at);
      v_sz[i] = *reinterpret_cast<const uint32_t*>(scales + at + TOK * groups * 4);
      if constexpr (BITS == 4) {
        n[i][0] = *reinterpret_cast<const uint32_t*>(k_from + at);
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(k_from + at);
        n[i][0] = x.x;
        n[i][BITS / 4 - 1] = x.y;
      }
#pragma unroll
      for (int k = 0; k < BITS / 4; ++k) u[i][k] = *reinterpret_cast<const uint4*>(v_from + at + k * 512);
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int h = h0 + i * a.step;
      if (h >= heads) break;
      put(const_cast<void*>(a.k), k_to + h * a.k_head, n[i], k_sz[i]);
      uint32_t v[BITS / 4];
#pragma unroll
      for (int k = 0; k < BITS / 4; ++k) v[k] = __byte_perm(__byte_perm(u[i][k].x, u[i][k].y, pick), __byte_perm(u[i][k].z, u[i][k].w, pick), 0x5410);
      put(const_cast<void*>(a.v), v_to + h * a.v_head, v, v_sz[i]);
    }
  }
}

// ------------------------------------------------------------------------------------ plan
// A query slot is one (row, q head of the kv head's group) of a sequence; up to `a.chunk` slots of one
// sequence and kv head are a unit, and its keys are walked in stages of 16, 32 or 64.  The chunks (units of all
// kv heads at once) stand in a table with the number of stages before them; CTA b of the attention
// takes the stages [b T / B, (b + 1) T / B) of all T, so that every CTA has the same work whatever the
// lengths.  One CTA of 1024 threads plans (4 us for one sequence, 5.5 for 256: loads that wait for one another);
// a step's layers share the plan.
constexpr int PLAN_THREADS = 1024, MAX_LENGTH = 1 << 30;

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

__device__ __forceinline__ int length_of(const QuantAttnArgs& a, int row) {
  const int n = a.seq_lens[row];
  if (n > MAX_LENGTH) {
    report_error(a.err, kErrBadShape);
    return 0;
  }
  return max(n, 0);
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
    p.lens[r] = length_of(a, r);
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
        e.len = max(e.len, p.lens[r]);
        // A row whose slots are in two chunks is entered by both, with the same numbers.
        p.rows[r] = make_int2(p.offset[lo], r0);
      }
      e.stages = (e.len + a.stage - 1) / a.stage;
    }
    const long long cost = (long long)e.stages * a.num_kv_heads;
    e.before = base + block_scan(cost, warps, &all);
    if (c < chunks) p.table[c] = e;
    base += all;
  }
  __syncthreads();
  const int ctas = base > 0 ? ctas_of(base, a.grid, a.least) : 0;
  for (int b = threadIdx.x; b < ctas; b += PLAN_THREADS) {
    const long long first = base * b / ctas;
    int lo = 0, hi = chunks;   // the last chunk that starts at or before it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (p.table[mid].before <= first) lo = mid;
      else hi = mid;
    }
    p.start[b] = lo;
  }
  if (threadIdx.x == 0) {
    p.total[0] = base;
    p.total[1] = a.rows;
  }
}

// ------------------------------------------------------------------------------- attention
constexpr int MAX_RING = 8;
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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

// A variant: head dim, bits, tiles of 8 slots of a warp, warps of a CTA, blocks of 16 keys of a stage,
// CTAs of an SM, and whether the weights keep what f16 cuts off (f16 outputs).
template <int D_, int BITS_, int NT_, int WARPS_, int KB_, int CTAS_, bool FINE_>
struct Shape {
  static constexpr int D = D_, BITS = BITS_, NT = NT_, WARPS = WARPS_, KB = KB_, CTAS = CTAS_;
  static constexpr bool FINE = FINE_;
  // V's numbers all times 16 (see fold_offsets); elsewhere every second one of 4 bits.  What a sum is then multiplied by.
  static constexpr bool HIGH = FINE && BITS == 4;
  static constexpr float EVEN = HIGH ? 0x1p44f : 0x1p48f, ODD = BITS == 4 ? 0x1p44f : 0x1p48f;
  static constexpr int FOLD = FINE ? 1 : 8;         // stages between additions of the offsets' sums
  static constexpr int KS = D / 16;                 // tiles of 16 dims of V
  static constexpr int NG = D / GROUP;
  static constexpr int CODES = code_bytes(D, BITS);
  static constexpr int BLOCK = block_bytes(D, BITS);
  static constexpr int KEYS = KB * TOK;             // of a stage
  static constexpr int STAGE_BYTES = KB * BLOCK;
  static constexpr int SLOTS = 8 * NT;
  // Queries: a lane has 8 dims of a slot, so a warp has 1, 2 or 4 slots at a time.
  static constexpr int Q_LANES = D / 8, Q_EACH = 32 / Q_LANES, Q_PASSES = (SLOTS + WARPS * Q_EACH - 1) / (WARPS * Q_EACH);
  // The join of the warps, a tile of 8 slots at a time: its items are (group, column), of 8 sums of V and one of the offsets
  // a lane, and every warp but an item's owner leaves its own.
  static constexpr int ITEMS = 2 * NG, ITEM = 9;
  static constexpr int JOIN = ITEMS * (WARPS - 1) * ITEM * 128;
  static constexpr int BARS = WARPS * MAX_RING * 8;
  static constexpr int FIXED = BARS + SLOTS * (NG + 2) * 4 + KS * NT * 256 + 3 * WARPS * SLOTS * 4 + JOIN;
};

struct Piece {
  int chunk, head, first, n;   // stages [first, first + n) of the unit
  int row, slot, slot0, count, len;
};

// What a warp holds of its slots: column j of tile n is slot 8 n + 2 t + j, and register r of a sum is
// one of its dims (g's).
template <class S>
struct State {
  float o[S::KS][S::NT][4], oz[S::NG][S::NT][2], l[S::NT][2];
  float ref[S::NT][2], lift[S::NT][2];   // the reference's score, and LIFT + ABOVE minus its rest
  float fac[S::NT][2];
  int lens[S::NT][2];
};

// Sequences with few slots.  S^T = K Q^T and O^T += V^T P^T on m16n8k16 (a tile of 8 slots is the narrow side, so
// that 8 slots waste nothing), every warp at its own stages of its own ring of bulk copies: no warp waits for
// another before the end of a piece.  Measured with the join: 256 sequences of up to 1280 keys, 16 q heads on 2 kv heads
// of 256 dims, 4 bits 52 us (2.8 TB/s); 61 sequences of up to 4001 keys, 8 heads of 128 dims, 8 bits 72 us (5.6 TB/s); 7
// sequences of up to 65 535 keys, 32 on 4 heads of 128 dims, 4 bits, f16 61.5 us (3.5 TB/s).  With 8 bits it is bound by memory.
// With 4 bits no unit is full (issue slots 50 %, tensor pipe 20 %, DRAM 38 %): the 11 warps that an SM has room for, at 164
// registers, issue an instruction every 5.5 cycles each, of which 1.4 wait for the one before, 0.6 for another warp's turn, 0.5
// for shared memory and 0.4 each for the math pipes, the join's barriers and the instructions themselves.  e4m3 products for K
// are emulated here and took 61 -> 70 us; smaller CTAs, and warps of their own for the copies, were no faster.
//
// One stage: the scores of its keys, their weights, and what they add to the sums.  With MASK a key at or
// behind a slot's length is left out whatever the cache holds there.
template <class S, bool MASK>
__device__ __forceinline__ void stage_step(State<S>& st, const uint8_t* in, const uint8_t* qf, const float* qsum, int key0, int g,
                                           int t) {
  constexpr int NT = S::NT, NG = S::NG, KS = S::KS, KB = S::KB, BITS = S::BITS;
  float sc[KB][NT][4];
  uint32_t sz[KB][2 * NG];   // of tokens 2g and 2g + 1, which are rows g and g + 8 of a fragment
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) lds(sz[kb], in + kb * S::BLOCK + 2 * S::CODES + g * NG * 8);
  // Groups are walked side by side (GB at a time): every chain of four products then has others between its links.
  constexpr int GB = NG * KB * NT <= 4 ? NG : NG * KB * NT <= 8 ? (NG + 1) / 2 : 1;
#pragma unroll
  for (int g0 = 0; g0 < NG; g0 += GB) {
    uint32_t w[GB][KB][BITS];
#pragma unroll
    for (int gi = 0; gi < GB; ++gi)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < BITS / 4; ++r) {
          uint32_t u[4];
          lds(u, in + kb * S::BLOCK + (g0 + gi) * (BITS * 128) + r * 512 + (g * 4 + t) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) w[gi][kb][4 * r + j] = u[j];
        }
    float acc[GB][KB][NT][4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int gi = 0; gi < GB; ++gi) {
        uint32_t bq[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) lds(bq[n], qf + (((g0 + gi) * 4 + k) * NT + n) * 256);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t a0, a1, a2, a3;   // rows g and g + 8
          if (BITS == 4) {
            const uint32_t x = w[gi][kb][k >> 1] >> (8 * (k & 1)), y = w[gi][kb][2 + (k >> 1)] >> (8 * (k & 1));
            a0 = x & 0x000F000Fu;
            a1 = y & 0x000F000Fu;
            a2 = x & 0x00F000F0u;
            a3 = y & 0x00F000F0u;
          } else {
            const uint32_t x = w[gi][kb][k], y = w[gi][kb][(4 + k) % BITS];
            a0 = x & 0x00FF00FFu;
            a1 = y & 0x00FF00FFu;
            a2 = (x >> 8) & 0x00FF00FFu;
            a3 = (y >> 8) & 0x00FF00FFu;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (k == 0) mma16816_first(acc[gi][kb][n], a0, a1, a2, a3, bq[n][0], bq[n][1]);
            else mma16816(acc[gi][kb][n], a0, a1, a2, a3, bq[n][0], bq[n][1]);
          }
        }
      }
#pragma unroll
    for (int gi = 0; gi < GB; ++gi)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 qs = *reinterpret_cast<const float2*>(qsum + (g0 + gi) * S::SLOTS + n * 8 + 2 * t);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = sz[kb][(j >> 1) * NG + g0 + gi];
            const float y = j & 1 ? qs.y : qs.x;
            sc[kb][n][j] = fmaf(scale_of(x), acc[gi][kb][n][j], g0 + gi == 0 ? offset_of(x) * y : fmaf(offset_of(x), y, sc[kb][n][j]));
          }
      }
  }
  // V's scales: the largest exponent among this lane's keys bounds them all, and tells whether a reference may have to
  // move.  The bits of a scale grow with it; a poisoned one is negative.
  constexpr int FLOOR = 0x1F800000;   // 2^-64
  const auto exponent = [](int bits) { return __uint_as_float(0x4B000000u | (uint32_t)(bits >> 23)) - (8388608.f + 127.f); };
  int top = FLOOR;
  int longest = 0;
  if (MASK) {   // what stands behind the sequence may be anything
#pragma unroll
    for (int n = 0; n < NT; ++n) longest = max(longest, max(st.lens[n][0], st.lens[n][1]));
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    lds(sz[kb], in + kb * S::BLOCK + 2 * S::CODES + TOK * NG * 4 + g * NG * 8);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int gi = 0; gi < NG; ++gi)
        if (!MASK || key0 + kb * 16 + 2 * g + r < longest) top = max(top, (int)(sz[kb][r * NG + gi] << 16));
  }
  const float ex = exponent(top);
  bool move = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float m = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = sc[kb][n][2 * r + j] * st.fac[n][j];
          if (MASK && key0 + kb * 16 + 2 * g + r >= st.lens[n][j]) x = -INFINITY;
          sc[kb][n][2 * r + j] = x;
          m = fmaxf(m, x);
        }
      move = move || (m - st.ref[n][j]) + (ex + st.lift[n][j]) > LIFT + ABOVE + SLACK;
    }
  if (__any_sync(0xffffffff, move)) {
    // A slot's reference moves for what the slot sees, every key with its own exponent: a large value that it does not see,
    // or that has no weight, leaves the others their bits.
    float own[KB][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        int x = FLOOR;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) x = max(x, (int)(sz[kb][r * NG + gi] << 16));
        own[kb][r] = exponent(x);
      }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // fmaxf takes no NaN: -inf - -inf, where neither a key nor a reference is there.
        const auto most = [&](float from, bool with_own) {
          float m = -INFINITY;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 2; ++r) m = fmaxf(m, (sc[kb][n][2 * r + j] - from) + (with_own ? own[kb][r] : 0.f));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffff, m, x));
          return m;
        };
        const float at = st.ref[n][j], lift = st.lift[n][j];
        const float to = fmaxf(at, most(0.f, false)), rest = most(to, true);
        const bool grow = (to - at) + (rest + lift) > LIFT + ABOVE + SLACK;
        const float to_lift = fminf(lift + (to - at), LIFT + ABOVE - rest);
        const float f = grow ? ex2((at - to) + (to_lift - lift)) : 1.f;
        if (grow) {
          st.ref[n][j] = to;
          st.lift[n][j] = to_lift;
        }
        st.l[n][j] *= f;
#pragma unroll
        for (int gi = 0; gi < NG; ++gi) st.oz[gi][n][j] *= f;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          st.o[i][n][j] *= f;
          st.o[i][n][2 + j] *= f;
        }
      }
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // A masked score is -inf; where the reference still is too, the difference would be NaN.
        float p = ex2((sc[kb][n][j] - st.ref[n][j & 1]) + st.lift[n][j & 1]);
        if (MASK && key0 + kb * 16 + 2 * g + (j >> 1) >= st.lens[n][j & 1]) p = 0.f;
        sc[kb][n][j] = p;
        st.l[n][j & 1] += p;
      }
    float low[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) low[n][j] = sc[kb][n][j] * BELOW;
#pragma unroll
    for (int gi = 0; gi < NG; ++gi) {
      // V's numbers of the tokens 4t..4t+3 (columns 2t, 2t + 8, 2t + 1 and 2t + 9 of a fragment) for this lane's
      // 8 dims of the group, which are rows g and g + 8 of four tiles.
      uint32_t u[BITS];
#pragma unroll
      for (int h = 0; h < BITS / 4; ++h) {
        uint32_t x[4];
        lds(x, in + kb * S::BLOCK + S::CODES + gi * (BITS * 128) + h * 512 + (g * 4 + t) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[4 * h + j] = x[j];
      }
      uint32_t bp[NT][2], bl[NT][2], f[4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float ps[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = sz[kb][(j >> 1) * NG + gi];
          ps[j] = low[n][j] * scale_of(x);
          float& oz = st.oz[gi][n][j & 1];
          if (MASK) {   // nothing of a masked key, NaN among it, is taken
            const bool out = key0 + kb * 16 + 2 * g + (j >> 1) >= st.lens[n][j & 1];
            ps[j] = out ? 0.f : ps[j];
            oz = out ? oz : fmaf(sc[kb][n][j], offset_of(x), oz);
          } else {
            oz = fmaf(sc[kb][n][j], offset_of(x), oz);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t hi = pack_f16(ps[2 * h], ps[2 * h + 1]);
          bp[n][h] = transpose8x8(hi);
          if (S::FINE) {
            const float2 cut = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            bl[n][h] = transpose8x8(pack_f16(ps[2 * h] - cut.x, ps[2 * h + 1] - cut.y));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a0, a1, a2, a3;
        if (S::HIGH) {
          const uint32_t x = u[i];
          a0 = (x << 4) & 0x00F000F0u;
          a1 = x & 0x00F000F0u;
          a2 = (x >> 4) & 0x00F000F0u;
          a3 = (x >> 8) & 0x00F000F0u;
        } else if (BITS == 4) {
          const uint32_t x = u[i], y = u[i] >> 8;
          a0 = x & 0x000F000Fu;
          a1 = x & 0x00F000F0u;
          a2 = y & 0x000F000Fu;
          a3 = y & 0x00F000F0u;
        } else {
          const uint32_t x = u[(2 * i) % BITS], y = u[(2 * i + 1) % BITS];
          a0 = x & 0x00FF00FFu;
          a1 = y & 0x00FF00FFu;
          a2 = (x >> 8) & 0x00FF00FFu;
          a3 = (y >> 8) & 0x00FF00FFu;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816(st.o[gi * 4 + i][n], a0, a1, a2, a3, bp[n][0], bp[n][1]);
        if (S::FINE) {   // a tile behind, so that its sum's last product has left the pipe
          if (i > 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(st.o[gi * 4 + i - 1][n], f[0], f[1], f[2], f[3], bl[n][0], bl[n][1]);
          }
          if (i == 3) {
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(st.o[gi * 4 + 3][n], a0, a1, a2, a3, bl[n][0], bl[n][1]);
          }
          f[0] = a0;
          f[1] = a1;
          f[2] = a2;
          f[3] = a3;
        }
      }
    }
  }
}

// The numbers of V are not negative, so that their sums grow with the keys, and the offsets' sums take most of that away
// again in the end.  The products cut what they add to a sum behind some 24 bits, always towards zero, which leaves a bias that
// the keys add up.  It has two parts, measured for f16 outputs over 65 535 keys as multiples of the outputs' own rounding:
// how large the sums are when they are added to, so the offsets' sums are added every FOLD stages, while both are small (2.2
// without, 1.5 every 8 stages, 1.17 every 2, 1.11 every one); and how the products are lined up, by their operands' exponent
// fields, which for 4-bit numbers as subnormals n 2^-24 are up to 10 bits above them: the low bits of a sum were lost for every
// dim whose numbers are taken as they are (1.9 for these, 1.004 for those times 16).  f16 outputs take all of V's numbers times 16
// (1.007 altogether; 64.6 -> 66.5 us for 7 sequences).  For bf16 outputs, whose rounding is eight times as large, FOLD 8 and the
// cheaper form are enough (1.01).
template <class S>
__device__ __forceinline__ void fold_offsets(State<S>& st) {
#pragma unroll
  for (int gi = 0; gi < S::NG; ++gi)
#pragma unroll
    for (int n = 0; n < S::NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float zz = st.oz[gi][n][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) zz += __shfl_xor_sync(0xffffffff, zz, x);
        st.oz[gi][n][j] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          st.o[gi * 4 + i][n][j] = fmaf(zz, 1.f / S::EVEN, st.o[gi * 4 + i][n][j]);
          st.o[gi * 4 + i][n][2 + j] = fmaf(zz, 1.f / S::ODD, st.o[gi * 4 + i][n][2 + j]);
        }
      }
}

template <class S>
__global__ void __launch_bounds__(S::WARPS * 32, S::CTAS) attend_kernel(const QuantAttnArgs a) {
  constexpr int KS = S::KS, NG = S::NG, NT = S::NT, D = S::D, BITS = S::BITS, BLOCK = S::BLOCK, WARPS = S::WARPS, KB = S::KB, SLOTS = S::SLOTS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Piece pieces[2];
  pdl_wait();
  pdl_trigger();
  const Plan plan = plan_of(a);
  const long long total = stages_of(plan, a);
  int chunk = plan.start[blockIdx.x];   // of the CTA's first stage
  const int ring = a.ring, B = ctas_of(total, gridDim.x, a.least), b = blockIdx.x;
  if (b >= B || total == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int group = a.num_q_heads / a.num_kv_heads;

  uint64_t* full = reinterpret_cast<uint64_t*>(smem) + warp * MAX_RING;
  float* qsum = reinterpret_cast<float*>(smem + S::BARS);         // [NG][SLOTS]
  float* qfac = qsum + NG * SLOTS;                                // [SLOTS]
  int* qlen = reinterpret_cast<int*>(qfac + SLOTS);               // [SLOTS]
  uint8_t* qfrag = reinterpret_cast<uint8_t*>(qlen + SLOTS);      // [KS][NT][32 lanes][8 bytes]
  float* refs = reinterpret_cast<float*>(qfrag + KS * NT * 256);  // [WARPS][SLOTS] score of the reference, its rest, l
  float* sums = refs + 3 * WARPS * SLOTS;                         // [ITEMS][WARPS - 1][ITEM][32]
  uint8_t* stage0 = smem + a.ring_offset + warp * ring * S::STAGE_BYTES;

  // The CTA's stages go piece by piece; the walker is the one thread that looks the next one up (n = 0: none).
  const long long hi = total * (b + 1) / B;
  long long pos = total * b / B;
  const bool walker = threadIdx.x == 32;
  // A plan for units of more slots, in longer stages, is walked by a row of CTAs for each SLOTS of a unit.
  const int part = blockIdx.y * SLOTS, per_stage = a.stage / S::KEYS;
  auto walk = [&](Piece* p) {
    Piece x = {};
    while (pos < hi && x.n == 0) {
      Chunk e = plan.table[chunk];
      while (e.before + (long long)e.stages * a.num_kv_heads <= pos) e = plan.table[++chunk];
      const int r = (int)(pos - e.before), first = r % e.stages, n = (int)min((long long)(e.stages - first), hi - pos);
      pos += n;
      if (e.count <= part) continue;
      x.chunk = chunk;
      x.head = r / e.stages;
      x.first = first * per_stage;
      x.n = min((first + n) * per_stage, (e.len + S::KEYS - 1) / S::KEYS) - x.first;
      x.row = e.row;
      x.slot = e.slot;
      x.slot0 = e.first + part;
      x.count = min(SLOTS, e.count - part);
      x.len = e.len;
    }
    *p = x;
  };
  if (walker) walk(&pieces[0]);
  if (lane == 0) {
    for (int j = 0; j < ring; ++j) mbar_init(&full[j], 1);
    fence_barrier_init();
  }
  __syncthreads();

  // Each warp loads for itself.  Lane j holds where block j % KB of stage j / KB is.
  constexpr int AHEAD = 32 / KB;
  int at_block = 0, at_next = 0, issued = 0, fill = 0, src_n = 0;   // stages issued and in all of the piece that is loaded
  Piece src;
  const int bshift = a.page_shift - 4;
  auto page_ids = [&](int i0) {   // raw, so that nothing waits for it here
    const int i = i0 + lane / KB;
    const int blk = (src.first + warp + i * WARPS) * KB + lane % KB;
    if (i >= src_n || blk * TOK >= src.len) return INT_MIN;
    const int index = blk >> bshift;
    if (src.slot < 0 || src.slot >= a.num_slots || index >= a.max_pages) return -1;
    return a.page_table[(size_t)src.slot * a.max_pages + index];
  };
  auto blocks_of = [&](int page, int i0) {   // -1: behind the sequence's end
    if (page == INT_MIN) return -1;
    if (page < 0 || page >= a.num_pages) {
      report_error(a.err, kErrBadShape);
      page = 0;
    }
    const int blk = (src.first + warp + (i0 + lane / KB) * WARPS) * KB + lane % KB;
    return ((page * a.num_kv_heads + src.head) << bshift) + (blk & ((1 << bshift) - 1));
  };
  auto issue = [&]() {   // the next stage of the piece into the place that was read last
    if (issued >= src_n) return;
    const int k = issued % AHEAD * KB;
    const int b0 = __shfl_sync(0xffffffff, at_block, k);
    const int b1 = KB == 2 ? __shfl_sync(0xffffffff, at_block, (k + 1) & 31) : -1;
    if (lane == 0) {
      uint8_t* to = stage0 + fill * S::STAGE_BYTES;
      mbar_expect_tx(&full[fill], b1 >= 0 ? 2 * BLOCK : BLOCK);
      bulk_load(to, a.data + (size_t)(unsigned)b0 * BLOCK, BLOCK, &full[fill]);
      if (b1 >= 0) bulk_load(to + BLOCK, a.data + (size_t)(unsigned)b1 * BLOCK, BLOCK, &full[fill]);
    }
    if (++fill == ring) fill = 0;
    if (++issued % AHEAD == 0 && issued < src_n) {
      at_block = blocks_of(at_next, issued);
      at_next = page_ids(issued + AHEAD);
    }
  };

  // Queries: slot and first dim of the lane in a pass.
  const int q_slot = warp * S::Q_EACH + lane / S::Q_LANES, q_dim = lane % S::Q_LANES * 8;
  uint4 q_raw[S::Q_PASSES];
  int q_len[S::Q_PASSES];
  // The page ids, the queries and their lengths of a piece are asked for together, then its first stages.
  auto start = [&](const Piece& p) {
    src = p;
    src_n = p.n > warp ? (p.n - warp + WARPS - 1) / WARPS : 0;
    issued = 0;
    const int now = page_ids(0);
    at_next = src_n > AHEAD ? page_ids(AHEAD) : INT_MIN;
#pragma unroll
    for (int x = 0; x < S::Q_PASSES; ++x) {
      const int s = q_slot + x * WARPS * S::Q_EACH, id = p.slot0 + s, row = p.row + id / group;
      const bool real = s < p.count;
      q_raw[x] = real ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (size_t)row * a.q_row +
                                                         (size_t)(p.head * group + id % group) * a.q_head + q_dim)
                      : make_uint4(0, 0, 0, 0);
      q_len[x] = real ? plan.lens[row] : p.len;
    }
    at_block = blocks_of(now, 0);
    for (int i = 0; i < ring; ++i) issue();
  };

  int use = 0, use_phase = 0;   // the ring's place to be read
  Piece cur = pieces[0];
  if (cur.n == 0) return;   // none of the CTA's units has so many slots
  start(cur);
  for (int k = 0;; ++k) {
    if (walker) walk(&pieces[(k + 1) & 1]);
    // A power of two brings a slot's numbers to [2^13, 2^14), where f16 is exact down to 2^-27 of the largest; the numbers
    // that meet w & 0x00F000F0 are divided by 16.
#pragma unroll
    for (int y = 0; y < S::Q_PASSES; ++y) {
      const int s = q_slot + y * WARPS * S::Q_EACH;
      const uint32_t w[4] = {q_raw[y].x, q_raw[y].y, q_raw[y].z, q_raw[y].w};
      float x[8], big = 0.f, nan = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = two_floats(w[j], a.half);
        x[2 * j] = f.x;
        x[2 * j + 1] = f.y;
        big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
        nan = fmaf(f.x, 0.f, fmaf(f.y, 0.f, nan));
      }
      if (nan != 0.f) big = INFINITY;
#pragma unroll
      for (int o = 1; o < S::Q_LANES; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffff, big, o));
      const int e = 13 - min(max((int)(__float_as_uint(big) >> 23) - 127, -100), 100);
      const float up = big < MAX_QUERY ? __uint_as_float((uint32_t)(e + 127) << 23) : NAN;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] *= up;
        sum += x[j];
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
      if (s < SLOTS) {
        const int gi = q_dim >> 6, word = q_dim >> 3 & 1, ln = (s & 7) * 4 + ((q_dim & 63) >> 4);
        if ((q_dim & 63) == 0) qsum[gi * SLOTS + s] = sum * 0x1p-24f;
        if (q_dim == 0) {
          qfac[s] = a.sm_scale * 1.4426950408889634f * __uint_as_float((uint32_t)(24 - e + 127) << 23);
          qlen[s] = q_len[y];
        }
        // Steps 2 word and 2 word + 1 of the group have these dims: with 4 bits numbers 0, 4 (1, 5 times 16) and 2, 6 (3, 7) of a
        // word, with 8 bits 0, 2 (1, 3) of two words.
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          uint2 f;
          if (BITS == 4) f = make_uint2(pack_f16(x[2 * z], x[2 * z + 4]), pack_f16(x[2 * z + 1] * 0.0625f, x[2 * z + 5] * 0.0625f));
          else f = make_uint2(pack_f16(x[4 * z], x[4 * z + 2]), pack_f16(x[4 * z + 1], x[4 * z + 3]));
          *reinterpret_cast<uint2*>(qfrag + (((gi * 4 + word * 2 + z) * NT + (s >> 3)) * 32 + ln) * 8) = f;
        }
      }
    }
    __syncthreads();

    State<S> st;
    int shortest = INT_MAX;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int i = 0; i < KS; ++i) st.o[i][n][j] = st.o[i][n][2 + j] = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) st.oz[i][n][j] = 0.f;
        st.l[n][j] = 0.f;
        st.ref[n][j] = -INFINITY;
        st.lift[n][j] = LIFT + ABOVE;
        st.lens[n][j] = qlen[n * 8 + 2 * t + j];
        st.fac[n][j] = qfac[n * 8 + 2 * t + j];
        shortest = min(shortest, st.lens[n][j]);
      }
    shortest = __reduce_min_sync(0xffffffff, shortest);

    const int n_mine = src_n;
    for (int it = 0; it < n_mine; ++it) {
      mbar_wait(&full[use], use_phase, a.err);
      const uint8_t* in = stage0 + use * S::STAGE_BYTES;
      const int key0 = (cur.first + warp + it * WARPS) * S::KEYS;
      if (key0 + S::KEYS <= shortest) stage_step<S, false>(st, in, qfrag + lane * 8, qsum, key0, g, t);
      else stage_step<S, true>(st, in, qfrag + lane * 8, qsum, key0, g, t);
      __syncwarp();
      if (++use == ring) {
        use = 0;
        use_phase ^= 1;
      }
      issue();
      if (it % S::FOLD == S::FOLD - 1) fold_offsets(st);
    }

    // The next piece's first stages are on their way while this one's warps are joined.
    const Piece done = cur;
    cur = pieces[(k + 1) & 1];
    if (cur.n > 0) start(cur);
    // All warps' sums of a slot are brought to the largest reference and added by an item's owner, which also writes them.
    const size_t rec = (size_t)done.chunk * a.num_kv_heads + done.head + b;
    float* to = a.partial + rec * a.chunk * (D + RECORD_REST) + part * D;
    float* to_rest = a.partial + rec * a.chunk * (D + RECORD_REST) + a.chunk * D + part * RECORD_REST;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = st.l[n][j];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffff, l, x);
        if (g == 0) {
          float* mine = refs + warp * SLOTS + n * 8 + 2 * t + j;
          mine[0] = st.ref[n][j];
          mine[WARPS * SLOTS] = -st.lift[n][j];
          mine[2 * WARPS * SLOTS] = l;
        }
      }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int s = n * 8 + 2 * t + j;
        const auto of_warp = [&](int w) { return Reference{refs[w * SLOTS + s], refs[(WARPS + w) * SLOTS + s]}; };
        Reference top{LOWEST, LOWEST};
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top.score = fmaxf(top.score, of_warp(w).score);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top.rest = fmaxf(top.rest, (of_warp(w).score - top.score) + of_warp(w).rest);
        f[j] = factor_to(Reference{st.ref[n][j], -st.lift[n][j]}, top);
        if (warp == 0 && g == 0 && s < done.count) {
#pragma unroll
          for (int w = 0; w < WARPS; ++w) l += refs[(2 * WARPS + w) * SLOTS + s] * factor_to(of_warp(w), top);
          *reinterpret_cast<float4*>(to_rest + RECORD_REST * s) = make_float4(top.score, top.rest, l, 0.f);
        }
      }
      if (n > 0) __syncthreads();   // the tile before has been added up
#pragma unroll
      for (int item = 0; item < S::ITEMS; ++item) {
        const int gi = item >> 1, j = item & 1, owner = item % WARPS;
        if (owner == warp) continue;
        float* out = sums + ((item * (WARPS - 1) + (warp < owner ? warp : warp - 1)) * S::ITEM) * 32 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          out[64 * i] = st.o[gi * 4 + i][n][j] * f[j];
          out[64 * i + 32] = st.o[gi * 4 + i][n][2 + j] * f[j];
        }
        out[256] = st.oz[gi][n][j] * f[j];
      }
      __syncthreads();
#pragma unroll
      for (int item = 0; item < S::ITEMS; ++item) {
        const int gi = item >> 1, j = item & 1, s = n * 8 + 2 * t + j;
        if (item % WARPS != warp) continue;
        float v[8], zz = st.oz[gi][n][j] * f[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = st.o[gi * 4 + i][n][j] * f[j];
          v[2 * i + 1] = st.o[gi * 4 + i][n][2 + j] * f[j];
        }
        const float* in = sums + item * (WARPS - 1) * S::ITEM * 32 + lane;
#pragma unroll
        for (int w = 0; w < WARPS - 1; ++w) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += in[(w * S::ITEM + i) * 32];
          zz += in[(w * S::ITEM + 8) * 32];
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) zz += __shfl_xor_sync(0xffffffff, zz, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], i & 1 ? S::ODD : S::EVEN, zz);
        if (s < done.count) {
          float4* to4 = reinterpret_cast<float4*>(to + s * D + gi * GROUP + g * 8);
          to4[0] = make_float4(v[0], v[1], v[2], v[3]);
          to4[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
      }
    }
    if (cur.n == 0) break;
  }
}

// Joins the records of a (row, q head): PARTS warps, which take every PARTS-th record, one of 32 a lane
// first for its weight, then four at a time.  With one pair of a long sequence there is a record in every CTA.
constexpr int JOIN_WARPS = 8;

template <int D, int PARTS, bool WIDE>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(const QuantAttnArgs a) {
  constexpr int PER = D / 32;
  pdl_wait();
  pdl_trigger();
  const Plan plan = plan_of(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % PARTS;
  const int items = a.rows * a.num_q_heads;
  const int at_item = blockIdx.x * (JOIN_WARPS / PARTS) + warp / PARTS;
  const int item = min(at_item, items - 1);
  const int row = item / a.num_q_heads, head = item % a.num_q_heads;
  const int group = a.num_q_heads / a.num_kv_heads, kvh = head / group;
  const long long total = stages_of(plan, a);
  const int2 where = plan.rows[row];
  const int len = plan.lens[row];
  uint32_t gate[PER / 2];
  if (a.gate != nullptr) {
    const uint16_t* gp = static_cast<const uint16_t*>(a.gate) + (size_t)row * a.gate_row + (size_t)head * a.gate_head + lane * PER;
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) gate[j] = reinterpret_cast<const uint32_t*>(gp)[j];
  }
  int n = 0, at = 0;
  const float* rec = a.partial;
  if (where.x >= 0 && total > 0) {
    const int s = (row - where.y) * group + head % group;
    const int chunk = where.x + s / a.chunk;
    at = s % a.chunk;
    const Chunk e = plan.table[chunk];
    if (e.stages > 0) {
      // CTA b has the stages from floor(b T / B): stage x is of CTA floor(((x + 1) B - 1) / T).
      const int B = ctas_of(total, a.grid, a.least);
      const long long p0 = e.before + (long long)kvh * e.stages, p1 = p0 + e.stages - 1;
      const int first = (int)(((p0 + 1) * B - 1) / total);
      n = (int)(((p1 + 1) * B - 1) / total) - first + 1;
      rec += ((size_t)chunk * a.num_kv_heads + kvh + first) * a.chunk * (D + RECORD_REST);
    }
  }
  const size_t step = (size_t)PARTS * a.chunk * (D + RECORD_REST);
  rec += part * (size_t)a.chunk * (D + RECORD_REST);
  const int mine = n > part ? (n - part + PARTS - 1) / PARTS : 0;
  Reference m{LOWEST, LOWEST};
  float l = 0.f, o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int i0 = 0; i0 < mine; i0 += 32) {
    float4 ml = make_float4(-INFINITY, 0.f, 0.f, 0.f);
    if (i0 + lane < mine) ml = *reinterpret_cast<const float4*>(rec + (i0 + lane) * step + a.chunk * D + RECORD_REST * at);
    const Reference own{ml.x, ml.y};
    Reference top;
    top.score = fmaxf(m.score, warp_max(own.score));
    top.rest = fmaxf(fmaxf(LOWEST, (m.score - top.score) + m.rest), warp_max((own.score - top.score) + own.rest));
    const float f = factor_to(m, top), w = factor_to(own, top);
    m = top;
    l = l * f + warp_sum(w * ml.z);
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] *= f;
    const int cnt = min(32, mine - i0);
    const float* from = rec + i0 * step + at * D;
    for (int i = 0; i < cnt; i += 4) {
      float x[4][PER];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < cnt) {
#pragma unroll
          for (int j = 0; j < PER; j += 2) {
            if (WIDE) {   // dim 8 g + j of a group is at 8 j + perm(g) there
              const int d = lane * PER + j, g = (d & 63) >> 3, to = (d & ~63) + (d & 7) * 8 + ((2 * g + (g >> 2)) & 7);
              x[k][j] = from[(i + k) * step + to];
              x[k][j + 1] = from[(i + k) * step + to + 8];
            } else {
              const float2 y = *reinterpret_cast<const float2*>(from + (i + k) * step + lane * PER + j);
              x[k][j] = y.x;
              x[k][j + 1] = y.y;
            }
          }
        }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float wk = __shfl_sync(0xffffffff, w, (i + k) & 31);
        if (i + k < cnt) {
#pragma unroll
          for (int j = 0; j < PER; ++j) o[j] = fmaf(wk, x[k][j], o[j]);
        }
      }
    }
  }
  if (PARTS > 1) {
    __shared__ float all[JOIN_WARPS][D + 3];
    float(*parts)[D + 3] = all + warp / PARTS * PARTS;
#pragma unroll
    for (int j = 0; j < PER; ++j) parts[part][j * 32 + lane] = o[j];
    if (lane == 0) {
      parts[part][D] = m.score;
      parts[part][D + 1] = m.rest;
      parts[part][D + 2] = l;
    }
    __syncthreads();
    if (part != 0) return;
    m = Reference{LOWEST, LOWEST};
#pragma unroll
    for (int x = 0; x < PARTS; ++x) m.score = fmaxf(m.score, parts[x][D]);
#pragma unroll
    for (int x = 0; x < PARTS; ++x) m.rest = fmaxf(m.rest, (parts[x][D] - m.score) + parts[x][D + 1]);
    l = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] = 0.f;
#pragma unroll
    for (int x = 0; x < PARTS; ++x) {
      const float w = factor_to(Reference{parts[x][D], parts[x][D + 1]}, m);
      l += w * parts[x][D + 2];
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] = fmaf(w, parts[x][j * 32 + lane], o[j]);
    }
  }
  if (at_item != item) return;
  // A row without keys gives 0, whatever its gate; one whose weights are all 0 (scores of -inf) or NaN gives NaN.
  const float inv = 1.f / l;
  const bool some = n > 0 && len > 0;
  float y[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) y[j] = some ? o[j] * inv : 0.f;
  if (a.gate != nullptr && some) {
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) {
      const float2 f = two_floats(gate[j], a.half);
      y[2 * j] *= sigmoidf_(f.x);
      y[2 * j + 1] *= sigmoidf_(f.y);
    }
  }
  if (a.out != nullptr) {
    uint32_t* to = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (size_t)item * D + lane * PER);
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) to[j] = two_halves(y[2 * j], y[2 * j + 1], a.half);
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
    for (int j = 0; j < PER; ++j) a.out_q[(size_t)item * D + lane * PER + j] = f32_to_e4m3(y[j] * si);
    if (lane % (32 / PER) == 0) {
      const int kb = (head * D + lane * PER) >> 5;
      a.out_sf[((size_t)(row >> 7) * (a.num_q_heads * D >> 7) + (kb >> 2)) * 512 + sf_atom_offset(row & 127, kb & 3)] = code;
    }
  }
}

int check_rows(const QuantRowsArgs& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return -1;
  if ((a.bits != 4 && a.bits != 8) || a.page_shift < 4 || a.page_shift > 8) return -1;
  if (a.rows < 0 || a.num_kv_heads < 1 || a.num_pages < 1 || a.num_slots < 1 || a.max_pages < 1) return -1;
  return 0;
}

// Warps that share four rows and a group: a head each where rows are few, so that the device fills up.
int row_blocks(QuantRowsArgs& a) {
  const long long some = ((long long)a.rows + 3) / 4 * (a.head_dim / GROUP);
  const long long want = (148 * 48 + some - 1) / some;
  a.step = (int)(want > a.num_kv_heads ? a.num_kv_heads : want);
  return (int)((some * a.step + ROW_WARPS - 1) / ROW_WARPS);
}

// More slots of a sequence than this go to quant_wide.cu (bf16; f16 stays here, in parts: launch_bits).  Measured with 64
// sequences of 4096 keys and 2 kv heads, in us: here with the most slots of one unit : there with 40 slots (nearly the same from
// 17 to 64) : here with two units, twice one.
//             4 bits           8 bits
//   64 dims   40 :  72 :  80   42 :  71 :  84
//   128 dims  75 :  77 : 150   83 :  80 : 165
//   256 dims  72 : 100 : 144   77 : 124 : 154
constexpr int most_narrow(int d) { return d == 256 ? 16 : 32; }

// The variant for sequences of so many query slots.
struct Variant {
  int tiles, warps, blocks, ctas;   // tiles of 8 slots of a warp; warps of a CTA; blocks of a stage; CTAs of an SM
};
constexpr Variant variant_of(int d, int bits, int slots) {
  if (d == 256) return slots <= 8 ? Variant{1, 4, 1, bits == 4 ? 3 : 2} : Variant{2, 8, 1, 1};
  if (slots <= 8) return {1, 8, d == 128 && bits == 8 ? 1 : 2, 2};
  if (slots <= 16) return {2, 8, 2, d == 64 ? 2 : 1};
  return {4, 8, d == 64 ? 2 : 1, 1};
}

template <int D, bool WIDE>
int launch_join(const QuantAttnArgs& a, cudaStream_t stream) {
  // Warps that share a pair's records: with few pairs a long sequence leaves a record in every CTA.
  const long long items = (long long)a.rows * a.num_q_heads;
  int parts = JOIN_WARPS;
  while (parts > 1 && items * parts > 4096) parts /= 2;
  const auto join = parts == 8 ? join_kernel<D, 8, WIDE> : parts == 4 ? join_kernel<D, 4, WIDE> : parts == 2 ? join_kernel<D, 2, WIDE> : join_kernel<D, 1, WIDE>;
  zs_launch(join, (int)((items * parts + JOIN_WARPS - 1) / JOIN_WARPS), JOIN_WARPS * 32, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

template <class S>
int launch_attend(QuantAttnArgs a, cudaStream_t stream) {
  const int room = (227 * 1024 / S::CTAS - 1024 * (S::CTAS > 1) - 128) & ~127;
  a.ring_offset = (S::FIXED + 127) & ~127;
  a.ring = (room - a.ring_offset) / (S::WARPS * S::STAGE_BYTES);
  if (a.ring > MAX_RING) a.ring = MAX_RING;
  if (a.ring < 1 || a.chunk % S::SLOTS != 0 || a.stage % S::KEYS != 0) return -1;
  const int bytes = a.ring_offset + S::WARPS * a.ring * S::STAGE_BYTES;
  const auto kernel = attend_kernel<S>;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  zs_launch(kernel, dim3(a.grid, a.chunk / S::SLOTS), S::WARPS * 32, bytes, stream, a);
  return launch_join<S::D, false>(a, stream);
}

template <int D, int BITS, int SLOTS, bool FINE>
int launch_variant(const QuantAttnArgs& a, cudaStream_t stream) {
  constexpr Variant v = variant_of(D, BITS, SLOTS);
  return launch_attend<Shape<D, BITS, v.tiles, v.warps, v.blocks, v.ctas, FINE>>(a, stream);
}

template <int D, int BITS, bool FINE>
int launch_tiles(const QuantAttnArgs& a, cudaStream_t stream) {
  if (a.tiles == 1) return launch_variant<D, BITS, 8, FINE>(a, stream);
  if (a.tiles == 2) return launch_variant<D, BITS, 16, FINE>(a, stream);
  if constexpr (D < 256) return launch_variant<D, BITS, 32, FINE>(a, stream);
  return -1;
}

template <int D>
int launch_bits(const QuantAttnArgs& a, cudaStream_t stream) {
  if (a.chunk == WIDE_SLOTS) {
    // f16 outputs: quant_wide.cu rounds K and V to f16, which with the outputs' own rounding gives up to 1.8 times the latter
    // (for bf16 outputs 1.03).  Every unit of 128 slots is then walked by parts, as exactly as few slots are, and the keys are
    // opened for each: 64 sequences of 4096 keys, 2 heads, 128 slots take 179, 363 and 645 us with 64, 128 and 256 dims (81, 92
    // and 129 in bf16).
    if (a.half) return a.bits == 4 ? launch_variant<D, 4, most_narrow(D), true>(a, stream) : launch_variant<D, 8, most_narrow(D), true>(a, stream);
    const int e = launch_wide(a, stream);
    return e ? e : launch_join<D, true>(a, stream);
  }
  if (a.bits == 4) return a.half ? launch_tiles<D, 4, true>(a, stream) : launch_tiles<D, 4, false>(a, stream);
  return a.half ? launch_tiles<D, 8, true>(a, stream) : launch_tiles<D, 8, false>(a, stream);
}

// CTAs of the attention, and the fewest stages that are worth one (a stage a warp).
void set_grid(QuantAttnArgs& a) {
  if (a.chunk == WIDE_SLOTS) {
    a.grid = 148;
    a.least = 1;
    return;
  }
  const Variant v = variant_of(a.head_dim, a.bits, 8 * a.tiles);
  a.grid = 148 * v.ctas;
  a.least = v.warps;
}

int check_attn(const QuantAttnArgs& a) {
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return -1;
  if ((a.bits != 4 && a.bits != 8) || a.num_kv_heads < 1 || a.num_q_heads % a.num_kv_heads != 0) return -1;
  if (a.rows < 0 || a.rows > a.max_rows || a.num_seqs < 0 || a.max_seq_rows < 1 || a.work == nullptr) return -1;
  return 0;
}

}  // namespace qc
}  // namespace zs

extern "C" int zs_quant_block_bytes(int head_dim, int bits) { return zs::qc::block_bytes(head_dim, bits); }

extern "C" int zs_quant_store(const QuantRowsArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_rows(*args)) return e;
  if (args->rows == 0) return 0;
  QuantRowsArgs a = *args;
  const int blocks = zs::qc::row_blocks(a);
  zs_launch(a.bits == 4 ? zs::qc::store_kernel<4> : zs::qc::store_kernel<8>, blocks, zs::qc::ROW_WARPS * 32, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_quant_load(const QuantRowsArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_rows(*args)) return e;
  if (args->rows == 0) return 0;
  QuantRowsArgs a = *args;
  const int blocks = zs::qc::row_blocks(a);
  zs_launch(a.bits == 4 ? zs::qc::load_kernel<4> : zs::qc::load_kernel<8>, blocks, zs::qc::ROW_WARPS * 32, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

// The variant for sequences of `slots` query slots: tiles of 8 slots of a unit, keys of a stage.
extern "C" void zs_quant_attn_shape(int head_dim, int bits, int slots, int* tiles, int* stage) {
  if (slots > zs::qc::most_narrow(head_dim)) {
    *tiles = zs::qc::WIDE_SLOTS / 8;
    *stage = zs::qc::WIDE_KEYS;
    return;
  }
  const zs::qc::Variant v = zs::qc::variant_of(head_dim, bits, slots);
  *tiles = v.tiles;
  *stage = v.blocks * zs::qc::TOK;
}

extern "C" long long zs_quant_attn_work(int max_chunks, int max_rows, int max_seqs) {
  return 32 + (long long)max_chunks * 32 + (long long)max_rows * 12 + (long long)(ZS_QUANT_CTAS + max_seqs) * 4;
}

extern "C" int zs_quant_attn_plan(const QuantAttnArgs* args, cudaStream_t stream) {
  if (int e = zs::qc::check_attn(*args)) return e;
  QuantAttnArgs a = *args;
  zs::qc::set_grid(a);
  zs_launch(zs::qc::plan_kernel, 1, zs::qc::PLAN_THREADS, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_quant_attn(const QuantAttnArgs* args, cudaStream_t stream) {
  using namespace zs::qc;
  QuantAttnArgs a = *args;
  if (int e = check_attn(a)) return e;
  set_grid(a);
  if (a.num_pages < 1 || a.num_slots < 1 || a.max_pages < 1 || a.page_shift < 4 || a.page_shift > 8 || a.partial == nullptr) return -1;
  if (a.rows == 0) return 0;
  if (a.head_dim == 64) return launch_bits<64>(a, stream);
  if (a.head_dim == 128) return launch_bits<128>(a, stream);
  return launch_bits<256>(a, stream);
}
