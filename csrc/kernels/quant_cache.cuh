// What the kernels of the quantised K/V cache share: its blocks, and the plan of a step's attention.
#pragma once

#include <cuda_fp16.h>

#include <climits>

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

__device__ __forceinline__ float ex2(float x) {   // 2^x, results below 2^-126 as 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The weights of a row are held as f16 numbers against a reference that bounds its scores (with the scales of V):
// at most 2^LIFT where it is exact, 2^(LIFT + SLACK) before it is moved, and twice that with a scale's mantissa.
// A row's sum of weights and its sum of weights times offsets are held 2^ABOVE larger, so that they leave 32 bits at neither
// end of what V may be.
constexpr float LIFT = 6.f, SLACK = 8.f, ABOVE = 24.f, BELOW = 0x1p-24f;
// The reference is in two parts, a score and what V's scales add to it, both in log2: beside a score of 2^25 the other would be
// lost, and with it the bound.  A weight is 2^((score - reference's score) + (rest)), whose first difference is exact where
// it counts.
struct Reference {
  float score, rest;   // score -inf: no key yet
};
constexpr float LOWEST = -0x1p126f;   // below every reference's parts, and finite: its distance to -inf is a number
// What sums held against `a` are multiplied by to be held against `top`, which is not below it and not below LOWEST.
__device__ __forceinline__ float factor_to(const Reference& a, const Reference& top) { return ex2((a.score - top.score) + (a.rest - top.rest)); }
// A record: a slot's sums of V's dims for all slots of a unit, then for each slot its reference, its sum of weights and nothing.
constexpr int RECORD_REST = ZS_QUANT_REST;
constexpr float MAX_QUERY = 0x1p101f;   // a slot with a query of this size gives NaN

struct Chunk {          // 32 bytes
  long long before;     // stages of the chunks before, all kv heads
  int row, slot;        // first row of the sequence, its page-table row
  int first, count;     // slots [first, first + count) of the sequence
  int len, stages;      // keys of the longest row among them, stages of one kv head
};

struct Plan {           // the workspace's integers
  long long* total;     // stages of all chunks, all kv heads; then the rows that were planned
  Chunk* table;         // [max_chunks]
  int2* rows;           // [max_rows] first chunk and first row of the row's sequence (-1: none)
  int* lens;            // [max_rows] keys of the row
  int* start;           // [ZS_QUANT_CTAS] chunk of a CTA's first stage
  int* offset;          // [max_seqs] chunks before the sequence
};

__host__ __device__ inline Plan plan_of(const QuantAttnArgs& a) {
  Plan p;
  uint8_t* w = reinterpret_cast<uint8_t*>(a.work);
  p.total = reinterpret_cast<long long*>(w);
  p.table = reinterpret_cast<Chunk*>(w + 32);
  p.rows = reinterpret_cast<int2*>(p.table + a.max_chunks);
  p.lens = reinterpret_cast<int*>(p.rows + a.max_rows);
  p.start = p.lens + a.max_rows;
  p.offset = p.start + ZS_QUANT_CTAS;
  return p;
}

// Stages of the plan, 0 if it is not of the rows that are asked for (a captured call whose plan was changed since).
__device__ __forceinline__ long long stages_of(const Plan& p, const QuantAttnArgs& a) {
  const longlong2 x = *reinterpret_cast<const longlong2*>(p.total);
  if (x.y == a.rows) return x.x;
  report_error(a.err, kErrBadShape);
  return 0;
}

// Number of CTAs that share T stages.
__device__ __forceinline__ int ctas_of(long long total, int grid, int least) {
  return (int)max(1ll, min((long long)grid, total / least));
}

// quant_wide.cu: sequences with more than 16 or 32 query slots.
constexpr int WIDE_SLOTS = 128, WIDE_KEYS = 64;   // slots of a unit, keys of a stage
int launch_wide(QuantAttnArgs a, cudaStream_t stream);

}  // namespace qc
}  // namespace zs
