// Gated GQA attention over a paged cache whose sequences share leading pages.
//
// The step's rows attend through segments: a segment is a list of rows and a range of page
// positions that all of them share (a common prompt's pages, or one sequence's own).  Row r
// sees key t of a segment when t < seq_lens[r]; its output is the softmax over the keys of all
// its segments, merged from one record (o, m, l) per (row, segment, head):
//   s_t = scale * q . k_t,  m = max s_t,  l = sum exp(s_t - m),  o = sum exp(s_t - m) v_t
//   out = sigmoid(gate) * (sum_j exp(m_j - M) o_j) / (sum_j exp(m_j - M) l_j),  M = max m_j.
// A row that sees no key gives 0.  Cache blocks are those of attention.cu.
#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace sattn {

constexpr int D = 256;
constexpr int PAGE = 16;
constexpr int PREC = D + 4;  // record: o[256], m, l, padding to 16 bytes

// Element offset of (token row r, dims d..d+7) inside a (page, kv head) block (d a multiple of 8).
ZS_DEVICE int swz(int r, int d) {
  return (r >> 3) * 2048 + (d >> 6) * 512 + (r & 7) * 64 + ((((d & 63) >> 3) ^ (r & 7)) << 3);
}

// One warp per (segment entry, q head); a lane owns 8 dims.
__global__ void __launch_bounds__(128) partial_kernel(const SharedAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item >= a.entries * a.num_q_heads) return;
  const int e = item / a.num_q_heads, h = item % a.num_q_heads, kvh = h / (a.num_q_heads / a.num_kv_heads);
  const int row = a.seg_rows[e], seg = a.entry_seg[e];
  const int len = min(a.seq_lens[row], a.max_pages * PAGE);
  const int t0 = a.seg_page0[seg] * PAGE, t1 = a.seg_page1[seg] < 0 ? len : min(len, a.seg_page1[seg] * PAGE);
  const int* pt = a.page_table + (size_t)a.row_slot[row] * a.max_pages;
  float q[8], o[8], m = -INFINITY, l = 0.f;
  const uint4 qv = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + ((size_t)row * a.num_q_heads + h) * D)[lane];
  const float qscale = a.sm_scale * 1.4426950408889634f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    q[j] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&qv)[j]) * qscale;
    o[j] = 0.f;
  }
  for (int t = t0; t < t1; ++t) {
    const int page = pt[t / PAGE];
    if (page < 0 || page >= a.num_pages) {
      report_error(a.err, kErrBadShape);
      break;
    }
    const size_t at = ((size_t)page * a.num_kv_heads + kvh) * PAGE * D + swz(t % PAGE, lane * 8);
    const uint4 kv = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.k_cache) + at);
    const uint4 vv = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.v_cache) + at);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s += q[j] * __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&kv)[j]);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), r = exp2f(m - mn), p = exp2f(s - mn);
    l = l * r + p;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = o[j] * r + p * __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&vv)[j]);
    m = mn;
  }
  float* rec = a.partial + (size_t)item * PREC;
#pragma unroll
  for (int j = 0; j < 8; ++j) rec[lane * 8 + j] = o[j];
  if (lane == 0) {
    rec[D] = m;
    rec[D + 1] = l;
  }
}

// One CTA per (row, q head), thread = dim.
__global__ void __launch_bounds__(D) merge_kernel(const SharedAttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x, h = blockIdx.y, d = threadIdx.x;
  float m = -INFINITY;
  for (int j = 0; j < a.levels; ++j) {
    const int e = a.row_entry[row * a.levels + j];
    if (e >= 0) m = fmaxf(m, a.partial[((size_t)e * a.num_q_heads + h) * PREC + D]);
  }
  float l = 0.f, o = 0.f;
  for (int j = 0; j < a.levels; ++j) {
    const int e = a.row_entry[row * a.levels + j];
    if (e < 0) continue;
    const float* rec = a.partial + ((size_t)e * a.num_q_heads + h) * PREC;
    if (rec[D] == -INFINITY) continue;
    const float sc = exp2f(rec[D] - m);
    l += rec[D + 1] * sc;
    o += rec[d] * sc;
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
  if (a.head_dim != D || a.page_size != PAGE || a.levels < 1 || a.num_segs < 0 || a.rows < 0) return -1;
  if (a.partial == nullptr || a.max_pages < 1 || a.max_pages > (1 << 26)) return -1;
  return 0;
}

}  // namespace sattn
}  // namespace zs

extern "C" int zs_shared_attn(const SharedAttnArgs* args, cudaStream_t stream) {
  const SharedAttnArgs& a = *args;
  if (int e = zs::sattn::check(a)) return e;
  if (a.rows == 0) return 0;
  const int items = a.entries * a.num_q_heads;
  if (items > 0) zs_launch(zs::sattn::partial_kernel, (items + 3) / 4, 128, 0, stream, a);
  zs_launch(zs::sattn::merge_kernel, dim3(a.rows, a.num_q_heads), zs::sattn::D, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
