// Sampled speculative decoding: token probabilities and the verification of drafted tokens.
//
// Verification keeps the target distribution exactly (accept draft d with probability
// min(1, p(d) / q(d)); on the first rejection draw from max(p - q, 0), after the last
// acceptance from p).  It is done in fixed point, so a sum has one value in any order and the
// tokens are the same for every grid and every implementation of the definition:
//
//   P(i) = floor(clamp(p_i, 0, 1) * 2^38), NaN -> 0;  Q(i) likewise (no draft probabilities:
//   all of it on the draft);  U = floor(clamp(u, 0, 1 - 2^-24) * 2^24)
//   draft j is accepted     iff U_j * Q(d_j) < P(d_j) * 2^24   (a 62-bit compare)
//   rejected at j           w_i = max(P_j(i) - Q_j(i), 0), or P_j(i) where all of those are 0
//   all accepted            w_i = P_m(i), m the number of drafts
//   token                   the first i with w_0 + .. + w_i > floor(U_k * sum(w) / 2^24)
//
// A probability below 2^-38 (4e-12) counts as 0: the mass that can lose is below 1e-6 of a row
// of 2^18 tokens, the rounding of a 32-bit softmax over it.
#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace spec {

constexpr int T = 1024;
constexpr float kFix = 274877906944.0f;  // 2^38
typedef unsigned long long u64;

ZS_DEVICE uint32_t okey(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
ZS_DEVICE float from_okey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

// NaN counts as masked, +inf as the largest number (two of them share the mass).
ZS_DEVICE float clean(float x) { return x != x ? -INFINITY : fminf(x, 3.4028234663852886e38f); }

template <typename V, typename F>
ZS_DEVICE V block_all(V v, V* red, F op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffff, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffff, v, o));
  return v;
}

// Probabilities of one row (a CTA each): max, top-k threshold (radix select over the ordered
// image of the logit, ties with the k-th kept), top-p threshold (the same over fixed-point
// masses, whose histogram sums have one value; ties kept), sum of the kept, quotients.
__global__ void __launch_bounds__(T) probs_kernel(const TokenProbsArgs a) {
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, V = a.vocab;
  const float* x = a.logits + blockIdx.x * a.ld;
  float* out = a.out + blockIdx.x * a.ld_out;
  __shared__ u64 red[32];
  __shared__ u64 hist[256];
  __shared__ uint32_t pick;
  __shared__ u64 left;
  // (largest logit, its lowest id) as one key
  u64 best = 0;
  for (int i = tid; i < V; i += T) {
    const u64 k = ((u64)okey(clean(x[i])) << 32) | (uint32_t)~i;
    best = k > best ? k : best;
  }
  best = block_all(best, red, [](u64 p, u64 q) { return p > q ? p : q; });
  const float top = from_okey((uint32_t)(best >> 32));
  const float temp = a.temperature[blockIdx.x];
  if (top == -INFINITY || !(temp > 0.f)) {  // nothing left, or greedy: all mass on the best token
    const int id = top == -INFINITY ? -1 : (int)~(uint32_t)best;
    for (int i = tid; i < V; i += T) out[i] = i == id ? 1.f : 0.f;
    return;
  }
  const float inv_t = fminf(1.f / temp, 3.4028234663852886e38f);
  auto mass = [&](float v) { return exp2f((v - top) * inv_t * 1.4426950408889634f); };
  uint32_t thr = 0;  // keep keys >= thr
  const int K = a.top_k != nullptr ? a.top_k[blockIdx.x] : 0;
  const float P = a.top_p != nullptr ? a.top_p[blockIdx.x] : 1.f;
  for (int phase = 0; phase < 2; ++phase) {
    const bool by_mass = phase == 1;
    if (by_mass ? !(P < 1.f) : !(K > 0 && K < V)) continue;
    u64 need = (u64)K;
    if (by_mass) {
      u64 sum = 0;
      for (int i = tid; i < V; i += T) {
        const float v = clean(x[i]);
        if (okey(v) >= thr) sum += (u64)(mass(v) * kFix);
      }
      sum = block_all(sum, red, [](u64 p, u64 q) { return p + q; });
      need = (u64)((double)fmaxf(P, 0.f) * (double)sum);
      if (need == 0) need = 1;
    }
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += T) {
        const float v = clean(x[i]);
        const uint32_t k = okey(v);
        if (k < thr || (shift < 24 && (k >> (shift + 8)) != (prefix >> (shift + 8)))) continue;
        atomicAdd(&hist[(k >> shift) & 255], by_mass ? (u64)(mass(v) * kFix) : 1ull);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255;
        for (; d > 0 && hist[d] < need; --d) need -= hist[d];
        pick = prefix | ((uint32_t)d << shift);
        left = need;
      }
      __syncthreads();
      prefix = pick;
      need = left;
    }
    thr = max(thr, prefix);
  }
  float sum = 0.f;
  for (int i = tid; i < V; i += T) {
    const float v = clean(x[i]);
    if (okey(v) >= thr) sum += mass(v);
  }
  sum = block_all(sum, reinterpret_cast<float*>(red), [](float p, float q) { return p + q; });
  const float inv = 1.f / sum;
  for (int i = tid; i < V; i += T) {
    const float v = clean(x[i]);
    out[i] = okey(v) >= thr ? mass(v) * inv : 0.f;
  }
}

ZS_DEVICE u64 fixed(float p) { return (u64)(fminf(fmaxf(p, 0.f), 1.f) * kFix); }
ZS_DEVICE u64 ubits(float u) { return (u64)(fminf(fmaxf(u, 0.f), 0.99999994f) * 16777216.f); }

struct Weights {
  const float *p, *q;  // q: draft probabilities, or null
  int less;            // without q: the rejected draft, -1 for none
  ZS_DEVICE u64 operator()(int i) const {
    const u64 w = fixed(p[i]);
    if (q != nullptr) {
      const u64 v = fixed(q[i]);
      return w > v ? w - v : 0;
    }
    return i == less ? 0 : w;
  }
};

// One CTA per sequence; each warp owns a contiguous part of the vocabulary.
__global__ void __launch_bounds__(T) verify_kernel(const DraftVerifyArgs a) {
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  __shared__ u64 part[33];
  __shared__ int taken_s;
  const int m = a.counts != nullptr ? min(max(a.counts[s], 0), a.k) : a.k;
  const int* drafts = a.drafts + (size_t)s * a.k;
  const float* u = a.uniform + (size_t)s * (a.k + 1);
  if (tid == 0) {
    int j = 0;
    for (; j < m; ++j) {
      const int d = drafts[j];
      if (d < 0 || d >= V) break;
      const u64 p = fixed(a.target[s * a.target_seq + j * a.target_row + d]);
      const u64 q = a.draft_probs != nullptr ? fixed(a.draft_probs[s * a.draft_seq + j * a.draft_row + d]) : (1ull << 38);
      if (!(ubits(u[j]) * q < (p << 24))) break;
    }
    taken_s = j;
  }
  __syncthreads();
  const int taken = taken_s;
  const bool rejected = taken < m;
  Weights w{a.target + s * a.target_seq + taken * a.target_row, nullptr, -1};
  if (rejected) {
    if (a.draft_probs != nullptr) w.q = a.draft_probs + s * a.draft_seq + taken * a.draft_row;
    else w.less = drafts[taken];
  }
  const int per = ((V + 31) / 32 + 31) / 32 * 32, i0 = min(V, warp * per), i1 = min(V, i0 + per);
  u64 total = 0;
  for (int round = 0; round < 2; ++round) {
    u64 sum = 0;
    for (int i = i0 + lane; i < i1; i += 32) sum += w(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
    __syncthreads();
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    total = 0;
    for (int j = 0; j < 32; ++j) total += part[j];
    if (total != 0 || !rejected) break;
    w.q = nullptr;  // p <= q everywhere: the target itself
    w.less = -1;
  }
  const u64 un = ubits(u[a.k]);
  const u64 goal = un * (total >> 24) + ((un * (total & 0xFFFFFFull)) >> 24);
  u64 before = 0;
  for (int j = 0; j < warp; ++j) before += part[j];
  int* rec = a.record + (size_t)s * (a.k + 2);
  if (tid == 0) {
    rec[0] = taken + 1;
    for (int j = 0; j <= a.k; ++j)
      if (j != taken) rec[1 + j] = j < taken ? drafts[j] : -1;
    if (total == 0) {
      rec[1 + taken] = 0;
      report_error(a.err, kErrBadShape);
    }
  }
  if (total != 0 && goal >= before && goal < before + part[warp]) {
    for (int i = i0; i < i1; i += 32) {
      u64 x = i + lane < i1 ? w(i + lane) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffff, x, o);
        if (lane >= o) x += y;
      }
      const uint32_t over = __ballot_sync(0xffffffff, before + x > goal);
      if (over != 0) {
        if (lane == 0) rec[1 + taken] = i + __ffs(over) - 1;
        break;
      }
      before += __shfl_sync(0xffffffff, x, 31);
    }
  }
}

}  // namespace spec
}  // namespace zs

extern "C" int zs_token_probs(const TokenProbsArgs* args, cudaStream_t stream) {
  const TokenProbsArgs& a = *args;
  if (a.vocab < 1 || a.rows < 0 || a.ld < a.vocab || a.ld_out < a.vocab || a.temperature == nullptr) return -1;
  if (a.rows == 0) return 0;
  zs_launch(zs::spec::probs_kernel, a.rows, zs::spec::T, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

extern "C" int zs_draft_verify(const DraftVerifyArgs* args, cudaStream_t stream) {
  const DraftVerifyArgs& a = *args;
  if (a.n < 0 || a.k < 1 || a.k > ZS_VERIFY_MAX_DRAFTS || a.vocab < 1 || a.vocab > (1 << 24)) return -1;
  if (a.n == 0) return 0;
  zs_launch(zs::spec::verify_kernel, a.n, zs::spec::T, 0, stream, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}
