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
#include <cooperative_groups.h>

#include "sm100_common.cuh"
#include "zs_kernels.h"

namespace zs {
namespace spec {

namespace cg = cooperative_groups;

constexpr float kMax = 3.4028234663852886e38f;
constexpr int kCluster = 16;             // CTAs on a row at most
typedef unsigned long long u64;

ZS_DEVICE uint32_t okey(float f) {
  const uint32_t b = __float_as_uint(f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
ZS_DEVICE float from_okey(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

// NaN counts as masked, +inf as the largest number (two of them share the mass).
ZS_DEVICE float clean(float x) { return x != x ? -INFINITY : fminf(x, kMax); }

ZS_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// floor(clamp(p, 0, 1) * 2^38).
ZS_DEVICE u64 fixed(float p) { return (u64)(fminf(fmaxf(p, 0.f), 1.f) * 274877906944.f); }

template <typename V, typename F>
ZS_DEVICE V warp_all(V v, F op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffff, v, o));
  return v;
}
// Over all threads of the block; red: a value per warp.
template <int WARPS, typename V, typename F>
ZS_DEVICE V block_all(V v, V* red, F op, V none) {
  v = warp_all(v, op);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_all((threadIdx.x & 31) < WARPS ? red[threadIdx.x & 31] : none, op);
}

// The other CTAs of a cluster may be written to once they run: announced at the start, waited for
// before the first access.
ZS_DEVICE void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
ZS_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
ZS_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
ZS_DEVICE void cluster_wait_started() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// ---------------------------------------------------------------------------------------
// Token probabilities.  A cluster of up to 16 CTAs holds a row in shared memory (64 KiB each, three
// CTAs to an SM, so that some load while others compute; with two, 256 rows of 248320 tokens took 141
// us plain instead of 110): the row is read once and written once whatever it asks for.  Those rows'
// 509 MB take 78 us to copy; they take 110 us plain, 123 greedy, 173 with k = 50, 282 with k = 200 and
// 541 with a nucleus of 500 tokens (the radix select): 21 clusters fit on the device, and a cluster's steps
// wait for one another.  What the CTAs have to know of one another goes through distributed
// shared memory.
//   plain     e = 2^((x - m) c) against the CTA's own maximum and its sum; (m, sum) of all CTAs;
//             one exchange.
//   greedy    the row's maximum, then its lowest id.
//   top-k     up to 256: the k-th largest of the warps' maxima (at least k logits are as large)
//             leaves little more than k candidates, which every CTA ranks for itself: exact
//             threshold, nucleus and sum from the sorted list.  Two exchanges.
//   top-p     the same with the candidates of k = 128, where the nucleus lies within them.
//   otherwise (a wide nucleus, k above 256, many ties): radix select by 8 bits of the distance of
//             ordered images from the top's over histograms of counts or of fixed-point masses, whose sums have
//             one value in any order.
constexpr int PT = 512, PW = PT / 32;
constexpr int kChunk = 16384;            // logits of a CTA at most
constexpr int kSmallK = 256;             // as many as a full row has warps
constexpr int kList = 256, kCand = 1024; // candidates of a CTA, of a row
constexpr int kHist = 4;                 // histograms of a CTA: one for every PW / 4 warps

struct ProbsSmem {
  float x[kChunk];
  union {
    struct {
      uint32_t warp_max[kCluster * PW];
      float list[kList], cand[kCand + 4];    // the CTA's candidates, the row's
    };
    struct {
      uint32_t low[kHist * 256], high[kHist * 256];  // 19 bits of a mass each
      u64 mine_hist[257];                // the CTA's, and what is outside
    };
    u64 total[257];                      // the row's
  };
  float2 part[kCluster];                 // (maximum, sum) of every CTA
  uint32_t first[kCluster];              // greedy: lowest id of the maximum
  int count[kCluster];                   // candidates of every CTA
  u64 red[PW], left;
  uint32_t pick;
  int mine;
  uint8_t vote[2][PW], found;
};
static_assert(3 * (sizeof(ProbsSmem) + 1024) <= 228 * 1024, "three CTAs on an SM");
static_assert((u64)kChunk / kHist << 19 < 1ull << 32, "a histogram's sums in 32 bits");

ZS_DEVICE void cp_async(void* dst, const void* src, bool wide) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if (wide) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(d), "l"(src) : "memory");
}

template <int VEC>
__global__ void __launch_bounds__(PT, 3) probs_kernel(const TokenProbsArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  ProbsSmem& s = *reinterpret_cast<ProbsSmem*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), row = blockIdx.x / n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = a.vocab;
  cluster_started();
  pdl_wait();
  pdl_trigger();
  const int chunk = ((V + n - 1) / n + 3) & ~3, base = rank * chunk, len = max(0, min(V - base, chunk));
  const float* in = a.logits + row * a.ld + base;
  float* out = a.out + row * a.ld_out + base;
  // A thread reads what it brought itself: groups of VEC logits, PT groups apart.
  for (int i = tid * VEC; i < len; i += PT * VEC) {
    if (VEC == 4 && i + 3 < len) {
      cp_async(s.x + i, in + i, true);
    } else {
      for (int k = 0; k < VEC; ++k) {
        if (i + k < len) cp_async(s.x + i + k, in + i + k, false);
        else s.x[i + k] = -INFINITY;
      }
    }
  }
  const float temp = a.temperature[row];
  const bool greedy = !(temp > 0.f);
  const int K = a.top_k != nullptr && a.top_k[row] < V ? a.top_k[row] : 0;                // <= 0: all
  const float P = a.top_p != nullptr && a.top_p[row] < 1.f ? fmaxf(a.top_p[row], 0.f) : 1.f;  // 1: all
  // exponents in the exp2 domain; above 0, so that masked logits stay so at an infinite temperature
  const float c = greedy ? 0.f : fmaxf(fminf(1.4426950408889634f / temp, kMax), 1e-45f);
  // f(place in the chunk, logit) for this thread's logits; the last group may pass len (masked there).
  auto each = [&](auto f) {
#pragma unroll 2
    for (int i = tid * VEC; i < len; i += PT * VEC) {
      if (VEC == 4) {
        const float4 v = *reinterpret_cast<const float4*>(s.x + i);
        f(i, clean(v.x));
        f(i + 1, clean(v.y));
        f(i + 2, clean(v.z));
        f(i + 3, clean(v.w));
      } else {
        f(i, clean(s.x[i]));
      }
    }
  };
  // out = value(place, logit).
  auto store = [&](auto value) {
#pragma unroll 2
    for (int i = tid * VEC; i < len; i += PT * VEC) {
      if (VEC == 4 && i + 3 < len) {
        const float4 v = *reinterpret_cast<const float4*>(s.x + i);
        __stcs(reinterpret_cast<float4*>(out + i),
               make_float4(value(i, clean(v.x)), value(i + 1, clean(v.y)), value(i + 2, clean(v.z)), value(i + 3, clean(v.w))));
      } else {
        for (int k = 0; k < VEC; ++k)
          if (i + k < len) __stcs(out + i + k, value(i + k, clean(s.x[i + k])));
      }
    }
  };
  asm volatile("cp.async.wait_all;" ::: "memory");
  float top = -INFINITY;
  each([&](int, float x) { top = fmaxf(top, x); });
  cluster_wait_started();

  if (!greedy && K <= 0 && P == 1.f) {
    top = block_all<PW>(top, reinterpret_cast<float*>(s.red), [](float p, float q) { return fmaxf(p, q); }, -INFINITY);
    const float off = top == -INFINITY ? 0.f : top;
    const auto e = [&](float x) { return ex2((clean(x) - off) * c); };
    float sum = 0.f;
#pragma unroll 2
    for (int i = tid * VEC; i < len; i += PT * VEC) {  // the exponentials take the logits' place
      if (VEC == 4) {
        float4 v = *reinterpret_cast<const float4*>(s.x + i);
        v = make_float4(e(v.x), e(v.y), e(v.z), e(v.w));
        sum += (v.x + v.y) + (v.z + v.w);
        *reinterpret_cast<float4*>(s.x + i) = v;
      } else {
        sum += s.x[i] = e(s.x[i]);
      }
    }
    sum = block_all<PW>(sum, reinterpret_cast<float*>(s.red), [](float p, float q) { return p + q; }, 0.f);
    if (tid < n) cluster.map_shared_rank(s.part, tid)[rank] = make_float2(top, sum);
    cluster.sync();
    const float2 p = lane < n ? s.part[lane] : make_float2(-INFINITY, 0.f);
    const float all = warp_max(p.x);
    const float z = warp_sum(p.x == -INFINITY ? 0.f : p.y * ex2((p.x - all) * c));
    const float scale = top == -INFINITY ? 0.f : ex2((top - all) * c) / z;
    store([&](int, float e) { return e * scale; });
    return;
  }

  // The row's maximum, and every warp's.
  {
    const uint32_t k = __reduce_max_sync(0xffffffff, okey(top));
    if (lane < n) cluster.map_shared_rank(s.warp_max, lane)[rank * PW + warp] = k;
  }
  if (tid == 0) s.mine = 0;
  cluster.sync();
  uint32_t top_key = 0;
  for (int i = lane; i < n * PW; i += 32) top_key = max(top_key, s.warp_max[i]);
  top = from_okey(__reduce_max_sync(0xffffffff, top_key));

  if (greedy || top == -INFINITY) {  // all mass on the best token, none where every token is masked
    uint32_t first = 0xFFFFFFFFu;
    if (top > -INFINITY)
      each([&](int i, float x) {
        if (x == top) first = min(first, (uint32_t)(base + i));
      });
    first = block_all<PW>(first, reinterpret_cast<uint32_t*>(s.red), [](uint32_t p, uint32_t q) { return min(p, q); }, 0xFFFFFFFFu);
    if (tid < n) cluster.map_shared_rank(s.first, tid)[rank] = first;
    cluster.sync();
    first = __reduce_min_sync(0xffffffff, lane < n ? s.first[lane] : 0xFFFFFFFFu);
    store([&](int i, float) { return (uint32_t)(base + i) == first ? 1.f : 0.f; });
    return;
  }

  auto mass = [&](float v) { return ex2((v - top) * c); };
  float thr = -INFINITY, inv = 0.f;  // keep x >= thr
  bool done = false;
  // A nucleus without top-k: is it within the candidates of 128 maxima?
  const int k_bound = K > 0 ? K : min(128, n * PW);
  if (k_bound <= min(kSmallK, n * PW)) {
    // A lower bound of the k-th largest of the warp maxima, the upper 16 bits of its image, by digits of
    // 4 bits: every warp counts for one digit.  (Ranking the maxima read shared memory for 3 us.)
    uint32_t bound_key = 0;
    {
      uint32_t key[kCluster * PW / 32];
#pragma unroll
      for (int x = 0; x < kCluster * PW / 32; ++x) key[x] = x * 32 + lane < n * PW ? s.warp_max[x * 32 + lane] : 0;
#pragma unroll 1
      for (int shift = 28; shift >= 16; shift -= 4) {
        const uint32_t t = bound_key | (uint32_t)warp << shift;
        uint32_t c = 0;
#pragma unroll
        for (int x = 0; x < kCluster * PW / 32; ++x) c += key[x] >= t;
        c = __reduce_add_sync(0xffffffff, c);
        if (lane == 0) s.vote[shift >> 2 & 1][warp] = warp == 0 || c >= (uint32_t)k_bound;
        __syncthreads();
        bound_key |= (uint32_t)(31 - __clz(__ballot_sync(0xffffffff, lane < PW && s.vote[shift >> 2 & 1][lane & (PW - 1)]))) << shift;
      }
    }
    const float bound = from_okey(bound_key);  // a NaN where fewer than k warps have an unmasked logit
    if (bound > -INFINITY) {
      each([&](int, float x) {
        if (x >= bound) {
          const int at = atomicAdd(&s.mine, 1);
          if (at < kList) s.list[at] = x;
        }
      });
    }
    __syncthreads();
    // No bound (fewer than K warps have an unmasked logit), too many candidates: the general way.
    if (tid < n) cluster.map_shared_rank(s.count, tid)[rank] = bound > -INFINITY ? s.mine : kList + 1;
    if (K <= 0) {  // the whole row's mass
      float sum = 0.f;
      each([&](int, float x) { sum += mass(x); });
      sum = block_all<PW>(sum, reinterpret_cast<float*>(s.red), [](float p, float q) { return p + q; }, 0.f);
      if (tid < n) cluster.map_shared_rank(s.part, tid)[rank] = make_float2(0.f, sum);
    }
    cluster.sync();
    const float row_z = warp_sum(K <= 0 && lane < n ? s.part[lane].y : 0.f);
    __syncthreads();  // s.part is used again
    int cnt = lane < n ? s.count[lane] : 0;
    const int total = (int)__reduce_add_sync(0xffffffff, (unsigned)min(cnt, kList + 1));
    done = __all_sync(0xffffffff, cnt <= kList) && total <= kCand;
    if (done) {
      // One list, ranked: larger values first.  (Compared four at a time, by one comparison each: k = 200
      // took 389 us with two comparisons a value, 318 so.)
      int before = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffff, before, o);
        if (lane >= o) before += y;
      }
      before -= cnt;
      for (int r = warp; r < n; r += PW) {
        const int at = __shfl_sync(0xffffffff, before, r), m = __shfl_sync(0xffffffff, cnt, r);
        const float* list = cluster.map_shared_rank(s.list, r);
        for (int i = lane; i < m; i += 32) s.cand[at + i] = list[i];
      }
      if (tid < 3) s.cand[total + tid] = -INFINITY;  // the last group of 4
      __syncthreads();
      cluster_arrive();  // the others' lists are read
      float v[kCand / PT];
      int above[kCand / PT];
#pragma unroll
      for (int q = 0; q < kCand / PT; ++q) {
        // Equal values stay in the list's order: before this warp's own 32 `>=` counts, behind them `>`.
        const int i = tid + q * PT, own = i & ~31;
        v[q] = i < total ? s.cand[i] : 0.f;
        above[q] = 0;
        if (own >= total) break;
        const float4* list = reinterpret_cast<const float4*>(s.cand);
#pragma unroll 2
        for (int y = 0; y < own / 4; ++y) {
          const float4 o = list[y];
          above[q] += (o.x >= v[q]) + (o.y >= v[q]) + (o.z >= v[q]) + (o.w >= v[q]);
        }
        for (int y = own; y < min(own + 32, total); ++y) above[q] += s.cand[y] > v[q] || (s.cand[y] == v[q] && y < i);
#pragma unroll 2
        for (int y = own / 4 + 8; y < (total + 3) / 4; ++y) {
          const float4 o = list[y];
          above[q] += (o.x > v[q]) + (o.y > v[q]) + (o.z > v[q]) + (o.w > v[q]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kCand / PT; ++q)
        if (tid + q * PT < total) s.cand[above[q]] = v[q];
      __syncthreads();
      // Threshold, nucleus and sum by the first warp, in sorted order.
      if (warp == 0) {
        thr = K > 0 ? s.cand[K - 1] : bound;
        float z = 0.f;
        int kept = 0;
        for (int i = lane; i < total; i += 32) {
          const float v = s.cand[i];
          if (v >= thr) z += mass(v), ++kept;
        }
        z = warp_sum(z);
        kept = (int)__reduce_add_sync(0xffffffff, (unsigned)kept);
        if (P < 1.f) {  // tokens in descending order while the mass before them is below P
          const float goal = P * (K > 0 ? z : row_z);
          if (K <= 0 && z < goal) kept = 0;  // it reaches beyond them
          float run = 0.f, keep_z = 0.f, last = s.cand[0];
          for (int i0 = 0; i0 < kept; i0 += 32) {
            const float v = i0 + lane < kept ? s.cand[i0 + lane] : -INFINITY, mv = v == -INFINITY ? 0.f : mass(v);
            float inc = mv;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const float y = __shfl_up_sync(0xffffffff, inc, o);
              if (lane >= o) inc += y;
            }
            const uint32_t in = __ballot_sync(0xffffffff, v > -INFINITY && (run + inc - mv < goal || i0 + lane == 0));
            if (in != 0) last = __shfl_sync(0xffffffff, v, 31 - __clz(in));
            run += __shfl_sync(0xffffffff, inc, 31);
            if (in != 0xffffffffu) break;
          }
          thr = last;
          for (int i = lane; i < kept; i += 32)
            if (s.cand[i] >= thr) keep_z += mass(s.cand[i]);
          z = warp_sum(keep_z);
        }
        if (lane == 0) s.part[0] = make_float2(thr, kept > 0 ? z : 0.f);
      }
      __syncthreads();
      thr = s.part[0].x;
      inv = 1.f / s.part[0].y;
      done = s.part[0].y > 0.f;
      cluster_wait();  // nobody reads this CTA's list any more
    }
  } else {
    __syncthreads();  // every warp has read warp_max: the histograms take its place
  }

  if (!done) {
    // A logit's place: how far its ordered image is below the top's, in digits of 8 bits.  Most of what
    // counts is within 2^24 of the top, so the first digit is taken for 0, and looked at only if that is
    // wrong (256 rows with a nucleus of 500 tokens: 788 us with that digit first, when most logits fall
    // into few bins, 582 so; 541 with every CTA adding up its share of the bins, not all of them, and
    // masses only where they are asked for).
    const uint32_t top_image = okey(top);
    uint32_t far = 0xFFFFFFFFu;  // places up to here are kept
    for (int phase = 0; phase < 2; ++phase) {
      const bool by_mass = phase == 1;
      if (by_mass ? P == 1.f : K <= 0) continue;
      u64 need = (u64)K;
      uint32_t prefix = 0;
      bool first = true;
      for (int shift = 16; shift >= 0;) {
        for (int i = tid; i < kHist * 256; i += PT) s.low[i] = s.high[i] = 0;
        __syncthreads();
        u64 outside = 0;
        each([&](int, float x) {
          const uint32_t k = top_image - okey(x);
          if (!(x > -INFINITY) || k > far) return;
          const bool in = shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8));
          if (!in && !(by_mass && first)) return;
          const u64 v = by_mass ? fixed(mass(x)) : 1;
          if (!in) {
            outside += v;
            return;
          }
          const int bin = warp % kHist * 256 + ((k >> shift) & 255);
          atomicAdd(&s.low[bin], (uint32_t)v & 0x7FFFF);
          if (by_mass) atomicAdd(&s.high[bin], (uint32_t)(v >> 19));
        });
        if (by_mass && first) outside = block_all<PW>(outside, s.red, [](u64 p, u64 q) { return p + q; }, (u64)0);
        __syncthreads();
        if (tid < 256) {
          u64 sum = 0;
          for (int i = 0; i < kHist; ++i) sum += s.low[i * 256 + tid] + ((u64)s.high[i * 256 + tid] << 19);
          s.mine_hist[tid] = sum;
        } else if (tid == 256) {
          s.mine_hist[256] = outside;
        }
        cluster.sync();
        // Every CTA adds up its share of the bins and tells all: a thread per bin and CTA, n of them side
        // by side.  (The first one's ninth warp does the same with what is outside.)
        if (tid < 256 || (rank == 0 && warp == 8)) {
          const int r = tid & (n - 1), bin = tid < 256 ? (rank * 256 + tid) / n : 256;
          u64 sum = cluster.map_shared_rank(s.mine_hist, r)[bin];
          for (int o = 1; o < n; o <<= 1) sum += __shfl_xor_sync(0xffffffff, sum, o);
          cluster.map_shared_rank(s.total, r)[bin] = sum;
        }
        cluster.sync();
        if (warp == 0) {  // lane l: bins 8 l and the 7 behind
          u64 sum = 0;
          for (int d = 0; d < 8; ++d) sum += s.total[8 * lane + d];
          u64 upto = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffff, upto, o);
            if (lane >= o) upto += y;
          }
          if (by_mass && first) {
            need = (u64)((double)P * (double)(__shfl_sync(0xffffffff, upto, 31) + s.total[256]));
            if (need == 0) need = 1;
          }
          const uint32_t enough = __ballot_sync(0xffffffff, upto >= need);
          if (lane == (enough != 0 ? __ffs(enough) - 1 : 31)) {
            u64 left = need - (upto - sum);
            int d = 8 * lane;
            const int high = d + 7;
            for (; d < high && s.total[d] < left; ++d) left -= s.total[d];
            s.found = enough != 0 || !(first && shift == 16);
            s.pick = prefix | ((uint32_t)d << shift);
            s.left = s.found ? left : need;
          }
        }
        __syncthreads();
        need = s.left;
        if (s.found) {
          prefix = s.pick;
          shift -= 8;
        } else {
          shift = 24;
        }
        first = false;
      }
      far = min(far, prefix);
    }
    thr = far > top_image ? -INFINITY : from_okey(top_image - far);
    float sum = 0.f;
    each([&](int, float x) {
      if (x >= thr) sum += mass(x);
    });
    sum = block_all<PW>(sum, reinterpret_cast<float*>(s.red), [](float p, float q) { return p + q; }, 0.f);
    if (tid < n) cluster.map_shared_rank(s.part, tid)[rank] = make_float2(0.f, sum);
    cluster.sync();
    inv = 1.f / warp_sum(lane < n ? s.part[lane].y : 0.f);
  }
  store([&](int, float x) { return x >= thr ? mass(x) * inv : 0.f; });
}

// Vocabularies that 16 CTAs do not hold: a CTA per row reads it once per step.
constexpr int T = 1024;

__global__ void __launch_bounds__(T) probs_wide_kernel(const TokenProbsArgs a) {
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
  best = block_all<32>(best, red, [](u64 p, u64 q) { return p > q ? p : q; }, (u64)0);
  const float top = from_okey((uint32_t)(best >> 32));
  const float temp = a.temperature[blockIdx.x];
  if (top == -INFINITY || !(temp > 0.f)) {  // nothing left, or greedy: all mass on the best token
    const int id = top == -INFINITY ? -1 : (int)~(uint32_t)best;
    for (int i = tid; i < V; i += T) out[i] = i == id ? 1.f : 0.f;
    return;
  }
  const float inv_t = fmaxf(fminf(1.f / temp, kMax), 1e-44f);
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
        if (okey(v) >= thr) sum += fixed(mass(v));
      }
      sum = block_all<32>(sum, red, [](u64 p, u64 q) { return p + q; }, (u64)0);
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
        atomicAdd(&hist[(k >> shift) & 255], by_mass ? fixed(mass(v)) : 1ull);
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
  sum = block_all<32>(sum, reinterpret_cast<float*>(red), [](float p, float q) { return p + q; }, 0.f);
  const float inv = 1.f / sum;
  for (int i = tid; i < V; i += T) {
    const float v = clean(x[i]);
    out[i] = okey(v) >= thr ? mass(v) * inv : 0.f;
  }
}

ZS_DEVICE u64 ubits(float u) { return (u64)(fminf(fmaxf(u, 0.f), 0.99999994f) * 16777216.f); }

// ---------------------------------------------------------------------------------------
// Verification: a cluster per sequence; CTA r and warp w own contiguous parts of the vocabulary.
// The row to draw from is read once for the parts' sums, which every CTA gets through
// distributed shared memory; the warp whose part holds the drawn mass reads that part again.
constexpr int VT = 512, VW = VT / 32;

struct Weights {
  const float *p, *q;  // q: draft probabilities, or null
  int less;            // without q: the rejected draft, -1 for none
  ZS_DEVICE u64 of(float x, float y, int i) const {
    const u64 w = fixed(x);
    if (q != nullptr) {
      const u64 v = fixed(y);
      return w > v ? w - v : 0;
    }
    return i == less ? 0 : w;
  }
  ZS_DEVICE u64 operator()(int i) const { return of(p[i], q != nullptr ? q[i] : 0.f, i); }
};

template <int VEC>
__global__ void __launch_bounds__(VT, 2) verify_kernel(const DraftVerifyArgs a) {
  __shared__ u64 part[kCluster * VW];  // sums of every warp of the row's CTAs
  cg::cluster_group cluster = cg::this_cluster();
  const int n = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), s = blockIdx.x / n;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.vocab;
  cluster_started();
  pdl_wait();
  pdl_trigger();
  const int m = a.counts != nullptr ? min(max(a.counts[s], 0), a.k) : a.k;
  const int* drafts = a.drafts + (size_t)s * a.k;
  const float* u = a.uniform + (size_t)s * (a.k + 1);
  int taken = m;  // every warp finds it for itself: a lane per draft
  for (int j0 = 0; j0 < m; j0 += 32) {
    bool ok = true;
    if (j0 + lane < m) {
      const int j = j0 + lane, d = drafts[j];
      ok = d >= 0 && d < V;
      if (ok) {
        const u64 p = fixed(a.target[s * a.target_seq + j * a.target_row + d]);
        const u64 q = a.draft_probs != nullptr ? fixed(a.draft_probs[s * a.draft_seq + j * a.draft_row + d]) : (1ull << 38);
        ok = ubits(u[j]) * q < (p << 24);
      }
    }
    const uint32_t no = __ballot_sync(0xffffffff, !ok);
    if (no != 0) {
      taken = j0 + __ffs(no) - 1;
      break;
    }
  }
  const bool rejected = taken < m;
  Weights w{a.target + s * a.target_seq + taken * a.target_row, nullptr, -1};
  if (rejected) {
    if (a.draft_probs != nullptr) w.q = a.draft_probs + s * a.draft_seq + taken * a.draft_row;
    else w.less = drafts[taken];
  }
  // A warp's part is read in up to 32 blocks; lane b keeps the sum of block b.
  const int per = ((V + n * VW - 1) / (n * VW) + 127) / 128 * 128, i0 = min(V, (rank * VW + warp) * per), i1 = min(V, i0 + per);
  const int block = (per + 32 * 512 - 1) / (32 * 512) * 512;
  u64 total = 0, mine = 0;
  for (int round = 0; round < 2; ++round) {
    mine = 0;
    for (int b = 0; i0 + b * block < i1; ++b) {
      u64 sum = 0;
      const int end = min(i1, i0 + (b + 1) * block);
      for (int i = i0 + b * block; i < end; i += 512) {
        if (VEC == 4) {  // V and so `end` are multiples of 4
          float4 x[4], y[4];  // all on their way together
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = i + j * 128 + lane * 4;
            x[j] = y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at < end) {
              x[j] = __ldg(reinterpret_cast<const float4*>(w.p + at));
              if (w.q != nullptr) y[j] = __ldg(reinterpret_cast<const float4*>(w.q + at));
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = i + j * 128 + lane * 4;
            sum += w.of(x[j].x, y[j].x, at) + w.of(x[j].y, y[j].y, at + 1) + w.of(x[j].z, y[j].z, at + 2) + w.of(x[j].w, y[j].w, at + 3);
          }
        } else {
          float x[16], y[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int at = i + j * 32 + lane;
            x[j] = at < end ? __ldg(w.p + at) : 0.f;
            y[j] = w.q != nullptr && at < end ? __ldg(w.q + at) : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) sum += w.of(x[j], y[j], i + j * 32 + lane);
        }
      }
      sum = warp_all(sum, [](u64 p, u64 q) { return p + q; });
      if (lane == b) mine = sum;
    }
    const u64 sum = warp_all(mine, [](u64 p, u64 q) { return p + q; });
    if (round == 0) cluster_wait_started();
    else cluster.sync();  // the first round's sums are read
    if (lane < n) cluster.map_shared_rank(part, lane)[rank * VW + warp] = sum;
    cluster.sync();
    total = 0;
    for (int j = lane; j < n * VW; j += 32) total += part[j];
    total = warp_all(total, [](u64 p, u64 q) { return p + q; });
    if (total != 0 || !rejected) break;
    w.q = nullptr;  // p <= q everywhere: the target itself
    w.less = -1;
  }
  const u64 un = ubits(u[a.k]);
  const u64 goal = un * (total >> 24) + ((un * (total & 0xFFFFFFull)) >> 24);
  int* rec = a.record + (size_t)s * (a.k + 2);
  if (rank == 0 && tid <= a.k) {
    if (tid == 0) rec[0] = taken + 1;
    if (tid != taken) rec[1 + tid] = tid < taken ? drafts[tid] : -1;
    else if (total == 0) {
      rec[1 + tid] = 0;
      report_error(a.err, kErrBadShape);
    }
  }
  if (total == 0) return;
  u64 before = 0;
  for (int j = lane; j < rank * VW + warp; j += 32) before += part[j];
  before = warp_all(before, [](u64 p, u64 q) { return p + q; });
  if (goal < before || goal >= before + part[rank * VW + warp]) return;
  // The block, then its tokens, 128 at a time.
  u64 upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffff, upto, o);
    if (lane >= o) upto += y;
  }
  const int b = __ffs(__ballot_sync(0xffffffff, goal < before + upto)) - 1;
  before += __shfl_sync(0xffffffff, upto - mine, b);
  const int end = min(i1, i0 + (b + 1) * block);
#pragma unroll 4
  for (int i = i0 + b * block; i < end; i += 128) {
    u64 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + lane * 4 + k < end ? w(i + lane * 4 + k) : 0;
    u64 sum = x[0] + x[1] + x[2] + x[3];
    const u64 own = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffff, sum, o);
      if (lane >= o) sum += y;
    }
    const uint32_t over = __ballot_sync(0xffffffff, goal < before + sum);
    if (over != 0) {
      if (lane == __ffs(over) - 1) {
        u64 run = before + sum - own + x[0];
        int k = 0;
        if (run <= goal) run += x[1], k = 1;
        if (run <= goal && k == 1) run += x[2], k = 2;
        if (run <= goal && k == 2) k = 3;
        rec[1 + taken] = i + lane * 4 + k;
      }
      return;
    }
    before += __shfl_sync(0xffffffff, sum, 31);
  }
}

// `kernel` on `rows` clusters of n CTAs.
template <typename Args>
int launch_clusters(void (*kernel)(Args), int rows, int n, int threads, size_t smem, cudaStream_t stream, const Args& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * n);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = n;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = zs_pdl_enabled() ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (n > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  cudaLaunchKernelEx(&cfg, kernel, a);
  return cudaGetLastError() == cudaSuccess ? 0 : -2;
}

bool aligned16(const void* p, long long stride) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 4 == 0; }

}  // namespace spec
}  // namespace zs

extern "C" int zs_token_probs(const TokenProbsArgs* args, cudaStream_t stream) {
  using namespace zs::spec;
  const TokenProbsArgs& a = *args;
  if (a.vocab < 1 || a.rows < 0 || a.ld < 0 || a.ld_out < a.vocab || a.temperature == nullptr) return -1;
  if (a.rows == 0) return 0;
  int n = 1;
  while (n < kCluster && (long long)n * kChunk < a.vocab) n *= 2;
  if ((long long)n * kChunk < a.vocab || (long long)a.rows * n > 0x7FFFFFFF) {
    zs_launch(probs_wide_kernel, a.rows, T, 0, stream, a);
    return cudaGetLastError() == cudaSuccess ? 0 : -2;
  }
  const bool vec = aligned16(a.logits, a.rows > 1 ? a.ld : 0) && aligned16(a.out, a.rows > 1 ? a.ld_out : 0);
  return launch_clusters(vec ? probs_kernel<4> : probs_kernel<1>, a.rows, n, PT, sizeof(ProbsSmem), stream, a);
}

extern "C" int zs_draft_verify(const DraftVerifyArgs* args, cudaStream_t stream) {
  using namespace zs::spec;
  const DraftVerifyArgs& a = *args;
  if (a.n < 0 || a.k < 1 || a.k > ZS_VERIFY_MAX_DRAFTS || a.vocab < 1 || a.vocab > (1 << 24)) return -1;
  if (a.n == 0) return 0;
  // CTAs of a sequence: a part of some 8000 tokens keeps one busy, and two fit on an SM; further waves
  // only repeat the latencies (128 sequences of 248320 tokens: 54 us with 2 CTAs each, 67 with 1, 59
  // with 4; 64 sequences: 33 us with 4, 40 with 2, 37 with 8; 32 sequences: 19 us with 8, 22 with 4).
  int n = 1;
  while (n < kCluster && (long long)n * VT * 16 < a.vocab && 2ll * n * a.n <= 148 * 2) n *= 2;
  if ((long long)a.n * n > 0x7FFFFFFF) return -1;
  const bool vec = a.vocab % 4 == 0 && aligned16(a.target, a.target_row) && a.target_seq % 4 == 0 &&
                   (a.draft_probs == nullptr || (aligned16(a.draft_probs, a.draft_row) && a.draft_seq % 4 == 0));
  return launch_clusters(vec ? verify_kernel<4> : verify_kernel<1>, a.n, n, VT, 0, stream, a);
}
