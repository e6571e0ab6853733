// Grouped expert routing. Per token, with logits l_e of E experts in G groups
// of S = E / G consecutive experts:
//   s_e   = 1 / (1 + exp(-l_e))  or  exp(l_e - max l) / sum exp(l - max l)
//   key_e = s_e + b_e                       (b: balance bias, selection only)
//   G_g   = sum of the group's best 1 or 2 keys; the topk_group best groups
//           stay (equal sums: the lower group)
//   the K best keys of those groups are selected (equal keys: the lower
//   expert id) and written in descending order of their keys
//   w_k   = s_{e_k}, divided by (sum of the K scores + 1e-20) if normalised,
//           times the routing scale, rounded once to fp32
// NaN keys and sums rank above every number. Scores, keys and sums are held
// in 64 bits, so that a selection is the one of the formula and not of one
// rounding of it.
//
// One warp per token. Each group has 32 / P lanes, P the power of two >= G;
// lane `sub` of a group holds its experts sub, sub + L, ... (L = 32 / P), at
// most NL of them.
#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;

// Monotone map double -> uint64; NaN above every number, 0 below everything.
__device__ __forceinline__ unsigned long long order64(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);   // -0 becomes +0
  return b < 0 ? ~static_cast<unsigned long long>(b) : (static_cast<unsigned long long>(b) | (1ull << 63));
}

// Best (key, then lowest index) over the warp.
__device__ __forceinline__ void warp_best(unsigned long long& key, int& idx) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    const unsigned long long k2 = __shfl_xor_sync(kFull, key, o);
    const int i2 = __shfl_xor_sync(kFull, idx, o);
    if (k2 > key || (k2 == key && i2 < idx)) {
      key = k2;
      idx = i2;
    }
  }
}

template <int NL>
__global__ void __launch_bounds__(256) route_grouped_kernel(const RouteParams p) {
  const int t = (blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (t >= p.T) return;
  const int L = 32 / p.P;               // lanes per group
  const int g = lane / L, sub = lane % L;
  const bool live = g < p.G;

  double score[NL], key[NL];
  double mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int o = sub + L * i;
    double v = -INFINITY;
    if (live && o < p.S) {
      const long long at = (long long)t * p.ld + g * p.S + o;
      v = p.bf16 ? static_cast<double>(__bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.logits)[at]))
                 : static_cast<double>(reinterpret_cast<const float*>(p.logits)[at]);
    }
    score[i] = v;
    mx = v > mx ? v : mx;
  }
  if (p.softmax) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const double m2 = __shfl_xor_sync(kFull, mx, o);
      mx = m2 > mx ? m2 : mx;
    }
    double sum = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int o = sub + L * i;
      score[i] = (live && o < p.S) ? exp(score[i] - mx) : 0.0;
      sum += score[i];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
#pragma unroll
    for (int i = 0; i < NL; ++i) score[i] /= sum;
  } else {
#pragma unroll
    for (int i = 0; i < NL; ++i) score[i] = 1.0 / (1.0 + exp(-score[i]));
  }
  uint32_t open = 0;   // bit i: this lane's expert i may still be selected
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int o = sub + L * i;
    if (live && o < p.S) {
      open |= 1u << i;
      key[i] = p.bias ? score[i] + static_cast<double>(p.bias[g * p.S + o]) : score[i];
    } else {
      key[i] = 0;
    }
  }

  if (p.keep < p.G) {
    // ---- the group's best keys, then the best groups
    unsigned long long b1 = 0, b2 = 0;
    double v1 = 0, v2 = 0;
    auto put = [&](unsigned long long k, double v) {
      if (k > b1) {
        b2 = b1;
        v2 = v1;
        b1 = k;
        v1 = v;
      } else if (k > b2) {
        b2 = k;
        v2 = v;
      }
    };
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if ((open >> i) & 1u) put(order64(key[i]), key[i]);
    for (int o = 1; o < L; o <<= 1) {
      const unsigned long long c1 = __shfl_xor_sync(kFull, b1, o), c2 = __shfl_xor_sync(kFull, b2, o);
      const double w1 = __shfl_xor_sync(kFull, v1, o), w2 = __shfl_xor_sync(kFull, v2, o);
      put(c1, w1);
      put(c2, w2);
    }
    const double total = v1 + ((p.top == 2 && p.S > 1) ? v2 : 0.0);
    const unsigned long long mine = order64(total);
    int rank = 0;
    for (int h = 0; h < p.G; ++h) {
      const unsigned long long other = __shfl_sync(kFull, mine, h * L);
      if (other > mine || (other == mine && h < g)) ++rank;
    }
    if (rank >= p.keep) open = 0;
  }

  // ---- K rounds of the best open key
  int sel = 0;
  double w = 0;
  for (int k = 0; k < p.K; ++k) {
    unsigned long long bk = 0;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      if ((open >> i) & 1u) {
        const unsigned long long c = order64(key[i]);
        if (c > bk || bi == 0x7fffffff) {
          bk = c;
          bi = g * p.S + sub + L * i;
        }
      }
    }
    warp_best(bk, bi);
    double got = 0;
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (live && bi == g * p.S + sub + L * i && sub + L * i < p.S) {
        got = score[i];
        open &= ~(1u << i);
      }
    got = __shfl_sync(kFull, got, (bi / p.S) * L + (bi % p.S) % L);
    if (lane == k) {
      sel = bi;
      w = got;
    }
  }
  const bool mine = lane < p.K;
  if (p.normalize) {
    double sum = mine ? w : 0.0;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    w /= sum + 1e-20;
  }
  if (mine) {
    p.scores[(long long)t * p.K + lane] = static_cast<float>(w * static_cast<double>(p.scale));
    p.indices[(long long)t * p.K + lane] = sel;
    if (p.counts) atomicAdd(&p.counts[sel], 1);
  }
}

}  // namespace

cudaError_t launch_route_grouped(cudaStream_t st, const RouteParams& p) {
  const int per_lane = (p.S * p.P + 31) / 32;   // ceil(S / L), L = 32 / P
  const int blocks = (p.T + 7) / 8;
  if (per_lane <= 4) route_grouped_kernel<4><<<blocks, 256, 0, st>>>(p);
  else if (per_lane <= 8) route_grouped_kernel<8><<<blocks, 256, 0, st>>>(p);
  else if (per_lane <= 16) route_grouped_kernel<16><<<blocks, 256, 0, st>>>(p);
  else route_grouped_kernel<32><<<blocks, 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace b200
