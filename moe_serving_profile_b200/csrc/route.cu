// Grouped expert routing. Per token, with logits l_e of E experts in G groups
// of S = E / G consecutive experts:
//   s_e   = 1 / (1 + exp(-l_e))  or  exp(l_e - max l) / sum exp(l - max l)
//   key_e = s_e + b_e                       (b: balance bias, selection only)
//   G_g   = sum of the group's best 1 or 2 keys; the topk_group best groups
//           stay (equal sums: the lower group)
//   the K best keys of those groups are selected (equal keys: the lower
//   expert id) and written in descending order of their keys
//   w_k   = s_{e_k}, divided by (sum of the K scores + 1e-20) if normalised,
//           times the routing scale
// NaN keys and sums rank above every number.
//
// The selection is the one of the formula in 64-bit arithmetic. It is made in
// fp32 with a bound on every key's error, and a token whose order that bound
// does not settle (two neighbours of the selection, the last selected and the
// first left out, the last kept and the first dropped group) is selected again
// in 64 bits; so is every token with NaN. Of random tokens that is less than
// one in a hundred.
//
// One warp per token. Each group has L = 32 / P lanes, P the power of two >= G;
// lane `sub` of a group holds its experts 4 (sub + L j) .. + 3, j = 0, 1, ...,
// so that a lane reads 16 (fp32) or 8 (bf16) bytes at a time. A key in a lane
// is one word: the float's bits made monotone, their low bits replaced by the
// slot, so that a sort of the lane's keys and the search over the warp move
// words and the winner's place is known from its word.
#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 512;
constexpr float kUlp = 1.1920929e-7f;   // 2^-23

__device__ __forceinline__ float load_logit(const RouteParams& p, int t, int e) {
  const long long at = (long long)t * p.ld + e;
  return p.bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.logits)[at])
                : reinterpret_cast<const float*>(p.logits)[at];
}

// Offset in its group of slot i of lane sub.
__device__ __forceinline__ int slot_offset(int sub, int L, int i) { return 4 * (sub + L * (i >> 2)) + (i & 3); }

// ------------------------------------------------------------ 64-bit selection
// Monotone map double -> uint64; NaN above every number, 0 below everything.
__device__ __forceinline__ unsigned long long order64(double v) {
  if (v != v) return ~0ull;
  const long long b = __double_as_longlong(v + 0.0);   // -0 becomes +0
  return b < 0 ? ~static_cast<unsigned long long>(b) : (static_cast<unsigned long long>(b) | (1ull << 63));
}

// Score in 64 bits; mx and sum: the row's largest logit and softmax sum.
__device__ __forceinline__ double score64(const RouteParams& p, float x, double mx, double sum) {
  const double v = static_cast<double>(x);
  return p.softmax ? exp(v - mx) / sum : 1.0 / (1.0 + exp(-v));
}

// Lane k < K gets the k-th selected expert. Only the keys stay in registers:
// the call is rare, and its registers bound the kernel's.
template <int NL>
__device__ __noinline__ int select64(const RouteParams& p, int t) {
  const int lane = threadIdx.x & 31;
  const int L = 32 / p.P;
  const int g = lane / L, sub = lane % L;
  auto holds = [&](int i) { return g < p.G && slot_offset(sub, L, i) < p.S; };
  auto expert = [&](int i) { return g * p.S + slot_offset(sub, L, i); };
  double mx = -INFINITY, sum = 0;
  if (p.softmax) {
#pragma unroll 1
    for (int i = 0; i < NL; ++i)
      if (holds(i)) {
        const double v = static_cast<double>(load_logit(p, t, expert(i)));
        mx = v > mx ? v : mx;
      }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const double m2 = __shfl_xor_sync(kFull, mx, o);
      mx = m2 > mx ? m2 : mx;
    }
#pragma unroll 1
    for (int i = 0; i < NL; ++i)
      if (holds(i)) sum += exp(static_cast<double>(load_logit(p, t, expert(i))) - mx);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  }
  unsigned long long key[NL];          // 0: no expert, or none that may still be selected
  unsigned long long b1 = 0, b2 = 0;   // the lane's best keys
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
  for (int i = 0; i < NL; ++i) {
    key[i] = 0;
    if (holds(i)) {
      double v = score64(p, load_logit(p, t, expert(i)), mx, sum);
      if (p.bias) v += static_cast<double>(p.bias[expert(i)]);
      key[i] = order64(v);
      put(key[i], v);
    }
  }
  if (p.keep < p.G) {
    for (int o = 1; o < L; o <<= 1) {
      const unsigned long long c1 = __shfl_xor_sync(kFull, b1, o), c2 = __shfl_xor_sync(kFull, b2, o);
      const double w1 = __shfl_xor_sync(kFull, v1, o), w2 = __shfl_xor_sync(kFull, v2, o);
      put(c1, w1);
      put(c2, w2);
    }
    const unsigned long long mine = order64(v1 + ((p.top == 2 && p.S > 1) ? v2 : 0.0));
    int rank = 0;
    for (int h = 0; h < p.G; ++h) {
      const unsigned long long other = __shfl_sync(kFull, mine, h * L);
      if (other > mine || (other == mine && h < g)) ++rank;
    }
    if (rank >= p.keep) {
#pragma unroll
      for (int i = 0; i < NL; ++i) key[i] = 0;
    }
  }
  int sel = 0;
#pragma unroll 1
  for (int k = 0; k < p.K; ++k) {
    unsigned long long bk = 0;
    int bi = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (key[i] > bk) {
        bk = key[i];
        bi = expert(i);
      }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
      const unsigned long long k2 = __shfl_xor_sync(kFull, bk, o);
      const int i2 = __shfl_xor_sync(kFull, bi, o);
      if (k2 > bk || (k2 == bk && i2 < bi)) {
        bk = k2;
        bi = i2;
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (bi == expert(i) && holds(i)) key[i] = 0;
    if (lane == k) sel = bi;
  }
  return sel;
}

// ------------------------------------------------------------ fp32 selection
// Monotone map float -> uint32 and back; NaN above every number.
__device__ __forceinline__ uint32_t order32(float f) {
  const uint32_t b = __float_as_uint(f);
  const uint32_t u = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return f != f ? 0xffffffffu : u;
}
__device__ __forceinline__ float unorder32(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u ^ 0x80000000u) : ~u);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Descending order of a lane's words: Batcher's odd-even merge sort.
template <int N>
__device__ __forceinline__ void sort_desc(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p <<= 1)
#pragma unroll
    for (int q = p; q >= 1; q >>= 1)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + q];
            k[i + j] = max(a, b);
            k[i + j + q] = min(a, b);
          }
}

// A selected expert's full-precision values in lane k, and the bound on its
// key's distance from the formula's: s (the exp's argument is rounded once,
// 2^-24 of it; exp, sum and quotient a few units) and the sum with the bias.
struct Pick {
  float x, b, s, key, err;
};

__device__ __forceinline__ Pick eval(const RouteParams& p, int t, int e, float mx, float inv) {
  Pick r;
  r.x = load_logit(p, t, e);
  r.b = p.bias ? p.bias[e] : 0.f;
  const float a = p.softmax ? r.x - mx : r.x;
  r.s = p.softmax ? expf(a) * inv : 1.f / (1.f + expf(-a));
  r.key = r.s + r.b;
  r.err = (r.s * (16.f + fmaxf(-a, 0.f)) + fabsf(r.key)) * kUlp + 1e-37f;
  return r;
}

template <int NL, bool VEC>
__global__ void __launch_bounds__(kThreads, NL <= 8 ? 2 : 1)
    route_grouped_kernel(const __grid_constant__ RouteParams p) {
  constexpr uint32_t kSlots = NL - 1;   // low bits of a word: NL - 1 - slot
  __shared__ int hist[512];
  const int lane = threadIdx.x & 31;
  const int L = 32 / p.P;
  const int g = lane / L, sub = lane & (L - 1);
  const int E = p.S * p.G;
  if (p.counts) {
    for (int e = threadIdx.x; e < E; e += kThreads) hist[e] = 0;
    __syncthreads();
  }
  uint32_t live = 0;   // slots that hold an expert
  float bias[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int o = slot_offset(sub, L, i);
    const bool in = g < p.G && o < p.S;
    live |= in ? 1u << i : 0u;
    bias[i] = in && p.bias ? p.bias[g * p.S + o] : 0.f;
  }
  const int warps = gridDim.x * (kThreads / 32);
  for (int t = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); t < p.T; t += warps) {
    // ---- keys
    float x[NL];
    if (VEC) {   // S % 4 == 0: the four slots of a vector are live together
#pragma unroll
      for (int i = 0; i < NL; i += 4) {
        x[i] = x[i + 1] = x[i + 2] = x[i + 3] = -INFINITY;
        if ((live >> i) & 1u) {
          const long long at = (long long)t * p.ld + g * p.S + slot_offset(sub, L, i);
          if (p.bf16) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p.logits) + at));
            x[i] = __uint_as_float(v.x << 16);
            x[i + 1] = __uint_as_float(v.x & 0xffff0000u);
            x[i + 2] = __uint_as_float(v.y << 16);
            x[i + 3] = __uint_as_float(v.y & 0xffff0000u);
          } else {
            const float4 v = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.logits) + at));
            x[i] = v.x;
            x[i + 1] = v.y;
            x[i + 2] = v.z;
            x[i + 3] = v.w;
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i)
        x[i] = ((live >> i) & 1u) ? load_logit(p, t, g * p.S + slot_offset(sub, L, i)) : -INFINITY;
    }
    constexpr float kLog2e = 1.44269504f;
    float mx = 0.f, inv = 1.f;
    if (p.softmax) {
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NL; ++i) mx = fmaxf(mx, x[i]);
      mx = unorder32(__reduce_max_sync(kFull, order32(mx)));
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        x[i] = ex2((x[i] - mx) * kLog2e);
        sum += ((live >> i) & 1u) ? x[i] : 0.f;
      }
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      inv = 1.f / sum;
#pragma unroll
      for (int i = 0; i < NL; ++i) x[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) x[i] = rcp(1.f + ex2(-kLog2e * x[i]));
    }
    uint32_t key[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i)
      key[i] = ((live >> i) & 1u) ? (order32(x[i] + bias[i]) & ~kSlots) | (kSlots - i) : 0u;
    sort_desc(key);
    bool sure = true;

    // ---- groups: a key is off by at most 2^-19 of the row's largest score
    // (its approximations) and 2^-23 NL of itself (its low bits)
    if (p.keep < p.G) {
      uint32_t k1 = key[0], k2 = key[1];
      for (int o = 1; o < L; o <<= 1) {
        const uint32_t c1 = __shfl_xor_sync(kFull, k1, o), c2 = __shfl_xor_sync(kFull, k2, o);
        k2 = max(min(k1, c1), max(k2, c2));
        k1 = max(k1, c1);
      }
      const float f1 = unorder32(k1 & ~kSlots);
      const float f2 = p.top == 2 && p.S > 1 ? unorder32(k2 & ~kSlots) : 0.f;
      const float total = f1 + f2;
      const float off = (fabsf(f1) + fabsf(f2)) * ((NL + 2) * kUlp) + inv * (32.f * kUlp);
      int rank = 0;
      for (int h = 0; h < p.G; ++h) {
        const float other = __shfl_sync(kFull, total, h * L);
        rank += other > total || (other == total && h < g) ? 1 : 0;
      }
      const bool kept = rank < p.keep, real = g < p.G;
      const uint32_t low = __reduce_min_sync(kFull, real && kept ? order32(total - off) : 0xffffffffu);
      const uint32_t high = __reduce_max_sync(kFull, real && !kept ? order32(total + off) : 0u);
      // NaN and infinite sums are compared in 64 bits
      sure = low > high && !__any_sync(kFull, real && !(fabsf(total) + off < INFINITY));
      if (!kept) key[0] = 0;
    }

    // ---- K rounds of the best word, and the first one left out
    int sel = 0, border = -1;
#pragma unroll 1
    for (int k = 0; k <= p.K; ++k) {
      const uint32_t m = __reduce_max_sync(kFull, key[0]);
      if (m == 0) break;   // every expert of the kept groups is selected
      const int src = __ffs(__ballot_sync(kFull, key[0] == m)) - 1;
      const int slot = kSlots - (m & kSlots);
      const int e = (src / L) * p.S + slot_offset(src & (L - 1), L, slot);
      if (k == p.K) {
        border = e;
        break;
      }
      if (lane == k) sel = e;   // equal words of several lanes have one slot: the first lane's expert is the lowest
      if (lane == src) {
#pragma unroll
        for (int i = 0; i + 1 < NL; ++i) key[i] = key[i + 1];
        key[NL - 1] = 0;
      }
    }

    // ---- full-precision keys of the selected, and whether their order is sure
    Pick c = eval(p, t, lane < p.K ? sel : (border >= 0 ? border : sel), mx, inv);
    auto ordered = [&]() {
      const float nk = __shfl_down_sync(kFull, c.key, 1), ne = __shfl_down_sync(kFull, c.err, 1);
      const float nx = __shfl_down_sync(kFull, c.x, 1), nb = __shfl_down_sync(kFull, c.b, 1);
      const int ni = __shfl_down_sync(kFull, sel, 1);
      bool ok = c.key - nk > c.err + ne || (c.x == nx && c.b == nb && sel < ni);
      return __all_sync(kFull, ok || lane >= p.K - 1);
    };
    if (!ordered()) {
      // the low bits that the words lack: rank the selected by their keys
      int rank = 0;
      for (int j = 0; j < p.K; ++j) {
        const float kj = __shfl_sync(kFull, c.key, j);
        const int ij = __shfl_sync(kFull, sel, j);
        rank += kj > c.key || (kj == c.key && ij < sel) ? 1 : 0;
      }
      int from = lane;
      for (int j = 0; j < p.K; ++j) {
        const int rj = __shfl_sync(kFull, rank, j);
        if (rj == lane && lane < p.K) from = j;
      }
      sel = __shfl_sync(kFull, sel, from);
      c.x = __shfl_sync(kFull, c.x, from);
      c.b = __shfl_sync(kFull, c.b, from);
      c.s = __shfl_sync(kFull, c.s, from);
      c.key = __shfl_sync(kFull, c.key, from);
      c.err = __shfl_sync(kFull, c.err, from);
      sure = ordered() && sure;
    }
    if (border >= 0) {
      // the first one left out stands for all of them: their words are not
      // above its word, their keys at most its low bits above its key
      Pick n;
      if (p.K < 32) {
        n.key = __shfl_sync(kFull, c.key, p.K);
        n.err = __shfl_sync(kFull, c.err, p.K);
      } else {
        n = eval(p, t, border, mx, inv);
      }
      const float last = __shfl_sync(kFull, c.key, p.K - 1), le = __shfl_sync(kFull, c.err, p.K - 1);
      sure = sure && last - n.key > le + n.err + fabsf(n.key) * (2 * NL * kUlp) + inv * (32.f * kUlp);
    } else {
      sure = sure && __all_sync(kFull, c.key == c.key);
    }
    if (!sure) {
      sel = select64<NL>(p, t);
      c = eval(p, t, sel, mx, inv);
    }
    float w = c.s;

    const bool mine = lane < p.K;
    if (p.normalize) {
      float sum = mine ? w : 0.f;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      w /= sum + 1e-20f;
    }
    if (mine) {
      p.scores[(long long)t * p.K + lane] = w * p.scale;
      p.indices[(long long)t * p.K + lane] = sel;
      if (p.counts) atomicAdd(&hist[sel], 1);
    }
  }
  if (p.counts) {
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += kThreads) {
      const int n = hist[e];
      if (gridDim.x == 1) p.counts[e] = n;
      else if (n) atomicAdd(&p.counts[e], n);
    }
  }
}

}  // namespace

int route_grouped_blocks(int T, int sm_count) {
  const int all = (T + kThreads / 32 - 1) / (kThreads / 32);
  return all < 2 * sm_count ? all : 2 * sm_count;
}

cudaError_t launch_route_grouped(cudaStream_t st, const RouteParams& p, int blocks) {
  const int L = 32 / p.P;
  const int per_lane = 4 * ((p.S + 4 * L - 1) / (4 * L));   // slots of a lane, in fours
  const uintptr_t item = p.bf16 ? 2 : 4;
  const bool vec = p.S % 4 == 0 && p.ld % 4 == 0 && reinterpret_cast<uintptr_t>(p.logits) % (4 * item) == 0;
#define B200_ROUTE(NL_)                                                    \
  do {                                                                     \
    if (vec) route_grouped_kernel<NL_, true><<<blocks, kThreads, 0, st>>>(p); \
    else route_grouped_kernel<NL_, false><<<blocks, kThreads, 0, st>>>(p);    \
  } while (0)
  if (per_lane <= 4) B200_ROUTE(4);
  else if (per_lane <= 8) B200_ROUTE(8);
  else if (per_lane <= 16) B200_ROUTE(16);
  else B200_ROUTE(32);
#undef B200_ROUTE
  return cudaGetLastError();
}

}  // namespace b200
