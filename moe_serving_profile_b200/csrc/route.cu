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
// fp32 with a bound on every key's error (own_units). A token whose order that bound does
// not settle (two neighbours of the selection, the last selected and the first
// left out, the last kept and the first dropped group), or that has a NaN key,
// is put aside and selected in 64 bits when its warp is through: about two of
// a thousand tokens of random logits. bf16 logits tie often; without a bias and
// without sums of two keys their order is that of the scores, so they are the
// keys (LOGIT), in words that hold them and the expert exactly, and nothing is
// put aside but what 64 bits may round together: sigmoid of logits above 16,
// exponentials below e^-600, and rows that hold a logit other than zero below
// 2^-30 (of its size, the scores of 0 and 1e-20 are one number, and the lower
// id comes first). 4001 tokens, 160 experts: 18 us with scores as keys, one
// token in ten put aside.
//
// One warp per token. Each group has L = 32 / P lanes, P the power of two >= G;
// lane `sub` of a group holds its experts 4 (sub + L j) .. + 3, j = 0, 1, ...,
// so that a lane reads 16 (fp32) or 8 (bf16) bytes at a time. A key in a lane
// is one word: the float's bits made monotone, their low bits replaced by the
// slot, so that a sort of the lane's keys and the search over the warp move
// words and the winner's place is known from its word.
//
// 16384 tokens of 256 fp32 logits in 8 groups, K = 8: 23 us (3.7 us for one
// token), against 2.8 us for the bytes. 12.6 M warp instructions, which is half
// of that at full issue; the rest is a tail: the average SM is active for two
// thirds of the kernel, since each token put aside takes 12 k cycles after the
// last token of its warp, and few warps have one. With 64-bit keys of only the
// candidates, where a token is met, 25 us. Above 256 experts a lane has 16
// slots (one block an SM): 384 experts 58 us, 512 experts 56 us.
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

// The selection of one token, in lane k < K the k-th expert, with the row's
// largest logit and the reciprocal of its softmax sum (0 and 1 with sigmoid).
struct Selected {
  int e;
  float mx, inv;
};

// In 64 bits throughout: loads and exponentials of the lane's experts side by
// side, since each is a long chain (one after another they took 10 us a token).
template <int NL>
__device__ __noinline__ Selected select64(const RouteParams& p, int t) {
  const int lane = threadIdx.x & 31, L = 1 << p.lsh, g = lane >> p.lsh, sub = lane & (L - 1);
  Selected out{0, 0.f, 1.f};
  float x[NL], bias[NL];
  uint32_t live = 0;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int o = slot_offset(sub, L, i);
    const bool in = g < p.G && o < p.S;
    live |= in ? 1u << i : 0u;
    bias[i] = in && p.bias ? p.bias[g * p.S + o] : 0.f;
  }
  // (one branch for all loads: they are then under way together)
  const long long row = (long long)t * p.ld + g * p.S;
  if (p.bf16) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      x[i] = ((live >> i) & 1u) ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.logits)[row + slot_offset(sub, L, i)])
                                : -INFINITY;
  } else {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      x[i] = ((live >> i) & 1u) ? reinterpret_cast<const float*>(p.logits)[row + slot_offset(sub, L, i)]
                                : -INFINITY;
  }
  double v[NL];
  double mx = 0, sum = 0;
  if (p.softmax) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < NL; ++i) top = fmaxf(top, x[i]);   // not NaN: that comes out of the sum
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    out.mx = top;
    mx = static_cast<double>(top);
  }
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const double a = static_cast<double>(x[i]) - mx;
    v[i] = exp(p.softmax ? a : -a);
  }
  if (!p.softmax) {
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] = __drcp_rn(1.0 + v[i]);
  }
#pragma unroll
  for (int i = 0; i < NL; ++i) sum += ((live >> i) & 1u) ? v[i] : 0.0;
  if (p.softmax) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const double inv = __drcp_rn(sum);
#pragma unroll
    for (int i = 0; i < NL; ++i) v[i] *= inv;
    out.inv = static_cast<float>(inv);
  }
  unsigned long long key[NL];   // 0: no expert, or none that may still be selected
  unsigned long long b1 = 0, b2 = 0;
  double v1 = 0, v2 = 0;        // the best two
  auto put = [&](unsigned long long k, double f) {
    if (k > b1) {
      b2 = b1;
      v2 = v1;
      b1 = k;
      v1 = f;
    } else if (k > b2) {
      b2 = k;
      v2 = f;
    }
  };
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const bool in = (live >> i) & 1u;
    v[i] += static_cast<double>(bias[i]);
    key[i] = in ? order64(v[i]) : 0ull;
    put(key[i], v[i]);
  }
  if (p.keep < p.G) {
#pragma unroll 1
    for (int o = 1; o < L; o <<= 1) {
      const unsigned long long c1 = __shfl_xor_sync(kFull, b1, o), c2 = __shfl_xor_sync(kFull, b2, o);
      const double w1 = __shfl_xor_sync(kFull, v1, o), w2 = __shfl_xor_sync(kFull, v2, o);
      put(c1, w1);
      put(c2, w2);
    }
    const unsigned long long mine = order64(v1 + ((p.top == 2 && p.S > 1) ? v2 : 0.0));
    int rank = 0;
#pragma unroll 8
    for (int h = 0; h < p.G; ++h) {
      const unsigned long long other = __shfl_sync(kFull, mine, h << p.lsh);
      if (other > mine || (other == mine && h < g)) ++rank;
    }
    if (rank >= p.keep) {
#pragma unroll
      for (int i = 0; i < NL; ++i) key[i] = 0;
    }
  }
  // the lane's keys in descending order, equal ones by slot (a stable sort)
  int id[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) id[i] = g * p.S + slot_offset(sub, L, i);
#pragma unroll
  for (int j = 0; j < NL; ++j)
#pragma unroll
    for (int i = j & 1; i + 1 < NL; i += 2) {
      const bool swap = key[i + 1] > key[i];
      const unsigned long long ka = key[i], kb = key[i + 1];
      const int ia = id[i], ib = id[i + 1];
      key[i] = swap ? kb : ka;
      key[i + 1] = swap ? ka : kb;
      id[i] = swap ? ib : ia;
      id[i + 1] = swap ? ia : ib;
    }
#pragma unroll 1
  for (int k = 0; k < p.K; ++k) {
    const uint32_t hi = static_cast<uint32_t>(key[0] >> 32), lo = static_cast<uint32_t>(key[0]);
    const bool top = hi == __reduce_max_sync(kFull, hi);
    const uint32_t most = __reduce_max_sync(kFull, top ? lo : 0u);
    const bool mine = top && lo == most;
    const int best = __reduce_min_sync(kFull, mine ? id[0] : 0x7fffffff);
    if (lane == k) out.e = best;
    if (mine && id[0] == best) {
#pragma unroll
      for (int i = 0; i + 1 < NL; ++i) {
        key[i] = key[i + 1];
        id[i] = id[i + 1];
      }
      key[NL - 1] = 0;
    }
  }
  return out;
}

// ------------------------------------------------------------ fp32 selection
// Monotone map float -> uint32 (not for NaN) and back.
__device__ __forceinline__ uint32_t order32(float f) {
  const uint32_t b = __float_as_uint(f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
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

// Error bounds of the fp32 keys, in units of 2^-23 (a rounding is half a unit
// of its result; ex2.approx and expf are off by 2 at most, rcp.approx by 1).
//   softmax  Shared by the row's scores, through the reciprocal of their sum:
//            additions, at most 11 one after the other (a lane's slots in
//            fours, the fours in pairs, 5 steps over the warp) 5.5; ex2 2; its
//            argument (l - max) log2 e, two roundings and the constant's, 1.12
//            |l - max| in a term, 4.4 in the sum (the mean of |l - max| under
//            the scores is below 3.9 up to 512 experts); the quotient 0.5:
//            12.4. (One after the other, 31 additions of a lane had taken the
//            sum 13.5 units off.) A score of its own: by expf 2, its rounded
//            argument |l - max| / 2 and the product 0.5; by ex2 2.5 and 1.12
//            |l - max|, which is 0.42 of the row's largest score at most.
//   sigmoid  expf 2, sum 0.5, quotient 1; by ex2 2.2 of the score 1.
// Above them second-order terms. The sum with the bias adds half a unit of the
// key; the bound has a whole one, which holds the other key's half where a key
// is compared with the word of one that is left out.
__device__ __forceinline__ float own_units(bool softmax) { return softmax ? 16.f : 8.f; }

// An expert's full-precision values, and a bound on its key's distance from
// the formula's.
struct Pick {
  float x, b, s, key, err;
};

__device__ __forceinline__ Pick eval(const RouteParams& p, int t, int e, float mx, float inv) {
  Pick r;
  r.x = load_logit(p, t, e);
  r.b = p.bias ? p.bias[e] : 0.f;
  const float a = p.softmax ? r.x - mx : r.x;
  r.s = p.softmax ? expf(a) * inv : rcp(1.f + expf(-a));
  r.key = r.s + r.b;
  // below -104 the exp is zero, and so is the first term (-inf as well)
  r.err = (r.s * (own_units(p.softmax) + (p.softmax ? fminf(-a, 128.f) : 0.f)) + fabsf(r.key)) * kUlp + 1e-37f;
  return r;
}

// Zeroes the counts; the selection may begin meanwhile.
__global__ void __launch_bounds__(512) zero_counts_kernel(int* counts, int E) {
  grid_dep_begin();
  if (threadIdx.x < E) counts[threadIdx.x] = 0;
}

// MODE: 0 loads logits one by one, 1 in vectors of four, 2 also has an expert
// in every slot of every lane.
template <int NL, int MODE, bool LOGIT>
__global__ void __launch_bounds__(kThreads, NL <= 8 ? 2 : 1)
    route_grouped_kernel(const __grid_constant__ RouteParams p) {
  constexpr uint32_t kSlots = NL - 1;   // low bits of a word: NL - 1 - slot
  constexpr bool VEC = MODE >= 1, FULL = MODE == 2;
  __shared__ int hist[512];
  const int lane = threadIdx.x & 31;
  const int lsh = p.lsh, L = 1 << lsh;
  const int g = lane >> lsh, sub = lane & (L - 1);
  const int E = p.S * p.G;
  if (!p.zeroed) grid_dep_wait();   // zero_counts_kernel has waited for the logits
  // a block counts in shared memory (16384 tokens adding to one array in global
  // memory took 20 us longer)
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
    bias[i] = !LOGIT && in && p.bias ? p.bias[g * p.S + o] : 0.f;
  }
  auto fetch = [&](int t, float (&x)[NL]) {
    const long long row = (long long)t * p.ld + g * p.S + 4 * sub;
#pragma unroll
    for (int i = 0; i < NL; i += 4) {
      x[i] = x[i + 1] = x[i + 2] = x[i + 3] = -INFINITY;
      const long long at = row + L * i;
      if (VEC) {   // S % 4 == 0: the four slots of a vector are live together
        if (FULL || ((live >> i) & 1u)) {
          if (p.bf16) {
            const uint2 v = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(p.logits) + at);
            x[i] = __uint_as_float(v.x << 16);
            x[i + 1] = __uint_as_float(v.x & 0xffff0000u);
            x[i + 2] = __uint_as_float(v.y << 16);
            x[i + 3] = __uint_as_float(v.y & 0xffff0000u);
          } else {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.logits) + at);
            x[i] = v.x;
            x[i + 1] = v.y;
            x[i + 2] = v.z;
            x[i + 3] = v.w;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((live >> (i + j)) & 1u)
            x[i + j] = load_logit(p, t, g * p.S + slot_offset(sub, L, i + j));
      }
    }
  };

  auto write = [&](int t, int sel, float w) {   // lane k < K: the k-th expert and its score
    const bool mine = lane < p.K;
    if (p.normalize) {
      float sum = mine ? w : 0.f;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
      w *= rcp(sum + 1e-20f);
    }
    if (mine) {
      const long long at = (long long)t * p.K + lane;
      p.scores[at] = w * p.scale;
      p.indices[at] = sel;
      if (p.counts) atomicAdd(&hist[sel], 1);
    }
  };

  const int warps = gridDim.x * (kThreads / 32);
  int first = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  float next[NL];
  if (first < p.T) fetch(first, next);
  while (first < p.T) {   // 32 tokens of the warp at a time
    uint32_t aside = 0;   // those to select in 64 bits
    int t = first;
#pragma unroll 1
    for (int turn = 0; turn < 32 && t < p.T; ++turn, t += warps) {
      float x[NL];
#pragma unroll
      for (int i = 0; i < NL; ++i) x[i] = next[i];
      if (t + warps < p.T) fetch(t + warps, next);   // in flight while this token is selected

      // ---- keys
      constexpr float kLog2e = 1.44269504f;
      float mx = 0.f, inv = 1.f, total = 0.f;
      uint32_t key[NL];
      // Neighbouring bf16 logits a > b differ by 2^-8 |a| or more. From |a| =
      // 2^-30 on that is 2^-40 of a sigmoid (slope 1/4), 2^-38 of an exponential,
      // where 64 bits are off by 2^-51 and (600 + 4) 2^-53. Zeros tie exactly.
      constexpr uint32_t kTiny = 2u * 0x30800000u - 1u;   // 2^-30
      uint32_t least = 0xffffffffu;   // twice the least nonzero magnitude's bits, less one
      if (LOGIT) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          least = min(least, 2u * __float_as_uint(x[i]) - 1u);
          const uint32_t tag = 0xffffu - (g * p.S + slot_offset(sub, L, i));   // equal logits: the lower id first
          total += x[i];
          key[i] = FULL || ((live >> (VEC ? i & ~3 : i)) & 1u) ? (order32(x[i] + 0.f) & 0xffff0000u) | tag : 0u;   // -0 is 0
        }
      }
      if (p.softmax) {
        mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < NL; ++i) mx = fmaxf(mx, x[i]);
        mx = unorder32(__reduce_max_sync(kFull, order32(mx)));
        float part[NL / 4];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          x[i] = ex2((x[i] - mx) * kLog2e);   // 0 in a slot without an expert
          part[i / 4] = i % 4 == 0 ? x[i] : part[i / 4] + x[i];
        }
#pragma unroll
        for (int n = NL / 8; n >= 1; n >>= 1)
#pragma unroll
          for (int i = 0; i < n; ++i) part[i] += part[i + n];
        float sum = part[0];
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        inv = 1.f / sum;
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] *= inv;
      } else {
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] = rcp(1.f + ex2(-kLog2e * x[i]));
      }
      if (!LOGIT) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const float k = x[i] + bias[i];
          total += k;
          key[i] = FULL || ((live >> (VEC ? i & ~3 : i)) & 1u) ? (order32(k) & ~kSlots) | (kSlots - i) : 0u;
        }
      }
      // no NaN key (nor infinite ones of both signs), no tiny logit
      bool sure = !__any_sync(kFull, total != total || (LOGIT && least < kTiny));
      sort_desc(key);
      // whether 64 bits tell the score of logit a (less the largest, softmax; not tiny) from those of smaller ones
      auto apart = [&](float a) { return a > -600.f && (p.softmax || a <= 16.f); };

      // ---- groups. A key's score is off by own_units of the row's largest
      // (`inv` at most), and the key at most NL - 1 units above its word; a sum's
      // word has the group in its low bits. Two sums of two keys are compared
      if (p.keep < p.G) {
        uint32_t k1 = key[0], k2 = key[1];
        for (int o = 1; o < L; o <<= 1) {
          const uint32_t c1 = __shfl_xor_sync(kFull, k1, o), c2 = __shfl_xor_sync(kFull, k2, o);
          k2 = max(min(k1, c1), max(k2, c2));
          k1 = max(k1, c1);
        }
        const uint32_t gmask = (32u >> lsh) - 1;
        const bool real = g < p.G;
        float off = 0.f;
        uint32_t word = 0;
        if (LOGIT) {
          word = real ? (k1 & 0xffff0000u) | (gmask - g) : 0u;
        } else if (real) {
          const float f1 = unorder32(k1 & ~kSlots);
          const float f2 = p.top == 2 && p.S > 1 ? unorder32(k2 & ~kSlots) : 0.f;
          off = (fabsf(f1) + fabsf(f2)) * ((NL + 2) * kUlp) + inv * (4.f * own_units(p.softmax) * kUlp);
          word = (order32(f1 + f2) & ~gmask) | (gmask - g);
        }
        uint32_t low = 0xffffffffu, high = 0;   // the last kept and the first dropped sum
        for (int h = 0; h <= p.keep; ++h) {
          low = high ? high : low;
          high = __reduce_max_sync(kFull, h == 0 || word < low ? word : 0u);
        }
        if (LOGIT) {
          sure = sure && apart(unorder32(low & 0xffff0000u) - mx);
        } else {
          const float most = __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(off)));
          // (infinite sums are not told apart here)
          sure = sure && unorder32(low & ~gmask) - unorder32(high | gmask) > most;
        }
        if (word < low) key[0] = 0;
      }

      // ---- K rounds of the best word; lane k keeps the k-th and where it was
      uint32_t m = 0, wm = 0;
      int src = 0, ws = 0;
      auto best = [&]() {
        m = __reduce_max_sync(kFull, key[0]);   // 0: no expert is left
        // equal words of several lanes have one slot: the first lane's expert is the lowest
        src = __ffs(__ballot_sync(kFull, key[0] == m)) - 1;
      };
#pragma unroll 1
      for (int k = 0; k < p.K; ++k) {
        best();
        if (lane == k) {
          wm = m;
          ws = src;
        }
        if (lane == src) {
#pragma unroll
          for (int i = 0; i + 1 < NL; ++i) key[i] = key[i + 1];
          key[NL - 1] = 0;
        }
      }
      // ---- full-precision keys of the selected, and whether the selection is sure
      const int sel = lane >= p.K ? 0
                      : LOGIT     ? static_cast<int>(0xffffu - (wm & 0xffffu))
                                  : (ws >> lsh) * p.S + slot_offset(ws & (L - 1), L, static_cast<int>(kSlots - (wm & kSlots)));
      const Pick c = eval(p, t, sel, mx, inv);
      if (LOGIT) {
        sure = sure && (lane >= p.K || apart(c.x - mx));
      } else {
        const float nk = __shfl_down_sync(kFull, c.key, 1), ne = __shfl_down_sync(kFull, c.err, 1);
        const float nx = __shfl_down_sync(kFull, c.x, 1), nb = __shfl_down_sync(kFull, c.b, 1);
        const int ni = __shfl_down_sync(kFull, sel, 1);
        const bool ordered = c.key - nk > c.err + ne || (c.x == nx && c.b == nb && sel < ni) || lane >= p.K - 1;
        // the first one left out: no key left is above its word's range
        m = __reduce_max_sync(kFull, key[0]);
        const uint32_t high = m ? order32(__fadd_ru(unorder32(m | kSlots), inv * (own_units(p.softmax) * kUlp))) : 0u;
        sure = sure && ordered && (lane >= p.K || order32(__fsub_rd(c.key, c.err)) > high);
      }
      if (__all_sync(kFull, sure)) write(t, sel, c.s);
      else aside |= 1u << turn;
    }
    while (aside) {
      const int at = first + (__ffs(aside) - 1) * warps;
      aside &= aside - 1;
      const Selected r = select64<NL>(p, at);
      write(at, r.e, eval(p, at, r.e, r.mx, r.inv).s);
    }
    first = t;
  }
  if (p.counts) {
    __syncthreads();
    if (p.zeroed) grid_dep_wait();   // the counts are zero
    for (int e = threadIdx.x; e < E; e += kThreads) {
      const int n = hist[e];
      if (!p.zeroed) p.counts[e] = n;   // the only block
      else if (n) atomicAdd(&p.counts[e], n);
    }
  }
}

}  // namespace

int route_grouped_blocks(int T, int sm_count) {
  const int all = (T + kThreads / 32 - 1) / (kThreads / 32);
  return all < 2 * sm_count ? all : 2 * sm_count;
}

cudaError_t launch_route_grouped(cudaStream_t st, RouteParams p, int blocks) {
  const int L = 1 << p.lsh;
  const int per_lane = 4 * ((p.S + 4 * L - 1) / (4 * L));   // slots of a lane, in fours
  const uintptr_t item = p.bf16 ? 2 : 4;
  const bool vec = p.S % 4 == 0 && p.ld % 4 == 0 && reinterpret_cast<uintptr_t>(p.logits) % (4 * item) == 0;
  const bool logit = p.bf16 && p.bias == nullptr && (p.keep == p.G || p.top == 1 || p.S == 1);
  const bool full = vec && p.S == per_lane * L && p.G * L == 32;
  p.zeroed = blocks > 1 && p.counts;
  if (p.zeroed) {
    cudaError_t e = launch_dependent(zero_counts_kernel, 1, 512, st, p.counts, p.S * p.G);
    if (e != cudaSuccess) return e;
  }
#define B200_ROUTE_MODE(NL_, MODE_)                                                                        \
  return logit ? launch_dependent(route_grouped_kernel<NL_, MODE_, true>, blocks, kThreads, st, p)        \
               : launch_dependent(route_grouped_kernel<NL_, MODE_, false>, blocks, kThreads, st, p)
#define B200_ROUTE(NL_)                                    \
  do {                                                     \
    if (full && per_lane == NL_) B200_ROUTE_MODE(NL_, 2);  \
    if (vec) B200_ROUTE_MODE(NL_, 1);                      \
    B200_ROUTE_MODE(NL_, 0);                               \
  } while (0)
  if (per_lane <= 4) B200_ROUTE(4);
  if (per_lane <= 8) B200_ROUTE(8);
  if (per_lane <= 16) B200_ROUTE(16);
  B200_ROUTE(32);
#undef B200_ROUTE
#undef B200_ROUTE_MODE
}

}  // namespace b200
