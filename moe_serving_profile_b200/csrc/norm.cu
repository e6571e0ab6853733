// Row norms and row quantisers of the 8-bit paths.
//
// add_rmsnorm, per row: h = bf16(x + r) (the new residual, in the residual
// stream's own type; the norm reads the stored value, so a later reader of
// the residual sees what was normed), y = h * rsqrt(mean h^2 + eps) * w in
// fp32, out = bf16(y), and an 8-bit copy of y itself (not of its rounding):
//   e4m3: s_g = amax_g / 448 per 128 columns, q = e4m3(y / s_g) (nearest
//         even, saturating), s_g = 1 for a group of zeros
//   int8: s = amax / 127 per row, q = nearest even of y / s, s = 1 for a row
//         of zeros
// act_quant_int8: the int8 part for bf16 rows, each written to its `copies`
// places of the permuted order.
// amax is an unsigned maximum of the magnitudes' bits, which ranks NaN above
// infinity above every number. A row (group) that holds NaN or an infinity has
// values that no 8-bit code times a scale can stand for: its scale is NaN, and
// all its products come out NaN instead of plausible.
//
// Bound by memory: one block per row holds it in registers between the passes
// (V vectors of 8 columns per thread), all its loads issued before the first
// use. Quotients by the row's or group's scale are correctly rounded by
// Markstein's method (a rounded reciprocal, then two remainder steps): five
// multiply-adds a value, where a general division took most of the time of
// an earlier form of these kernels. Measured: 16384 x 4096 with residual, e4m3
// and bf16 output 93 us (6.5 TB/s); 8191 x 4096 with int8 output only 44 us
// (5.4 TB/s; with the weight loaded again in each pass 46 us); act_quant_int8
// of 8191 x 4096 22 us (4.6 TB/s).
#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

__device__ __forceinline__ uint32_t mag(float f) { return __float_as_uint(f) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t mag_max(const float (&f)[8], uint32_t m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, mag(f[j]));
  return m;
}

// Division by one scale: s = amax / top, 1 where that is zero (a row or group
// of zeros, or of values so small that the quotient underflows: they quantise
// to 0). The scale that is stored is NaN where s is not finite.
struct Divider {
  float s, r, top;
  bool plain;   // magnitudes at which the remainder steps could underflow, infinity and NaN
  __device__ __forceinline__ Divider(uint32_t amax, float top_) : top(top_) {
    s = __fdiv_rn(__uint_as_float(amax), top);
    s = s == 0.f ? 1.f : s;
    r = __frcp_rn(s);
    plain = !(s > 0x1p-80f && s < 0x1p125f);
  }
  __device__ __forceinline__ float stored() const { return s < INFINITY ? s : __uint_as_float(0x7fffffffu); }
  __device__ __forceinline__ float operator()(float x) const {
    if (plain) return fminf(fmaxf(__fdiv_rn(x, s), -top), top);   // a subnormal scale may be short of amax / top
    float t = x * r;
    t = fmaf(fmaf(-t, s, x), r, t);
    return fmaf(fmaf(-t, s, x), r, t);
  }
};

__device__ __forceinline__ uint32_t e4m3x2_rn(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}

__device__ __forceinline__ uint2 pack_e4m3(const float (&y)[8], const Divider& d) {
  return make_uint2(e4m3x2_rn(d(y[0]), d(y[1])) | (e4m3x2_rn(d(y[2]), d(y[3])) << 16),
                    e4m3x2_rn(d(y[4]), d(y[5])) | (e4m3x2_rn(d(y[6]), d(y[7])) << 16));
}

// Four values of at most 127 in magnitude to int8, nearest even: adding
// 1.5 * 2^23 leaves the integer in the sum's low byte.
__device__ __forceinline__ uint32_t s8x4(float a, float b, float c, float e) {
  constexpr float kMagic = 12582912.f;
  const uint32_t ab = __byte_perm(__float_as_uint(a + kMagic), __float_as_uint(b + kMagic), 0x0040);
  const uint32_t ce = __byte_perm(__float_as_uint(c + kMagic), __float_as_uint(e + kMagic), 0x0040);
  return __byte_perm(ab, ce, 0x5410);
}

__device__ __forceinline__ uint2 pack_s8(const float (&y)[8], const Divider& d) {
  return make_uint2(s8x4(d(y[0]), d(y[1]), d(y[2]), d(y[3])), s8x4(d(y[4]), d(y[5]), d(y[6]), d(y[7])));
}

// Sum / maximum over the block; every thread gets the result. `buf` (32 words)
// serves one call.
__device__ __forceinline__ float block_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = (threadIdx.x & 31) < nw ? buf[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
  return s;
}

__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* buf) {
  v = __reduce_max_sync(kFull, v);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(kFull, (threadIdx.x & 31) < nw ? buf[threadIdx.x & 31] : 0u);
}

// ROW8: the int8 form, whose one scale per row takes a second pass over it.
template <int V, bool ROW8>
__global__ void __launch_bounds__(V == 4 ? 1024 : 256) add_rmsnorm_kernel(const NormParams p) {
  __shared__ float sum_buf[32];
  __shared__ uint32_t max_buf[32];
  grid_dep_begin();
  const long long t = blockIdx.x;
  const int nvec = p.H >> 3;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.ldx);
  const uint4* r = p.res ? reinterpret_cast<const uint4*>(p.res + t * p.ldr) : nullptr;
  uint4 h[V], add[V], wv[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    h[i] = add[i] = wv[i] = make_uint4(0, 0, 0, 0);
    if (v < nvec) {
      h[i] = x[v];
      if (r) add[i] = r[v];
      if (!p.weight_f32) wv[i] = reinterpret_cast<const uint4*>(p.weight)[v];
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    float f[8];
    unpack8(h[i], f);
    if (r) {
      float g[8];
      unpack8(add[i], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += g[j];
      h[i] = pack8(f);
      unpack8(h[i], f);
      if (p.res_out && v < nvec) reinterpret_cast<uint4*>(p.res_out + t * p.ldro)[v] = h[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(f[j], f[j], sq);
  }
  const float mean = block_sum(sq, sum_buf) / static_cast<float>(p.H);
  const float rstd = 1.f / sqrtf(mean + p.eps);

  auto normed = [&](int i, float (&y)[8]) {   // zeros past the row's end
    const int v = threadIdx.x + i * blockDim.x;
    float w[8];
    unpack8(h[i], y);
    if (p.weight_f32) {
      if (v >= nvec) return;
      const float4 a = reinterpret_cast<const float4*>(p.weight)[2 * v];
      const float4 b = reinterpret_cast<const float4*>(p.weight)[2 * v + 1];
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
      unpack8(wv[i], w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = y[j] * rstd * w[j];
  };
  uint2* q = reinterpret_cast<uint2*>(p.q + t * p.k_pad);
  const int npad = p.k_pad >> 3;
  if (!ROW8) {
    // e4m3, one scale per 128 columns: 16 neighbouring threads hold a group
    const int groups = (p.k_pad + 127) >> 7;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      float y[8];
      normed(i, y);
      if (p.out && v < nvec) reinterpret_cast<uint4*>(p.out + t * p.ldo)[v] = pack8(y);
      if (p.quant == 0) continue;
      uint32_t m = v < nvec ? mag_max(y, 0) : 0u;
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
      const Divider d(m, 448.f);
      if (v < nvec) q[v] = pack_e4m3(y, d);
      else if (v < npad) q[v] = make_uint2(0, 0);
      if ((v & 15) == 0 && (v >> 4) < groups) p.scale[t * groups + (v >> 4)] = d.stored();
    }
    if (p.quant == 0) return;
    // columns and groups past the vectors that the threads hold
    for (int v = V * blockDim.x + threadIdx.x; v < npad; v += blockDim.x) {
      q[v] = make_uint2(0, 0);
      if ((v & 15) == 0) p.scale[t * groups + (v >> 4)] = 1.f;
    }
    return;
  }
  // int8, one scale per row
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    float y[8];
    normed(i, y);
    if (v < nvec) {
      amax = mag_max(y, amax);
      if (p.out) reinterpret_cast<uint4*>(p.out + t * p.ldo)[v] = pack8(y);
    }
  }
  const Divider d(block_max(amax, max_buf), 127.f);
  if (threadIdx.x == 0) p.scale[t] = d.stored();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    float y[8];
    normed(i, y);   // again: eight registers less per vector
    if (v < nvec) q[v] = pack_s8(y, d);
  }
  for (int v = nvec + threadIdx.x; v < npad; v += blockDim.x) q[v] = make_uint2(0, 0);
}

// The places in the permuted order of 32 copies of row t, from copy c0 on: lane
// c holds that of copy c0 + c, -1 for a place outside [lo, hi).
__device__ __forceinline__ int dest_rows(const int* inverse, long long t, int c0, int copies, int lo, int hi) {
  const int c = c0 + (threadIdx.x & 31);
  const int d = c < copies ? inverse[t * copies + c] : -1;
  return d >= lo && d < hi ? d : -1;
}

template <int V>
__global__ void __launch_bounds__(V == 4 ? 1024 : 256) act_quant_int8_kernel(const QuantInt8Params p) {
  __shared__ uint32_t max_buf[32];
  grid_dep_begin();
  const long long t = blockIdx.x;
  const int nvec = p.k_valid >> 3, npad = p.k_pad >> 3;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.ldx);
  uint4 h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    h[i] = v < nvec ? x[v] : make_uint4(0, 0, 0, 0);
  }
  int lo = 0, hi = p.rows_out;
  if (p.range) {
    lo = p.range[p.expert_lo];
    hi = min(hi, p.range[p.expert_hi]);
  }
  int dest = t >= lo && t < hi ? static_cast<int>(t) : -1;
  if (p.inverse) dest = dest_rows(p.inverse, t, 0, p.copies, lo, hi);
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float f[8];
    unpack8(h[i], f);
    amax = mag_max(f, amax);
  }
  const Divider d(block_max(amax, max_buf), 127.f);
  uint2 o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float f[8];
    unpack8(h[i], f);
    o[i] = pack_s8(f, d);
  }
  for (int c0 = 0; c0 < p.copies; c0 += 32) {
    if (c0) dest = dest_rows(p.inverse, t, c0, p.copies, lo, hi);
    for (int c = 0; c < min(32, p.copies - c0); ++c) {
      const int at = __shfl_sync(kFull, dest, c);
      if (at < 0) continue;
      uint2* q = reinterpret_cast<uint2*>(p.q + (long long)at * p.k_pad);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < nvec) q[v] = o[i];
      }
      for (int v = nvec + threadIdx.x; v < npad; v += blockDim.x) q[v] = make_uint2(0, 0);
      if (threadIdx.x == 0) p.scale[at] = d.stored();
    }
  }
}

// Rows of 8-bit values with `groups` scales each, copied to their places in
// the permuted order.
__global__ void __launch_bounds__(128) scatter_rows_8bit_kernel(const ScatterRowsParams p) {
  grid_dep_begin();
  const long long t = blockIdx.x;
  const int nvec = p.row_bytes >> 4;
  int lo = 0, hi = p.rows_out;
  if (p.range) {
    lo = p.range[p.expert_lo];
    hi = min(hi, p.range[p.expert_hi]);
  }
  const uint4* src = reinterpret_cast<const uint4*>(p.q + t * p.row_bytes);
  for (int c0 = 0; c0 < p.copies; c0 += 32) {
    const int dest = dest_rows(p.inverse, t, c0, p.copies, lo, hi);
    const int n = min(32, p.copies - c0);
    for (int v = threadIdx.x; v < (nvec + 31) / 32 * 32; v += blockDim.x) {   // whole warps: the copies are traded
      const uint4 val = v < nvec ? src[v] : make_uint4(0, 0, 0, 0);
      for (int c = 0; c < n; ++c) {
        const int at = __shfl_sync(kFull, dest, c);
        if (at >= 0 && v < nvec) reinterpret_cast<uint4*>(p.out + (long long)at * p.row_bytes)[v] = val;
      }
    }
    for (int c = 0; c < n; ++c) {
      const int at = __shfl_sync(kFull, dest, c);
      if (at < 0) continue;
      for (int g = threadIdx.x; g < p.groups; g += blockDim.x)
        p.out_scale[(long long)at * p.groups + g] = p.scale[t * p.groups + g];
    }
  }
}

// Vectors per thread: one for rows of up to 128 vectors, two up to 256, four
// beyond, so that small blocks hold several rows on an SM (16384 x 4096 with
// e4m3: one vector 121 us, two 98 us, four 93 us).
int row_vecs(int nvec) { return nvec <= 128 ? 1 : (nvec <= 256 ? 2 : 4); }
int row_threads(int nvec, int v) { return ((nvec + v - 1) / v + 31) / 32 * 32; }

}  // namespace

cudaError_t launch_add_rmsnorm(cudaStream_t st, const NormParams& p) {
  const int v = row_vecs(p.H >> 3), n = row_threads(p.H >> 3, v);
  if (p.quant == 2) {
    if (v == 1) return launch_dependent(add_rmsnorm_kernel<1, true>, p.T, n, st, p);
    if (v == 2) return launch_dependent(add_rmsnorm_kernel<2, true>, p.T, n, st, p);
    return launch_dependent(add_rmsnorm_kernel<4, true>, p.T, n, st, p);
  }
  if (v == 1) return launch_dependent(add_rmsnorm_kernel<1, false>, p.T, n, st, p);
  if (v == 2) return launch_dependent(add_rmsnorm_kernel<2, false>, p.T, n, st, p);
  return launch_dependent(add_rmsnorm_kernel<4, false>, p.T, n, st, p);
}

cudaError_t launch_act_quant_int8(cudaStream_t st, const QuantInt8Params& p) {
  const int v = row_vecs(p.k_valid >> 3), n = row_threads(p.k_valid >> 3, v);
  if (v == 1) return launch_dependent(act_quant_int8_kernel<1>, p.rows, n, st, p);
  if (v == 2) return launch_dependent(act_quant_int8_kernel<2>, p.rows, n, st, p);
  return launch_dependent(act_quant_int8_kernel<4>, p.rows, n, st, p);
}

cudaError_t launch_scatter_rows_8bit(cudaStream_t st, const ScatterRowsParams& p) {
  return launch_dependent(scatter_rows_8bit_kernel, p.rows, 128, st, p);
}

}  // namespace b200
