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
// infinity: a row that holds one gets a NaN or infinite scale and its products
// come out NaN instead of plausible.
//
// One block per row, the row in registers between the passes.
#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kVec = 4;   // 16-byte vectors per thread

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint32_t mag(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// amax / top, or 1 where that is zero (a row or group of zeros, or of values
// so small that the quotient underflows: they quantise to 0).
__device__ __forceinline__ float scale_of(uint32_t amax, float top) {
  const float s = __fdiv_rn(__uint_as_float(amax), top);
  return s == 0.f ? 1.f : s;
}

__device__ __forceinline__ uint32_t e4m3x2_rn(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x1), "f"(x0));
  return r;
}

__device__ __forceinline__ uint32_t s8_rn(float x) {
  int r;
  asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(r) : "f"(x));
  return static_cast<uint32_t>(r) & 0xffu;
}

__device__ __forceinline__ uint2 pack_s8(const float (&y)[8], float s) {
  uint2 o;
  o.x = s8_rn(__fdiv_rn(y[0], s)) | (s8_rn(__fdiv_rn(y[1], s)) << 8) | (s8_rn(__fdiv_rn(y[2], s)) << 16) |
        (s8_rn(__fdiv_rn(y[3], s)) << 24);
  o.y = s8_rn(__fdiv_rn(y[4], s)) | (s8_rn(__fdiv_rn(y[5], s)) << 8) | (s8_rn(__fdiv_rn(y[6], s)) << 16) |
        (s8_rn(__fdiv_rn(y[7], s)) << 24);
  return o;
}

// Sum / maximum over the block; every thread gets the result. `buf` holds 33
// words and is free again after the call's last barrier.
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

__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const NormParams p) {
  __shared__ float sum_buf[32];
  __shared__ uint32_t max_buf[32];
  const long long t = blockIdx.x;
  const int nvec = p.H >> 3;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.ldx);
  const uint4* r = p.res ? reinterpret_cast<const uint4*>(p.res + t * p.ldr) : nullptr;
  uint4 h[kVec];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    h[i] = make_uint4(0, 0, 0, 0);
    if (v >= nvec) continue;
    h[i] = x[v];
    float f[8];
    unpack8(h[i], f);
    if (r) {
      float g[8];
      unpack8(r[v], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] += g[j];
      h[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                        pack_bf16x2(f[6], f[7]));
      unpack8(h[i], f);
      if (p.res_out) reinterpret_cast<uint4*>(p.res_out + t * p.ldro)[v] = h[i];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(f[j], f[j], sq);
  }
  const float mean = block_sum(sq, sum_buf) / static_cast<float>(p.H);
  const float rstd = 1.f / sqrtf(mean + p.eps);

  uint32_t amax = 0;
  float y[kVec][8];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    unpack8(h[i], y[i]);
    if (v < nvec) {
      float w[8];
      if (p.weight_f32) {
        const float4 a = reinterpret_cast<const float4*>(p.weight)[2 * v];
        const float4 b = reinterpret_cast<const float4*>(p.weight)[2 * v + 1];
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      } else {
        unpack8(reinterpret_cast<const uint4*>(p.weight)[v], w);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[i][j] = y[i][j] * rstd * w[j];
        amax = max(amax, mag(y[i][j]));
      }
      if (p.out)
        reinterpret_cast<uint4*>(p.out + t * p.ldo)[v] =
            make_uint4(pack_bf16x2(y[i][0], y[i][1]), pack_bf16x2(y[i][2], y[i][3]), pack_bf16x2(y[i][4], y[i][5]),
                       pack_bf16x2(y[i][6], y[i][7]));
    }
  }
  if (p.quant == 0) return;
  uint2* q = reinterpret_cast<uint2*>(p.q + t * p.k_pad);
  const int npad = p.k_pad >> 3;
  if (p.quant == 2) {   // int8, one scale per row
    amax = block_max(amax, max_buf);
    const float s = scale_of(amax, 127.f);
    if (threadIdx.x == 0) p.scale[t] = s;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) q[v] = pack_s8(y[i], s);
    }
    for (int v = nvec + threadIdx.x; v < npad; v += blockDim.x) q[v] = make_uint2(0, 0);
    return;
  }
  // e4m3, one scale per 128 columns: 16 neighbouring threads hold a group
  const int groups = (p.k_pad + 127) >> 7;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    uint32_t m = 0;
    if (v < nvec) {
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, mag(y[i][j]));
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
    const float s = scale_of(m, 448.f);
    if (v < nvec) {
      q[v] = make_uint2(e4m3x2_rn(__fdiv_rn(y[i][0], s), __fdiv_rn(y[i][1], s)) |
                            (e4m3x2_rn(__fdiv_rn(y[i][2], s), __fdiv_rn(y[i][3], s)) << 16),
                        e4m3x2_rn(__fdiv_rn(y[i][4], s), __fdiv_rn(y[i][5], s)) |
                            (e4m3x2_rn(__fdiv_rn(y[i][6], s), __fdiv_rn(y[i][7], s)) << 16));
    } else if (v < npad) {
      q[v] = make_uint2(0, 0);
    }
    if ((v & 15) == 0 && (v >> 4) < groups) p.scale[t * groups + (v >> 4)] = s;
  }
  // columns and groups past the vectors that the threads hold
  for (int v = kVec * blockDim.x + threadIdx.x; v < npad; v += blockDim.x) {
    q[v] = make_uint2(0, 0);
    if ((v & 15) == 0) p.scale[t * groups + (v >> 4)] = 1.f;
  }
}

// Where row t's copies go: r itself, or its `copies` places in the permuted
// order, those of the launch's experts only.
__device__ __forceinline__ int dest_row(const QuantInt8Params& p, long long t, int c, int lo, int hi) {
  if (p.inverse == nullptr) return static_cast<int>(t);
  const int d = p.inverse[t * p.copies + c];
  return d >= lo && d < hi ? d : -1;
}

__global__ void __launch_bounds__(1024) act_quant_int8_kernel(const QuantInt8Params p) {
  __shared__ uint32_t max_buf[32];
  const long long t = blockIdx.x;
  const int nvec = p.k_valid >> 3, npad = p.k_pad >> 3;
  int lo = 0, hi = p.rows_out;
  if (p.range) {
    lo = p.range[p.expert_lo];
    hi = min(hi, p.range[p.expert_hi]);
  }
  if (p.inverse == nullptr && (t < lo || t >= hi)) return;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + t * p.ldx);
  uint4 h[kVec];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    h[i] = make_uint4(0, 0, 0, 0);
    if (v < nvec) h[i] = x[v];
    float f[8];
    unpack8(h[i], f);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, mag(f[j]));
  }
  amax = block_max(amax, max_buf);
  const float s = scale_of(amax, 127.f);
  uint2 o[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    float f[8];
    unpack8(h[i], f);
    o[i] = pack_s8(f, s);
  }
  for (int c = 0; c < p.copies; ++c) {
    const int d = dest_row(p, t, c, lo, hi);
    if (d < 0) continue;
    uint2* q = reinterpret_cast<uint2*>(p.q + (long long)d * p.k_pad);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) q[v] = o[i];
    }
    for (int v = nvec + threadIdx.x; v < npad; v += blockDim.x) q[v] = make_uint2(0, 0);
    if (threadIdx.x == 0) p.scale[d] = s;
  }
}

// Rows of 8-bit values with `groups` scales each, copied to their places in
// the permuted order.
__global__ void __launch_bounds__(128) scatter_rows_8bit_kernel(const ScatterRowsParams p) {
  const long long t = blockIdx.x;
  const int nvec = p.row_bytes >> 4;
  int lo = 0, hi = p.rows_out;
  if (p.range) {
    lo = p.range[p.expert_lo];
    hi = min(hi, p.range[p.expert_hi]);
  }
  const uint4* src = reinterpret_cast<const uint4*>(p.q + t * p.row_bytes);
  for (int c = 0; c < p.copies; ++c) {
    const int d = p.inverse[t * p.copies + c];
    if (d < lo || d >= hi) continue;
    uint4* dst = reinterpret_cast<uint4*>(p.out + (long long)d * p.row_bytes);
    for (int v = threadIdx.x; v < nvec; v += blockDim.x) dst[v] = src[v];
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x)
      p.out_scale[(long long)d * p.groups + g] = p.scale[t * p.groups + g];
  }
}

// Threads of a block that holds nvec vectors, kVec per thread at most, a
// multiple of 32.
int row_threads(int nvec) {
  const int per = (nvec + kVec - 1) / kVec;
  const int want = nvec <= 512 ? (nvec + 1) / 2 : per;   // short rows: two vectors a thread
  const int t = ((want > per ? want : per) + 31) / 32 * 32;
  return t < 32 ? 32 : t;
}

}  // namespace

cudaError_t launch_add_rmsnorm(cudaStream_t st, const NormParams& p) {
  add_rmsnorm_kernel<<<p.T, row_threads(p.H >> 3), 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_act_quant_int8(cudaStream_t st, const QuantInt8Params& p) {
  act_quant_int8_kernel<<<p.rows, row_threads(p.k_valid >> 3), 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_scatter_rows_8bit(cudaStream_t st, const ScatterRowsParams& p) {
  scatter_rows_8bit_kernel<<<p.rows, 128, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace b200
