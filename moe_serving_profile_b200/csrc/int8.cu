// Int8 grouped GEMM: int8 token rows with one scale each times int8 expert
// weights with one scale per output channel, on the tensor cores
// (tcgen05.mma kind::i8, exact int32 sums in tensor memory).
//
//   D[n, f] = qs[n] * ws[f] * sum_k Q[n, k] * W[f, k]  (+ bias[f])
//
// The whole sum over k is one integer, so the scales meet it once, in the
// epilogue, which works in fp32 and rounds once to bf16:
//   SwiGLU          bf16(g / (1 + exp(-g)) * u)
//   clamped SwiGLU  g = min(g, limit), u = clamp(u), bf16(g / (1 + exp(-alpha g)) * (u + 1))
//   down            bf16(D * routing weight of the row)
//
// Weights are the MMA's M = 128 operand, token rows its N: decode tiles of a
// few rows then waste no tensor work, and N follows each tile's row count. A
// weight tile's k-block (128 rows x 128 columns) is stored as the 16 KB image
// that the MMA reads (128-byte swizzle), so one bulk copy moves it. In a gated
// tile, rows 32 q + 0..15 are gate rows and 32 q + 16..31 the up rows of the
// same 16 features: one warp holds both halves of its features and trades
// them by a lane exchange.
//
// 352 threads: warp 0 copies weights, warp 10 token rows (a copy takes its
// issuing thread 100 to 200 cycles, so that one thread for both was the limit
// of large tiles), warp 1 issues the MMAs, warps 2-9 run the epilogue (two per
// 32-lane quarter of tensor memory, alternating 16-column chunks). Two
// accumulator slots let the epilogue of a tile overlap the next tile's products.
//
// Measured: gate/up of 128 experts, 2048 x 768, at 64 tokens of 8 experts 62 us
// (6.3 TB/s: the weights' stream bounds it); at 4096 tokens 118 us (1.7
// POP/s: the tensor pipe waits for tiles half of the time); dense 8191 x 4096 x
// 4096 85 us (3.2 POP/s, tensor pipe 87 % active).
#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace i8 {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = kInt8Threads;
constexpr int kEpi = 256;
constexpr int kRowWarp = 10;
constexpr uint32_t kAStage = 16384;   // 128 weight rows x 128 int8

enum { kEpiClampF32 = 3, kEpiSwigluF32 = 5, kEpiDownOnce = 6 };

// Accumulators of a tile: 2 slots x banks x BN columns fit tensor memory.
__host__ __device__ constexpr int banks(int bn) { return bn <= 64 ? 4 : bn == 128 ? 2 : 1; }

struct Tile {
  int e, ft, row0, nrows;
};

struct Ring {
  int n, idx;
  uint32_t phase;
  __device__ explicit Ring(int n_) : n(n_), idx(0), phase(0u) {}
  __device__ void next() {
    if (++idx == n) {
      idx = 0;
      phase ^= 1u;
    }
  }
};

// Tile t: feature tile (or pair of them) t % ftiles of row chunk t / ftiles. An
// expert's rows are cut into ceil(rows / BN) chunks of equal size rounded up to
// the MMA's N granule, so that no chunk is nearly empty.
template <int GRAN>
__device__ __forceinline__ Tile decode_tile(int t, int ftiles, const int* prefix, const int* starts,
                                            const Int8Params& p) {
  Tile r;
  const int u = t / ftiles;
  r.ft = t - u * ftiles;
  int lo = 0, hi = p.n_experts;   // largest lo with prefix[lo] <= u
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= u) lo = mid; else hi = mid;
  }
  r.e = lo;
  const int sub = u - prefix[lo], parts = prefix[lo + 1] - prefix[lo];
  const int start = starts[lo], cnt = starts[lo + 1] - start;
  const int size = ((cnt + parts - 1) / parts + GRAN - 1) / GRAN * GRAN;
  r.row0 = start + sub * size;
  r.nrows = min(size, cnt - sub * size);   // rounding up may leave the last chunk empty
  return r;
}

__device__ __forceinline__ float row_weight(const Int8Params& p, int row) {
  const int src = p.row_src[row];
  return p.row_w_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.row_w)[src])
                      : reinterpret_cast<const float*>(p.row_w)[src];
}

// g / (1 + exp(-a g)) * u with the hardware exp2 and reciprocal: off by
// |a g| + 8 steps of 2^-23 at most, far inside the bf16 rounding that follows.
// Where the reciprocal would be subnormal (a g below -87.3) the result is 0,
// which is off by less than 2^-119 |u / a|. NaN stays NaN.
__device__ __forceinline__ float glu(float g, float u, float nlog) {   // nlog = -a log2(e)
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * nlog));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * r * u;
}

__device__ __forceinline__ uint16_t bf16_bits(float f) { return __bfloat16_as_ushort(__float2bfloat16_rn(f)); }

// starts[e]: the permuted row where local expert e's rows begin (without
// offsets one expert holds all rows); prefix: exclusive prefix of the experts'
// row chunks. By warp 0, 128 experts at a time, so that their offsets arrive
// together. Offsets are kept within the launch's rows and a segment that ends
// before it begins is empty, so that no offset leads outside the row buffers.
// Returns the number of chunks.
template <int BN>
__device__ __forceinline__ int count_chunks(const Int8Params& p, int* prefix, int* starts) {
  const int lane = threadIdx.x & 31;
  int acc = 0;
  auto in_rows = [&](int v) { return min(max(v, 0), p.dense_rows); };
  if (lane == 0) prefix[0] = 0;
  for (int base = 0; base < p.n_experts; base += 128) {
    int at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = min(base + 32 * i + lane, p.n_experts);
      at[i] = p.offsets ? in_rows(p.offsets[p.expert_begin + e]) : (e ? p.dense_rows : 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = base + 32 * i + lane;
      if (e <= p.n_experts) starts[e] = at[i];
    }
    const int last = min(base + 128, p.n_experts);   // the next lane's start: from the next vector, or memory
    const int end = p.offsets ? in_rows(p.offsets[p.expert_begin + last]) : p.dense_rows;
    if (lane == 0) starts[last] = end;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = base + 32 * i + lane;
      int incl = e < p.n_experts ? (max(0, starts[e + 1] - at[i]) + BN - 1) / BN : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += v;
      }
      if (e < p.n_experts) prefix[e + 1] = acc + incl;
      acc += __shfl_sync(kFull, incl, 31);
    }
  }
  return acc;
}

// Tiles of a launch: none after a wait gave up. Ascending offsets give fewer
// than kInt8MaxTiles (the host has checked); others that give more are flagged.
__device__ __forceinline__ int tile_count(const Int8Params& p, int chunks, int feat_tiles, int gave_up) {
  const long long n = (long long)chunks * feat_tiles;
  if (n > kInt8MaxTiles) atomicOr(p.status, kStatusBadTile);
  return gave_up || n > kInt8MaxTiles ? 0 : static_cast<int>(n);
}

// Columns first * 16 .. + 15, + 32 .. + 47, ... of one accumulator (this
// warp's lanes at `acc`, NB banks of BN columns): added, scaled, gated or
// weighted, and stored as feature f of the rows at `out`.
template <int BN, int NB>
__device__ __forceinline__ void epilogue(const Int8Params& p, uint32_t acc, int first, int nrows, int f,
                                         const float* sa, const float* rw, float ws, float bias, float nlog,
                                         uint16_t* out) {
  const bool is_gate = (threadIdx.x & 31) < 16;
  for (int c0 = first * 16; c0 < nrows; c0 += 32) {
    uint32_t part[NB][16], v[16];
#pragma unroll
    for (int b = 0; b < NB; ++b) tmem_ld16(acc + static_cast<uint32_t>(b * BN + c0), part[b]);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      v[j] = part[0][j];
#pragma unroll
      for (int b = 1; b < NB; ++b) v[j] += part[b][j];
    }
    float d[16];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      d[j] = fmaf(static_cast<float>(static_cast<int>(v[j])), sa[c0 + j] * ws, bias);
    const bool whole = c0 + 16 <= nrows;
    if (p.gated) {
      // gate lanes take the even columns, up lanes the odd ones
      float g[8], u[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float got = __shfl_xor_sync(kFull, is_gate ? d[2 * j + 1] : d[2 * j], 16);
        g[j] = is_gate ? d[2 * j] : got;
        u[j] = is_gate ? got : d[2 * j + 1];
      }
      if (p.epi == kEpiClampF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          g[j] = g[j] > p.limit ? p.limit : g[j];
          u[j] = (u[j] < -p.limit ? -p.limit : (u[j] > p.limit ? p.limit : u[j])) + 1.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = glu(g[j], u[j], nlog);
      const int n0 = c0 + (is_gate ? 0 : 1);
      uint16_t* o = out + n0 * p.ldo;
      if (f < p.n_feat) {
        if (whole) {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[2 * j * p.ldo] = bf16_bits(g[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (n0 + 2 * j < nrows) o[2 * j * p.ldo] = bf16_bits(g[j]);
        }
      }
    } else if (f < p.n_feat) {
      uint16_t* o = out + c0 * p.ldo;
      if (whole) {
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j * p.ldo] = bf16_bits(d[j] * rw[c0 + j]);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (c0 + j < nrows) o[j * p.ldo] = bf16_bits(d[j] * rw[c0 + j]);
      }
    }
  }
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ Int8Params p) {
  constexpr int NB = banks(BN);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base_u32 = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sbase = smem_raw + (base_u32 - raw_u32);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint64_t* full = reinterpret_cast<uint64_t*>(sbase + p.bar_off);
  uint64_t* empty = full + p.ns;
  uint64_t* acc_full = empty + p.ns;    // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]
  uint64_t* mma_done = acc_empty + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(mma_done + 1);
  int* s_total = reinterpret_cast<int*>(s_tmem + 1);
  int* prefix = s_total + 1;            // [n_experts + 1]: row chunks of the experts before
  int* starts = prefix + p.n_experts + 1;   // [n_experts + 1]

  if (warp == 0) {
    // what the row chunks are counted from may come from the previous kernel
    if (!p.early) grid_dep_wait();
    const int gave_up = *reinterpret_cast<volatile int*>(p.status) & kStatusWaitTimeout;
    const int chunks = count_chunks<BN>(p, prefix, starts);
    if (lane == 0) {
      *s_total = tile_count(p, chunks, p.feat_tiles, gave_up);
      for (int i = 0; i < p.ns; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&acc_full[i], 1);
        mbar_init(&acc_empty[i], kEpi / 32);
      }
      mbar_init(mma_done, 1);
      fence_mbar_init();
      tma_prefetch_desc(&qmap);
    }
  }
  if (warp == 1) {
    tmem_alloc(s_tmem, p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int total = *s_total;

  if (warp == 0) {
    // ------------------------------------------------ weight copies
    if (lane == 0) {
      Ring ring(p.ns);
      int issued = 0;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const Tile tl = decode_tile<16>(t, p.feat_tiles, prefix, starts, p);
        if (tl.nrows <= 0) continue;
        const uint8_t* wt = p.wtiles + (long long)(tl.e * p.feat_tiles + tl.ft) * p.nkb * kAStage;
        const uint32_t bytes = kAStage + (tl.nrows + p.box - 1) / p.box * p.box * 128;   // with the token rows
        for (int k = 0; k < p.nkb; ++k, ring.next(), ++issued) {
          const int s = ring.idx;
          if (!wait_bounded(&empty[s], ring.phase ^ 1u, p.status)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[s], bytes);
          bulk_load(sbase + s * p.stage_bytes, wt + (long long)k * kAStage, kAStage, &full[s]);
        }
      }
      // every issued copy has landed before the CTA may exit
      for (int i = max(0, issued - p.ns); i < issued; ++i)
        wait_bounded(&full[i % p.ns], (i / p.ns) & 1, p.status, 32);
    }
  } else if (warp == kRowWarp) {
    // ------------------------------------------------ token row copies
    // (a row's bytes may land before the weight thread has announced them:
    // the phase does not end before that thread's arrival)
    if (lane == 0) {
      grid_dep_wait();   // also without a tile: this grid must not end before the previous one
      Ring ring(p.ns);
      bool ok = true;
      for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
        const Tile tl = decode_tile<16>(t, p.feat_tiles, prefix, starts, p);
        if (tl.nrows <= 0) continue;
        const int boxes = (tl.nrows + p.box - 1) / p.box;
        for (int k = 0; k < p.nkb; ++k, ring.next()) {
          const int s = ring.idx;
          if (!wait_bounded(&empty[s], ring.phase ^ 1u, p.status)) {
            ok = false;
            break;
          }
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(sbase + s * p.stage_bytes + kAStage + b * p.box * 128, &qmap, &full[s], k * 128,
                        tl.row0 + b * p.box);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMAs
    // The whole warp runs the loop and one lane issues: the descriptors are
    // then uniform values, where a loop of one lane moved each of them over
    // (116 cycles an MMA).
    Ring ring(p.ns);
    int tc = 0;
    bool ok = true;
    const uint32_t acc = __shfl_sync(kFull, tmem, 0);
    for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
      const Tile tl = decode_tile<16>(t, p.feat_tiles, prefix, starts, p);
      const int nrows = __shfl_sync(kFull, tl.nrows, 0);
      if (nrows <= 0) continue;
      const int slot = tc & 1;
      if (!__all_sync(kFull, wait_bounded(&acc_empty[slot], ((tc >> 1) & 1) ^ 1, p.status))) break;
      const uint32_t idesc = idesc_s8_s32(128, (nrows + 15) & ~15);
      const uint32_t d = acc + static_cast<uint32_t>(slot * NB * BN);
      for (int k = 0; k < p.nkb; ++k, ring.next()) {
        const int s = ring.idx;
        if (!__all_sync(kFull, wait_bounded(&full[s], ring.phase, p.status))) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = base_u32 + s * p.stage_bytes;
        const uint64_t ad = sdesc_k_sw128(st), bd = sdesc_k_sw128(st + kAStage);
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            umma_s8(d + (j % NB) * BN, ad + 2 * j, bd + 2 * j, idesc, k != 0 || j >= NB ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        __syncwarp();
      }
      if (elect_one()) umma_commit(&acc_full[slot]);
      __syncwarp();
      ++tc;
    }
    // all issued MMAs have finished before tensor memory is released
    if (elect_one()) umma_commit(mma_done);
    __syncwarp();
    wait_bounded(mma_done, 0, p.status);
  } else {
    // ------------------------------------------------ epilogue
    // Warp w reads lanes 32 (w % 4) .. + 31 of tensor memory: lane i holds
    // weight row r = 32 (w % 4) + i of the tile.
    const int q = warp & 3, r = q * 32 + lane;
    const int first = (warp - 2) >> 2;   // this warp's first 16-column chunk
    const int te = threadIdx.x - 64;
    const uint32_t tq = tmem + (static_cast<uint32_t>(q * 32) << 16);
    float* xs = reinterpret_cast<float*>(sbase + p.x_off);   // [2 tiles][row scales BN | row weights BN]
    const float nlog = -1.44269504f * (p.epi == kEpiClampF32 ? p.alpha : 1.f);
    int tc = 0;
    grid_dep_wait();   // row scales and routing weights are read, and rows written, below
    for (int t = blockIdx.x; t < total; t += gridDim.x) {
      const Tile tl = decode_tile<16>(t, p.feat_tiles, prefix, starts, p);
      if (tl.nrows <= 0) continue;
      const int slot = tc & 1;
      float* sa = xs + (tc & 1) * (2 * BN);
      float* rw = sa + BN;
      for (int n = te; n < BN; n += kEpi) {
        const bool in = n < tl.nrows;
        sa[n] = in ? p.qs[tl.row0 + n] : 0.f;
        rw[n] = in && p.row_w ? row_weight(p, tl.row0 + n) : 1.f;
      }
      const long long wrow = (long long)(tl.e * p.feat_tiles + tl.ft) * 128 + r;
      const float ws = p.wscale[wrow];
      const float bias = p.bias ? p.bias[wrow] : 0.f;
      const int f = p.gated ? tl.ft * 64 + q * 16 + (lane & 15) : tl.ft * 128 + r;
      // publishes the tile's scales and lets the eight warps agree on success
      if (!named_bar_and(1, kEpi, wait_bounded(&acc_full[slot], (tc >> 1) & 1, p.status))) break;
      tc_fence_after();
      uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (long long)tl.row0 * p.ldo + f;
      epilogue<BN, NB>(p, tq + static_cast<uint32_t>(slot * NB * BN), first, tl.nrows, f, sa, rw, ws, bias, nlog, out);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[slot]);
      ++tc;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

// As int8_gemm_kernel<256> on CTA pairs: a cluster of two takes two neighbouring
// feature tiles of a row chunk as one 256-row MMA (cta_group::2). Each CTA
// loads its own weight tile and half of the chunk's token rows, which the pair
// shares: a k-block brings 32 KB into an SM instead of 48, and its MMA reads as
// much less, where the shared memory's traffic was the limit. CTA 0's barriers
// `full` and `acc_empty` serve both, the commits arrive in both CTAs. Tried and
// not faster (gate/up at 4096 tokens, 118 us here): chunks of 512 rows with two
// accumulators that share the weights 138 us (no accumulator is left for the
// epilogue to overlap), token rows in boxes of their own count 118 to 121 us,
// several accumulators for few rows 122 us.
__global__ void __launch_bounds__(kThreads, 1)
    int8_pair_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ Int8Params p) {
  constexpr int BN = 256;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_u32 = smem_u32(smem_raw);
  const uint32_t base_u32 = (raw_u32 + 1023u) & ~1023u;
  uint8_t* sbase = smem_raw + (base_u32 - raw_u32);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  uint64_t* full = reinterpret_cast<uint64_t*>(sbase + p.bar_off);
  uint64_t* empty = full + p.ns;
  uint64_t* acc_full = empty + p.ns;    // [2]
  uint64_t* acc_empty = acc_full + 2;   // [2]
  uint64_t* mma_done = acc_empty + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(mma_done + 1);
  int* s_total = reinterpret_cast<int*>(s_tmem + 1);
  int* prefix = s_total + 1;
  int* starts = prefix + p.n_experts + 1;
  const int pairs = (p.feat_tiles + 1) / 2;

  if (warp == 0) {
    if (!p.early) grid_dep_wait();
    const int gave_up = *reinterpret_cast<volatile int*>(p.status) & kStatusWaitTimeout;
    const int chunks = count_chunks<BN>(p, prefix, starts);
    if (lane == 0) {
      *s_total = tile_count(p, chunks, pairs, gave_up);
      for (int i = 0; i < p.ns; ++i) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&acc_full[i], 1);
        mbar_init(&acc_empty[i], 2 * kEpi / 32);
      }
      mbar_init(mma_done, 1);
      fence_mbar_init();
      tma_prefetch_desc(&qmap);
      tma_prefetch_desc(&wmap);
    }
  }
  if (warp == 1) {
    tmem_alloc_pair(s_tmem, p.tmem_cols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  // the peer's barriers are initialised, and both CTAs saw the same status word
  // or not: the pair works on the smaller of the two totals
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  const int total = min(*s_total, static_cast<int>(ld_cluster_u32(mapa_shared(smem_u32(s_total), rank ^ 1u))));
  const int first_tile = blockIdx.x >> 1, step = gridDim.x >> 1;

  if (warp == 0) {
    // ------------------------------------------------ weight copies
    if (lane == 0) {
      Ring ring(p.ns);
      int issued = 0;
      bool ok = true;
      for (int t = first_tile; ok && t < total; t += step) {
        const Tile tl = decode_tile<32>(t, pairs, prefix, starts, p);
        if (tl.nrows <= 0) continue;
        const int ft = min(2 * tl.ft + static_cast<int>(rank), p.feat_tiles - 1);   // an odd last tile twice
        const int wrow = (tl.e * p.feat_tiles + ft) * p.nkb * 128;
        const int half = ((tl.nrows + 31) & ~31) >> 1;
        const uint32_t bytes = 2u * (kAStage + (half + p.box - 1) / p.box * p.box * 128);   // of both CTAs
        for (int k = 0; k < p.nkb; ++k, ring.next(), ++issued) {
          const int s = ring.idx;
          if (!wait_bounded(&empty[s], ring.phase ^ 1u, p.status)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full[s], bytes);
          tma_load_2d_pair(sbase + s * p.stage_bytes, &wmap, mapa_shared(smem_u32(&full[s]), 0), 0, wrow + k * 128);
        }
      }
      // every issued copy, the peer's as well, has landed before the CTAs may exit
      if (rank == 0)
        for (int i = max(0, issued - p.ns); i < issued; ++i)
          wait_bounded(&full[i % p.ns], (i / p.ns) & 1, p.status, 32);
    }
  } else if (warp == kRowWarp) {
    // ------------------------------------------------ token row copies
    if (lane == 0) {
      grid_dep_wait();
      Ring ring(p.ns);
      bool ok = true;
      for (int t = first_tile; ok && t < total; t += step) {
        const Tile tl = decode_tile<32>(t, pairs, prefix, starts, p);
        if (tl.nrows <= 0) continue;
        const int half = ((tl.nrows + 31) & ~31) >> 1;
        const int boxes = (half + p.box - 1) / p.box;
        const int row0 = tl.row0 + static_cast<int>(rank) * half;
        for (int k = 0; k < p.nkb; ++k, ring.next()) {
          const int s = ring.idx;
          if (!wait_bounded(&empty[s], ring.phase ^ 1u, p.status)) {
            ok = false;
            break;
          }
          for (int b = 0; b < boxes; ++b)
            tma_load_2d_pair(sbase + s * p.stage_bytes + kAStage + b * p.box * 128, &qmap,
                             mapa_shared(smem_u32(&full[s]), 0), k * 128, row0 + b * p.box);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMAs of the pair
    if (rank == 0) {
      Ring ring(p.ns);
      int tc = 0;
      bool ok = true;
      const uint32_t acc = __shfl_sync(kFull, tmem, 0);
      for (int t = first_tile; ok && t < total; t += step) {
        const Tile tl = decode_tile<32>(t, pairs, prefix, starts, p);
        const int nrows = __shfl_sync(kFull, tl.nrows, 0);
        if (nrows <= 0) continue;
        const int slot = tc & 1;
        if (!__all_sync(kFull, wait_bounded_cluster(&acc_empty[slot], ((tc >> 1) & 1) ^ 1, p.status))) break;
        const uint32_t idesc = idesc_s8_s32(256, (nrows + 31) & ~31);
        const uint32_t d = acc + static_cast<uint32_t>(slot * BN);
        for (int k = 0; k < p.nkb; ++k, ring.next()) {
          const int s = ring.idx;
          if (!__all_sync(kFull, wait_bounded(&full[s], ring.phase, p.status))) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t st = base_u32 + s * p.stage_bytes;
          const uint64_t ad = sdesc_k_sw128(st), bd = sdesc_k_sw128(st + kAStage);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j) umma_s8_pair(d, ad + 2 * j, bd + 2 * j, idesc, (k | j) != 0 ? 1u : 0u);
            umma_commit_pair(&empty[s]);
          }
          __syncwarp();
        }
        if (elect_one()) umma_commit_pair(&acc_full[slot]);
        __syncwarp();
        ++tc;
      }
      // all issued MMAs have finished before tensor memory is released
      if (elect_one()) umma_commit_pair(mma_done);
      __syncwarp();
    }
    wait_bounded(mma_done, 0, p.status);
  } else {
    // ------------------------------------------------ epilogue of this CTA's feature tile
    const int q = warp & 3, r = q * 32 + lane;
    const int first = (warp - 2) >> 2;
    const int te = threadIdx.x - 64;
    const uint32_t tq = tmem + (static_cast<uint32_t>(q * 32) << 16);
    float* xs = reinterpret_cast<float*>(sbase + p.x_off);
    const float nlog = -1.44269504f * (p.epi == kEpiClampF32 ? p.alpha : 1.f);
    int tc = 0;
    grid_dep_wait();
    for (int t = first_tile; t < total; t += step) {
      const Tile tl = decode_tile<32>(t, pairs, prefix, starts, p);
      if (tl.nrows <= 0) continue;
      const int slot = tc & 1;
      float* sa = xs + (tc & 1) * (2 * BN);
      float* rw = sa + BN;
      for (int n = te; n < BN; n += kEpi) {
        const bool in = n < tl.nrows;
        sa[n] = in ? p.qs[tl.row0 + n] : 0.f;
        rw[n] = in && p.row_w ? row_weight(p, tl.row0 + n) : 1.f;
      }
      const int ft = 2 * tl.ft + static_cast<int>(rank);
      const long long wrow = (long long)(tl.e * p.feat_tiles + min(ft, p.feat_tiles - 1)) * 128 + r;
      const float ws = p.wscale[wrow];
      const float bias = p.bias ? p.bias[wrow] : 0.f;
      const int f = p.gated ? ft * 64 + q * 16 + (lane & 15) : ft * 128 + r;   // past n_feat in a doubled tile
      if (!named_bar_and(1, kEpi, wait_bounded(&acc_full[slot], (tc >> 1) & 1, p.status))) break;
      tc_fence_after();
      uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (long long)tl.row0 * p.ldo + f;
      epilogue<BN, 1>(p, tq + static_cast<uint32_t>(slot * BN), first, tl.nrows, f, sa, rw, ws, bias, nlog, out);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&acc_empty[slot]), 0));
      ++tc;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // no MMA, copy or arrival of either CTA is still to come
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, p.tmem_cols);
  }
}

}  // namespace i8

uint32_t int8_tmem_columns(int bn) { return 2u * i8::banks(bn) * static_cast<uint32_t>(bn); }

// Row scales and routing weights of two tiles.
uint32_t int8_epilogue_bytes(int bn) { return 16u * static_cast<uint32_t>(bn); }

const void* int8_pair_kernel_ptr() { return reinterpret_cast<const void*>(&i8::int8_pair_kernel); }

const void* int8_kernel_ptr(int bn) {
  switch (bn) {
    case 16: return reinterpret_cast<const void*>(&i8::int8_gemm_kernel<16>);
    case 32: return reinterpret_cast<const void*>(&i8::int8_gemm_kernel<32>);
    case 64: return reinterpret_cast<const void*>(&i8::int8_gemm_kernel<64>);
    case 128: return reinterpret_cast<const void*>(&i8::int8_gemm_kernel<128>);
    case 256: return reinterpret_cast<const void*>(&i8::int8_gemm_kernel<256>);
    default: return nullptr;
  }
}

}  // namespace b200
