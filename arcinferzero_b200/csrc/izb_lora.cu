// Low-rank adapters of many requests beside a shared projection: the rows of a call come in segments, each with an adapter of its own
// or none,
//   u[t][j] = sum_k A[j][k] x[t][k],  x[t][k] = asc[k / 32][t] aq[t][k],      C[t][c_off + n] = base[t][n] + scale * sum_j B[n][j] u[t][j].
//
// Bound by bytes: the adapters' for decode rows, base in and outputs out for prompts (rank 64 over 17408 outputs: 64 operations per byte).  One kernel does
// both products, so that u never goes to memory and a call is one launch: a cluster of CTAs per tile of rows of one segment, each with a share of K for the
// first product; the partial sums meet in distributed shared memory, and each CTA goes on with its share of N.  The work is on mma.sync with 16-bit operands:
// the int8 values are exact in them, so the first product is exact up to its f32 sums; u enters the second one in pieces that add up to 22 bits or more of
// it (f16: two, after a power of two per row that brings the row's largest value below 2^14; bf16: three).  (The tcgen05 path would want 128 rows of one adapter
// per tile and its accumulators back through registers for the base; the tensor pipe is a tenth busy as it is.)
//
// Two forms.  lora_few_kernel: tiles of up to 8 rows, ranks (then outputs) on the instruction's 16-wide side and rows on the 8-wide one.
// lora_rows_kernel: tiles of up to 64 rows; in the second product the rows are on the 16-wide side, and the column order within 16 outputs is chosen so that
// a lane has four neighbouring ones: 16-byte loads of the base and stores.
#include <cuda_bf16.h>

#include "izb_common.cuh"

namespace {

constexpr int kThreads = 256, kWarps = 8, kMaxRank = 256, kMaxCluster = 16;

struct LoraArgs {
  const uint16_t *A, *B;
  const int32_t *ranks, *seg, *adapter;
  const float *scales, *asc, *base;
  const int8_t* aq;
  float* C;  // (its first column)
  int n_ad, R, N, K, T, Mp, n_seg, ldb, ldc, cluster;
};

// ---------------------------------------------------------------------------------------------- which rows
struct Tile {
  int row, rows, adapter, rank;  // rows = 0: a tile too many; adapter = -1: none
  float scale;
};
template <int kRows>
__device__ __forceinline__ Tile find_tile(const LoraArgs& p, int tile, Tile* s_tile, int* s_sum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_tile->rows = 0;
  for (int s0 = 0; s0 < p.n_seg; s0 += kThreads) {
    const int s = s0 + tid;
    int lo = 0, hi = 0, a = -1, rank = 0;
    float scale = 0.0f;
    if (s < p.n_seg) {
      lo = min(max(p.seg[s], 0), p.T);
      hi = min(max(p.seg[s + 1], lo), p.T);
      a = p.adapter[s];
      if (a < 0 || a >= p.n_ad) a = -1;
      if (a >= 0) {
        rank = p.ranks ? min(max(p.ranks[a], 0), p.R) : p.R;
        scale = p.scales[a];
      }
    }
    const int n = (hi - lo + kRows - 1) / kRows;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) incl += s_sum[w];
      total += s_sum[w];
    }
    const int i = tile - (incl - n);
    if (i >= 0 && i < n) {
      s_tile->row = lo + i * kRows;
      s_tile->rows = min(kRows, hi - lo - i * kRows);
      s_tile->adapter = a;
      s_tile->rank = rank;
      s_tile->scale = scale;
    }
    __syncthreads();
    if (tile < total) break;
    tile -= total;
  }
  return *s_tile;
}

// ---------------------------------------------------------------------------------------------- operands
template <bool kBf16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 elements of the inner dimension: a lane holds elements 8t .. 8t+7 of its row on either side (two instructions' worth)
template <bool kBf16>
__device__ __forceinline__ void mma32(float (&d)[4], uint4 r0, uint4 r1, uint4 c) {
  mma<kBf16>(d, r0.x, r1.x, r0.y, r1.y, c.x, c.y);
  mma<kBf16>(d, r0.z, r1.z, r0.w, r1.w, c.z, c.w);
}
// Two int8 values (bytes i, i + 1) as 16-bit floats.  f16: the byte with its sign bit flipped is v + 128, and under the exponent of 1024 it is 1152 + v.
// bf16 has seven bits of fraction: the byte without its sign bit under the exponent of 128, less 128 -- or 256 where the sign bit is set.
template <bool kBf16>
__device__ __forceinline__ uint32_t two_of(uint32_t v, int i) {
  if (kBf16) {
    const uint32_t m = __byte_perm(v, 0x43434343u, i ? 0x4342 : 0x4140);
    const uint32_t a = m & 0xFF7FFF7Fu, b = m & 0xFF80FF80u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const uint32_t m = __byte_perm(v ^ 0x80808080u, 0x64646464u, i ? 0x4342 : 0x4140), b = 0x64806480u;
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool kBf16>
__device__ __forceinline__ uint4 eight_of(uint2 v) {
  return make_uint4(two_of<kBf16>(v.x, 0), two_of<kBf16>(v.x, 2), two_of<kBf16>(v.y, 0), two_of<kBf16>(v.y, 2));
}

// u's pieces: [piece][row][R + 8] 16-bit values (the padding puts the rows' 16-byte pieces on different banks)
template <bool kBf16>
constexpr int kPieces = kBf16 ? 3 : 2;
// A warp makes the pieces of a row from its sums; the factor that the second product's result takes.  A row with a sum that is no finite number is NaN.
template <bool kBf16, class Sum>
__device__ __forceinline__ float make_pieces(uint16_t* to, size_t piece_stride, int rank, int padded, Sum sum) {
  const int lane = threadIdx.x & 31;
  if (kBf16) {
    for (int j = lane; j < padded; j += 32) {
      float u = j < rank ? sum(j) : 0.0f;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const __nv_bfloat16 h = __float2bfloat16_rn(u);
        to[i * piece_stride + j] = __bfloat16_as_ushort(h);
        u -= __bfloat162float(h);
      }
    }
    return 1.0f;
  }
  uint32_t most = 0u;
  float u[kMaxRank / 32];
#pragma unroll
  for (int i = 0; i < kMaxRank / 32; ++i) {
    const int j = i * 32 + lane;
    u[i] = j < rank ? sum(j) : 0.0f;
    most = max(most, __float_as_uint(u[i]) & 0x7FFFFFFFu);
  }
  most = __reduce_max_sync(0xFFFFFFFFu, most);
  const int ex = max((int)(most >> 23), 1) - 127;  // |u| < 2^(ex + 1)
  const bool none = most >= 0x7F800000u;
#pragma unroll
  for (int i = 0; i < kMaxRank / 32; ++i) {
    const int j = i * 32 + lane;
    if (j >= padded) break;
    const float v = none ? __uint_as_float(0x7FC00000u) : ldexpf(u[i], 13 - ex);
    const __half h = __float2half_rn(v);
    to[j] = __half_as_ushort(h);
    to[piece_stride + j] = __half_as_ushort(__float2half_rn(v - __half2float(h)));
  }
  return ldexpf(1.0f, ex - 13);
}

// ---------------------------------------------------------------------------------------------- clusters
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t at_rank(const void* here, int rank) {
  uint32_t to;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(here)), "r"(rank));
  return to;
}
__device__ __forceinline__ void remote_store(uint32_t to, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1,%2,%3,%4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
// share `i` of `n` things among `parts`
__device__ __forceinline__ int share(int n, int parts, int i) { return (int)((long long)n * i / parts); }

// rows without an adapter: the base, or zeros
__device__ __forceinline__ void copy_base(const LoraArgs& p, const Tile& tile, int rank_of_cta) {
  if (p.base == p.C) return;  // (in place: equal strides)
  const int n0 = share(p.N, p.cluster, rank_of_cta), n1 = share(p.N, p.cluster, rank_of_cta + 1);
  for (int t = 0; t < tile.rows; ++t)
    for (int n = n0 + (int)threadIdx.x; n < n1; n += kThreads)
      p.C[(size_t)(tile.row + t) * p.ldc + n] = p.base ? p.base[(size_t)(tile.row + t) * p.ldb + n] : 0.0f;
}

// ---------------------------------------------------------------------------------------------- up to 8 rows
constexpr int kFewRows = 8;
constexpr int kFewRanks = 4;  // rank tiles of 16 at a time
static size_t few_smem(int R, int cluster) {
  // partial sums of the warps | those of the CTAs | the pieces (three at most)
  return (size_t)kWarps * kFewRanks * 16 * 8 * 4 + (size_t)cluster * R * 8 * 4 + (size_t)3 * kFewRows * (R + 8) * 2;
}
template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 2) lora_few_kernel(LoraArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  __shared__ float s_factor[kFewRows];
  float* s_part = reinterpret_cast<float*>(smem);                                          // [warp][64 ranks][8 rows]
  float* s_all = s_part + kWarps * kFewRanks * 16 * 8;                                     // [CTA][R][8]
  uint16_t* s_u = reinterpret_cast<uint16_t*>(s_all + (size_t)p.cluster * p.R * 8);        // [piece][8][R + 8]
  const int rank_of_cta = blockIdx.x % p.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cluster_arrive();  // (waited for before anything is written to another CTA)
  pdl_launch_next();
  pdl_wait();
  const Tile tile = find_tile<kFewRows>(p, blockIdx.x / p.cluster, &s_tile, s_sum);
  if (!tile.rows || tile.rank == 0) {  // (the same in every CTA of the cluster)
    if (tile.rows) copy_base(p, tile, rank_of_cta);
    cluster_wait();
    return;
  }
  const uint16_t* A = p.A + (size_t)tile.adapter * p.R * p.K;
  const uint16_t* B = p.B + (size_t)tile.adapter * p.N * p.R;
  const int rank = (tile.rank + 15) & ~15;  // (the rows in between are zeros)

  // ---- u: 32-blocks of K, a share per CTA, dealt out to its warps
  const int kb1 = share(p.K / 32, p.cluster, rank_of_cta + 1), kb0 = share(p.K / 32, p.cluster, rank_of_cta);
  const int8_t* x = p.aq + (size_t)(tile.row + min(g, tile.rows - 1)) * p.K + 8 * t;
  const float* xs = p.asc + tile.row + min(2 * t, tile.rows - 1);
  const int second = 2 * t + 1 < tile.rows ? 1 : 0;
  for (int j0 = 0; j0 < rank; j0 += kFewRanks * 16) {
    float acc[kFewRanks][4] = {};
    const uint16_t* a = A + (size_t)(j0 + g) * p.K + 8 * t;
#pragma unroll 2
    for (int kb = kb0 + warp; kb < kb1; kb += kWarps) {
      uint4 r0[kFewRanks], r1[kFewRanks];
#pragma unroll
      for (int i = 0; i < kFewRanks; ++i)
        if (j0 + i * 16 < rank) {
          r0[i] = ldg_stream_v4(a + (size_t)i * 16 * p.K + kb * 32);
          r1[i] = ldg_stream_v4(a + (size_t)(i * 16 + 8) * p.K + kb * 32);
        }
      const uint4 v = eight_of<kBf16>(*reinterpret_cast<const uint2*>(x + kb * 32));
      const float s0 = xs[(size_t)kb * p.Mp], s1 = xs[(size_t)kb * p.Mp + second];
#pragma unroll
      for (int i = 0; i < kFewRanks; ++i)
        if (j0 + i * 16 < rank) {
          float d[4] = {};
          mma32<kBf16>(d, r0[i], r1[i], v);
          acc[i][0] = fmaf(s0, d[0], acc[i][0]);
          acc[i][1] = fmaf(s1, d[1], acc[i][1]);
          acc[i][2] = fmaf(s0, d[2], acc[i][2]);
          acc[i][3] = fmaf(s1, d[3], acc[i][3]);
        }
    }
#pragma unroll
    for (int i = 0; i < kFewRanks; ++i)
      if (j0 + i * 16 < rank) {
        float* to = s_part + (warp * kFewRanks * 16 + i * 16 + g) * 8 + 2 * t;
        *reinterpret_cast<float2*>(to) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(to + 64) = make_float2(acc[i][2], acc[i][3]);
      }
    __syncthreads();
    if (j0 == 0) cluster_wait();  // every CTA has begun
    // the warps' sums, four values per thread, to every CTA
    const int quads = min(rank - j0, kFewRanks * 16) * 2;
    if (tid < quads) {
      float4 v = *reinterpret_cast<const float4*>(s_part + tid * 4);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 b = *reinterpret_cast<const float4*>(s_part + w * kFewRanks * 16 * 8 + tid * 4);
        v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
      }
      const float* here = s_all + ((size_t)rank_of_cta * p.R + j0) * 8 + tid * 4;
      for (int c = 0; c < p.cluster; ++c) remote_store(at_rank(here, c), v);
    }
    __syncthreads();
  }
  cluster_arrive();
  cluster_wait();
  // ---- the sums of the CTAs in order; a warp per row
  const int padded = (rank + 31) & ~31, ld = p.R + 8;
  const size_t piece = (size_t)kFewRows * ld;
  {
    const float f = make_pieces<kBf16>(s_u + warp * ld, piece, warp < tile.rows ? rank : 0, min(padded, p.R), [&](int j) {
      float u = s_all[j * 8 + warp];
      for (int c = 1; c < p.cluster; ++c) u += s_all[((size_t)c * p.R + j) * 8 + warp];
      return u;
    });
    if (lane == 0) s_factor[warp] = f;
  }
  __syncthreads();

  // ---- outputs: 16 at a time, a share per CTA, dealt out to its warps
  const int tiles = (p.N + 15) / 16, n1 = share(tiles, p.cluster, rank_of_cta + 1);
  const float f0 = s_factor[min(2 * t, kFewRows - 1)], f1 = s_factor[min(2 * t + 1, kFewRows - 1)];
  const bool has0 = 2 * t < tile.rows, has1 = second;
  const uint16_t* u = s_u + g * ld;
#pragma unroll 2
  for (int nt = share(tiles, p.cluster, rank_of_cta) + warp; nt < n1; nt += kWarps) {
    const int n = nt * 16 + g;
    const uint16_t* b0 = B + (size_t)min(n, p.N - 1) * p.R;
    const uint16_t* b1 = B + (size_t)min(n + 8, p.N - 1) * p.R;
    float base[4] = {};
    const size_t row = tile.row + 2 * t;
    if (p.base) {
      if (has0 && n < p.N) base[0] = p.base[row * p.ldb + n];
      if (has1 && n < p.N) base[1] = p.base[(row + 1) * p.ldb + n];
      if (has0 && n + 8 < p.N) base[2] = p.base[row * p.ldb + n + 8];
      if (has1 && n + 8 < p.N) base[3] = p.base[(row + 1) * p.ldb + n + 8];
    }
    float d[4] = {};
    int j = 0;
#pragma unroll 2
    for (; j + 32 <= rank; j += 32) {
      const uint4 r0 = ldg_stream_v4(b0 + j + 8 * t), r1 = ldg_stream_v4(b1 + j + 8 * t);
#pragma unroll
      for (int i = 0; i < kPieces<kBf16>; ++i) mma32<kBf16>(d, r0, r1, *reinterpret_cast<const uint4*>(u + i * piece + j + 8 * t));
    }
    if (j < rank) {  // sixteen more
      const uint2 r0 = *reinterpret_cast<const uint2*>(b0 + j + 4 * t), r1 = *reinterpret_cast<const uint2*>(b1 + j + 4 * t);
#pragma unroll
      for (int i = 0; i < kPieces<kBf16>; ++i) {
        const uint2 v = *reinterpret_cast<const uint2*>(u + i * piece + j + 4 * t);
        mma<kBf16>(d, r0.x, r1.x, r0.y, r1.y, v.x, v.y);
      }
    }
    if (has0 && n < p.N) p.C[row * p.ldc + n] = fmaf(tile.scale, d[0] * f0, base[0]);
    if (has1 && n < p.N) p.C[(row + 1) * p.ldc + n] = fmaf(tile.scale, d[1] * f1, base[1]);
    if (has0 && n + 8 < p.N) p.C[row * p.ldc + n + 8] = fmaf(tile.scale, d[2] * f0, base[2]);
    if (has1 && n + 8 < p.N) p.C[(row + 1) * p.ldc + n + 8] = fmaf(tile.scale, d[3] * f1, base[3]);
  }
}

// ---------------------------------------------------------------------------------------------- up to 64 rows
constexpr int kRows = 64, kRowsCluster = 8, kOwn = kRows / kRowsCluster;  // a CTA joins the sums of kOwn rows
static size_t rows_smem(int R) {
  const int groups = R <= 32 ? 1 : R <= 64 ? 2 : R <= 128 ? 4 : 8;  // warps side by side on ranks
  const size_t part = (size_t)(kWarps / groups) * R * kRows * 4, pieces = (size_t)3 * kRows * (R + 8) * 2;
  return (part > pieces ? part : pieces) + (size_t)kRowsCluster * R * kOwn * 4;
}
template <bool kBf16, bool kVec>
__global__ void __launch_bounds__(kThreads, 2) lora_rows_kernel(LoraArgs p, int groups, size_t first_bytes) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  __shared__ float s_factor[kRows];
  float* s_part = reinterpret_cast<float*>(smem);                // [K part][R][64 rows]; then
  uint16_t* s_u = reinterpret_cast<uint16_t*>(smem);             // [piece][64][R + 8]
  float* s_all = reinterpret_cast<float*>(smem + first_bytes);   // [CTA][R][kOwn]
  const int rank_of_cta = blockIdx.x % kRowsCluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cluster_arrive();
  pdl_launch_next();
  pdl_wait();
  const Tile tile = find_tile<kRows>(p, blockIdx.x / kRowsCluster, &s_tile, s_sum);
  if (!tile.rows || tile.rank == 0) {
    if (tile.rows) copy_base(p, tile, rank_of_cta);
    cluster_wait();
    return;
  }
  const uint16_t* A = p.A + (size_t)tile.adapter * p.R * p.K;
  const uint16_t* B = p.B + (size_t)tile.adapter * p.N * p.R;
  const int rank = (tile.rank + 15) & ~15;

  // ---- u: a warp has 32 ranks x 64 rows, and every parts-th 32-block of the CTA's share of K
  const int parts = kWarps / groups, part = warp / groups, j0 = warp % groups * 32;
  {
    const int kb1 = share(p.K / 32, kRowsCluster, rank_of_cta + 1);
    float acc[2][8][4] = {};
    const uint16_t* a = A + (size_t)(j0 + g) * p.K + 8 * t;
    const bool one = j0 < rank, two = j0 + 16 < rank;
    for (int kb = share(p.K / 32, kRowsCluster, rank_of_cta) + part; one && kb < kb1; kb += parts) {
      uint4 r[2][2] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        r[0][h] = *reinterpret_cast<const uint4*>(a + (size_t)(8 * h) * p.K + kb * 32);
        if (two) r[1][h] = *reinterpret_cast<const uint4*>(a + (size_t)(16 + 8 * h) * p.K + kb * 32);
      }
      uint2 v[8];
      float s[8][2];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = make_uint2(0u, 0u);
        s[i][0] = s[i][1] = 0.0f;
        if (i * 8 + g < tile.rows) v[i] = *reinterpret_cast<const uint2*>(p.aq + (size_t)(tile.row + i * 8 + g) * p.K + kb * 32 + 8 * t);
        const float* xs = p.asc + (size_t)kb * p.Mp + tile.row + i * 8 + 2 * t;
        if (i * 8 + 2 * t < tile.rows) s[i][0] = xs[0];
        if (i * 8 + 2 * t + 1 < tile.rows) s[i][1] = xs[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i * 8 >= tile.rows) break;
        const uint4 c = eight_of<kBf16>(v[i]);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float d[4] = {};
          mma32<kBf16>(d, r[m][0], r[m][1], c);
          acc[m][i][0] = fmaf(s[i][0], d[0], acc[m][i][0]);
          acc[m][i][1] = fmaf(s[i][1], d[1], acc[m][i][1]);
          acc[m][i][2] = fmaf(s[i][0], d[2], acc[m][i][2]);
          acc[m][i][3] = fmaf(s[i][1], d[3], acc[m][i][3]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
      if (j0 + 16 * m < rank)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float* to = s_part + ((size_t)part * p.R + j0 + 16 * m + g) * kRows + 8 * i + 2 * t;
          *reinterpret_cast<float2*>(to) = make_float2(acc[m][i][0], acc[m][i][1]);
          *reinterpret_cast<float2*>(to + 8 * kRows) = make_float2(acc[m][i][2], acc[m][i][3]);
        }
  }
  __syncthreads();
  cluster_wait();  // every CTA has begun
  // the CTA's sums, four rows per thread, to the CTA that joins these rows
  for (int i = tid; i < rank * (kRows / 4); i += kThreads) {
    const int j = i / (kRows / 4), row = i % (kRows / 4) * 4;
    float4 v = *reinterpret_cast<const float4*>(s_part + (size_t)j * kRows + row);
    for (int w = 1; w < parts; ++w) {
      const float4 b = *reinterpret_cast<const float4*>(s_part + ((size_t)w * p.R + j) * kRows + row);
      v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
    }
    remote_store(at_rank(s_all + ((size_t)rank_of_cta * p.R + j) * kOwn + row % kOwn, row / kOwn), v);
  }
  cluster_arrive();
  cluster_wait();
  // ---- a warp per row of its CTA; the pieces go to every CTA (each has left s_part behind: it came to the barrier)
  const int padded = min((rank + 31) & ~31, p.R), ld = p.R + 8;
  const size_t piece = (size_t)kRows * ld;
  {
    static_assert(kOwn == kWarps, "a warp per row");
    const int row = rank_of_cta * kOwn + warp;
    const float f = make_pieces<kBf16>(s_u + row * ld, piece, row < tile.rows ? rank : 0, padded, [&](int j) {
      float u = s_all[(size_t)j * kOwn + warp];
#pragma unroll
      for (int c = 1; c < kRowsCluster; ++c) u += s_all[((size_t)c * p.R + j) * kOwn + warp];
      return u;
    });
    __syncwarp();
    for (int i = lane; i < kPieces<kBf16> * (padded / 8); i += 32) {
      const uint16_t* here = s_u + (i / (padded / 8)) * piece + row * ld + i % (padded / 8) * 8;
      const float4 v = *reinterpret_cast<const float4*>(here);
      for (int c = 0; c < kRowsCluster; ++c)
        if (c != rank_of_cta) remote_store(at_rank(here, c), v);
    }
    if (lane < kRowsCluster) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at_rank(&s_factor[row], lane)), "f"(f) : "memory");
  }
  cluster_arrive();
  cluster_wait();

  // ---- outputs: a warp has 16 rows, and 16 outputs at a time of its half of the CTA's share
  const int m0 = (warp & 3) * 16;
  if (m0 >= tile.rows) return;
  const int tiles = (p.N + 15) / 16, n1 = share(tiles, kRowsCluster, rank_of_cta + 1);
  const uint16_t *u0 = s_u + (m0 + g) * ld, *u1 = u0 + 8 * ld;
  const float f0 = s_factor[m0 + g], f1 = s_factor[m0 + g + 8];
  const bool has0 = m0 + g < tile.rows, has1 = m0 + g + 8 < tile.rows;
  const size_t row = tile.row + m0 + g;
  const float *base0 = p.base ? p.base + row * p.ldb : nullptr, *base1 = p.base ? base0 + 8 * (size_t)p.ldb : nullptr;
  float *c0 = p.C + row * p.ldc, *c1 = c0 + 8 * (size_t)p.ldc;
  const int col = 4 * (g >> 1) + (g & 1);  // column g of the first instruction; of the second one: two further
  constexpr int kAhead = 4;
  auto load_base = [&](const float* from, bool has, int n) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!from || !has) return v;
    if (kVec && n + 4 <= p.N) return *reinterpret_cast<const float4*>(from + n);
    if (n < p.N) v.x = from[n];
    if (n + 1 < p.N) v.y = from[n + 1];
    if (n + 2 < p.N) v.z = from[n + 2];
    if (n + 3 < p.N) v.w = from[n + 3];
    return v;
  };
  auto store = [&](float* to, bool has, int n, float4 v) {
    if (!has) return;
    if (kVec && n + 4 <= p.N) {
      *reinterpret_cast<float4*>(to + n) = v;
      return;
    }
    if (n < p.N) to[n] = v.x;
    if (n + 1 < p.N) to[n + 1] = v.y;
    if (n + 2 < p.N) to[n + 2] = v.z;
    if (n + 3 < p.N) to[n + 3] = v.w;
  };
  for (int nb = share(tiles, kRowsCluster, rank_of_cta) + (warp >> 2); nb < n1; nb += 2 * kAhead) {
    float4 old0[kAhead], old1[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int nt = nb + 2 * i, n = nt * 16 + 4 * t;
      old0[i] = load_base(base0, has0 && nt < n1, n);
      old1[i] = load_base(base1, has1 && nt < n1, n);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int nt = nb + 2 * i, n = nt * 16 + 4 * t;
      if (nt >= n1) break;
      const uint16_t* b0 = B + (size_t)min(nt * 16 + col, p.N - 1) * p.R;
      const uint16_t* b1 = B + (size_t)min(nt * 16 + col + 2, p.N - 1) * p.R;
      float d[2][4] = {};
      int j = 0;
#pragma unroll 2
      for (; j + 32 <= rank; j += 32) {
        const uint4 v0 = *reinterpret_cast<const uint4*>(b0 + j + 8 * t), v1 = *reinterpret_cast<const uint4*>(b1 + j + 8 * t);
#pragma unroll
        for (int k = 0; k < kPieces<kBf16>; ++k) {
          const uint4 r0 = *reinterpret_cast<const uint4*>(u0 + k * piece + j + 8 * t), r1 = *reinterpret_cast<const uint4*>(u1 + k * piece + j + 8 * t);
          mma32<kBf16>(d[0], r0, r1, v0);
          mma32<kBf16>(d[1], r0, r1, v1);
        }
      }
      if (j < rank) {
        const uint2 v0 = *reinterpret_cast<const uint2*>(b0 + j + 4 * t), v1 = *reinterpret_cast<const uint2*>(b1 + j + 4 * t);
#pragma unroll
        for (int k = 0; k < kPieces<kBf16>; ++k) {
          const uint2 r0 = *reinterpret_cast<const uint2*>(u0 + k * piece + j + 4 * t), r1 = *reinterpret_cast<const uint2*>(u1 + k * piece + j + 4 * t);
          mma<kBf16>(d[0], r0.x, r1.x, r0.y, r1.y, v0.x, v0.y);
          mma<kBf16>(d[1], r0.x, r1.x, r0.y, r1.y, v1.x, v1.y);
        }
      }
      store(c0, has0, n, make_float4(fmaf(tile.scale, d[0][0] * f0, old0[i].x), fmaf(tile.scale, d[0][1] * f0, old0[i].y), fmaf(tile.scale, d[1][0] * f0, old0[i].z),
                                     fmaf(tile.scale, d[1][1] * f0, old0[i].w)));
      store(c1, has1, n, make_float4(fmaf(tile.scale, d[0][2] * f1, old1[i].x), fmaf(tile.scale, d[0][3] * f1, old1[i].y), fmaf(tile.scale, d[1][2] * f1, old1[i].z),
                                     fmaf(tile.scale, d[1][3] * f1, old1[i].w)));
    }
  }
}

}  // namespace

extern "C" int izb_lora_add(int dtype, const void* d_A, const void* d_B, int n_adapters, int R, const int32_t* d_ranks, const float* d_scales, int N, int K,
                            const int8_t* d_aq, const float* d_asc, int T, int Mp, const int32_t* d_seg, const int32_t* d_adapter, int n_seg,
                            const float* d_base, int ldb, float* d_C, int ldc, int c_off, void* stream) {
  if (!d_A || !d_B || !d_scales || !d_aq || !d_asc || !d_seg || !d_adapter || !d_C) IZB_FAIL(IZB_ERR_ARG, "lora_add: null pointer");
  if (dtype != IZB_F16 && dtype != IZB_BF16) IZB_FAIL(IZB_ERR_TYPE, "lora_add: adapters of type %d are not taken (IZB_F16, IZB_BF16)", dtype);
  if (n_adapters < 1 || R < 16 || R > kMaxRank || R % 16) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: %d adapters of rank %d (16..%d, a multiple of 16: pad with zeros)", n_adapters, R, kMaxRank);
  if (N < 1 || K < 256 || K % 256) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: N=%d K=%d (K a multiple of 256)", N, K);
  if (T < 1 || Mp % 16 || Mp < T || n_seg < 1) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: T=%d Mp=%d n_seg=%d (Mp a multiple of 16, >= T)", T, Mp, n_seg);
  if (c_off < 0 || (T > 1 && (int64_t)ldc < (int64_t)c_off + N) || (d_base && T > 1 && ldb < N)) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: N=%d c_off=%d ldc=%d ldb=%d", N, c_off, ldc, ldb);
  if (!izb_aligned(d_A, 16) || !izb_aligned(d_B, 16) || !izb_aligned(d_aq, 16) || !izb_aligned(d_asc, 16))
    IZB_FAIL(IZB_ERR_ALIGN, "lora_add: A, B, aq and asc must be 16-byte aligned");
  if (!izb_aligned(d_C, 4) || !izb_aligned(d_base, 4)) IZB_FAIL(IZB_ERR_ALIGN, "lora_add: C and base must be 4-byte aligned");
  if (izb_overlap_in_part(d_base, ldb, d_C + c_off, ldc, T, N)) IZB_FAIL(IZB_ERR_ARG, "lora_add: base overlaps the outputs in part");
  int device = 0;
  IZB_CUDA(cudaGetDevice(&device));
  LoraArgs p = {(const uint16_t*)d_A, (const uint16_t*)d_B, d_ranks, d_seg, d_adapter, d_scales, d_asc, d_base, d_aq, d_C + c_off, n_adapters, R, N, K, T, Mp, n_seg, ldb, ldc, 0};
  cudaStream_t st = (cudaStream_t)stream;
  const bool bf16 = dtype == IZB_BF16, few = T <= 8 * (int64_t)n_seg;
  const int64_t tiles = (int64_t)T / (few ? kFewRows : kRows) + n_seg;  // (at most)
  p.cluster = !few ? kRowsCluster : tiles * 16 <= 2 * izb_sm_count(device) && R <= 128 ? 16 : 8;
  if (tiles * p.cluster > 0x7FFFFFFF) IZB_FAIL(IZB_ERR_LIMIT, "lora_add: %d rows in %d segments", T, n_seg);
  const dim3 grid((unsigned)(tiles * p.cluster));
  if (few) {
    const size_t smem = few_smem(R, p.cluster);
    for (auto kernel : {lora_few_kernel<false>, lora_few_kernel<true>}) {
      static izb_device_once once[2];
      if (int rc = once[kernel == lora_few_kernel<true>].run(device, [&]() -> int {
            IZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)few_smem(kMaxRank, kMaxCluster)));
            IZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            return IZB_OK;
          }))
        return rc;
    }
    IZB_LAUNCH("lora_add", st, izb_launch_pdl_cluster(bf16 ? lora_few_kernel<true> : lora_few_kernel<false>, p.cluster, grid, kThreads, smem, st, p));
    return IZB_OK;
  }
  const bool vec = izb_aligned(p.C, 16) && ldc % 4 == 0 && (!d_base || (izb_aligned(d_base, 16) && ldb % 4 == 0));
  auto kernel = bf16 ? (vec ? lora_rows_kernel<true, true> : lora_rows_kernel<true, false>) : (vec ? lora_rows_kernel<false, true> : lora_rows_kernel<false, false>);
  IZB_SMEM_OPTIN((lora_rows_kernel<true, true>), rows_smem(kMaxRank), device);
  IZB_SMEM_OPTIN((lora_rows_kernel<true, false>), rows_smem(kMaxRank), device);
  IZB_SMEM_OPTIN((lora_rows_kernel<false, true>), rows_smem(kMaxRank), device);
  IZB_SMEM_OPTIN((lora_rows_kernel<false, false>), rows_smem(kMaxRank), device);
  const int groups = R <= 32 ? 1 : R <= 64 ? 2 : R <= 128 ? 4 : 8;
  const size_t smem = rows_smem(R), first = smem - (size_t)kRowsCluster * R * kOwn * 4;
  IZB_LAUNCH("lora_add", st, izb_launch_pdl_cluster(kernel, kRowsCluster, grid, kThreads, smem, st, p, groups, first));
  return IZB_OK;
}
