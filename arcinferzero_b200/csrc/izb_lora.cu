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

template <bool kBf16>
constexpr int kPieces = kBf16 ? 3 : 2;
// A warp makes the pieces of a row from its sums; the factor that the second product's result takes.  A row with a sum that is no finite number is NaN.
// `swap`: what the places' numbers are xored with.
template <bool kBf16, class Sum>
__device__ __forceinline__ float make_pieces(uint16_t* to, size_t piece_stride, int rank, int padded, Sum sum, int swap = 0) {
  const int lane = threadIdx.x & 31;
  if (kBf16) {
    for (int j = lane; j < padded; j += 32) {
      float u = j < rank ? sum(j) : 0.0f;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const __nv_bfloat16 h = __float2bfloat16_rn(u);
        to[i * piece_stride + (j ^ swap)] = __bfloat16_as_ushort(h);
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
  const int ex = max((int)(most >> 23) - 127, -100);  // |u| < 2^(ex + 1)
  const bool none = most >= 0x7F800000u;
#pragma unroll
  for (int i = 0; i < kMaxRank / 32; ++i) {
    const int j = i * 32 + lane;
    if (j >= padded) break;
    const float v = none ? __uint_as_float(0x7FC00000u) : ldexpf(u[i], 13 - ex);
    const __half h = __float2half_rn(v);
    to[j ^ swap] = __half_as_ushort(h);
    to[piece_stride + (j ^ swap)] = __half_as_ushort(__float2half_rn(v - __half2float(h)));
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
constexpr int kFewRanks = 4;   // rank tiles of 16 at a time
constexpr int kFewSlots = 8;   // pieces of an adapter (16 rows x 32 elements, 1 KB) that a warp has asked for: 64 KB per CTA
static size_t few_smem(int R, int cluster) {
  // rings | partial sums of the warps | those of the CTAs | the pieces of u (three at most)
  return (size_t)kWarps * kFewSlots * 1024 + (size_t)kWarps * kFewRanks * 16 * 8 * 4 + (size_t)cluster * R * 8 * 4 + (size_t)3 * kFewRows * (R + 8) * 2;
}
// The adapter streams through a ring per warp: each lane copies what it will read itself (its 16 bytes of rows g and g + 8), so that nobody waits for
// anybody, and the second product's first pieces are on their way while the first one's sums are exchanged.
template <bool kBf16>
__global__ void __launch_bounds__(kThreads, 2) lora_few_kernel(LoraArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  __shared__ float s_factor[kFewRows];
  float* s_part = reinterpret_cast<float*>(smem + kWarps * kFewSlots * 1024);              // [warp][64 ranks][8 rows]
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
  // this warp's 32-blocks of K and its sixteens of outputs
  const int kb1 = share(p.K / 32, p.cluster, rank_of_cta + 1), kb0 = share(p.K / 32, p.cluster, rank_of_cta) + warp;
  const int tiles = (p.N + 15) / 16, nt0 = share(tiles, p.cluster * kWarps, rank_of_cta * kWarps + warp), nt1 = share(tiles, p.cluster * kWarps, rank_of_cta * kWarps + warp + 1);
  const int whole = p.N / 16;  // (a last tile may be cut off)

  // ---- the ring: pieces in the order in which they are used below
  unsigned char* ring = smem + warp * kFewSlots * 1024 + lane * 16;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  int ask_slot = 0, ask_j0 = kb0 < kb1 ? 0 : rank, ask_kb = kb0, ask_i = 0, ask_nt = nt0, ask_j = 0;
  const size_t eight_a = (size_t)8 * p.K, eight_b = (size_t)8 * p.R;
  const uint16_t* ask_a = A + (size_t)g * p.K + kb0 * 32 + 8 * t;  // of rank tile 0 and ask_kb
  const uint16_t* ask_b = B + (size_t)(nt0 * 16 + g) * p.R;        // of ask_nt
  auto ask = [&]() {
    const uint32_t to = ring_at + ask_slot * 1024;
    ask_slot = (ask_slot + 1) % kFewSlots;
    if (ask_j0 < rank) {  // of A
      const uint16_t* from = ask_a + 2 * (ask_j0 / 16 + ask_i) * eight_a;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n\tcp.async.cg.shared.global [%0+512], [%2], 16;" ::"r"(to), "l"(from), "l"(from + eight_a) : "memory");
      if (++ask_i == kFewRanks || ask_j0 + 16 * ask_i >= rank) {
        ask_i = 0;
        ask_kb += kWarps;
        ask_a += kWarps * 32;
        if (ask_kb >= kb1) {
          ask_a -= (ask_kb - kb0) * 32;
          ask_kb = kb0;
          ask_j0 += kFewRanks * 16;
        }
      }
    } else if (ask_nt < nt1) {  // of B
      const uint16_t *from0 = ask_b + ask_j, *from1 = from0 + eight_b;
      if (ask_nt >= whole) {
        from0 = B + (size_t)min(ask_nt * 16 + g, p.N - 1) * p.R + ask_j;
        from1 = B + (size_t)min(ask_nt * 16 + g + 8, p.N - 1) * p.R + ask_j;
      }
      if (ask_j + 32 <= rank)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n\tcp.async.cg.shared.global [%0+512], [%2], 16;" ::"r"(to), "l"(from0 + 8 * t), "l"(from1 + 8 * t) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n\tcp.async.ca.shared.global [%0+512], [%2], 8;" ::"r"(to), "l"(from0 + 4 * t), "l"(from1 + 4 * t) : "memory");
      ask_j += 32;
      if (ask_j >= rank) {
        ask_j = 0;
        ++ask_nt;
        ask_b += 2 * eight_b;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int slot = 0;
  auto take = [&](uint4& r0, uint4& r1) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kFewSlots - 1) : "memory");
    r0 = *reinterpret_cast<const uint4*>(ring + slot * 1024);
    r1 = *reinterpret_cast<const uint4*>(ring + slot * 1024 + 512);
    slot = (slot + 1) % kFewSlots;
    ask();
  };
#pragma unroll
  for (int i = 0; i < kFewSlots; ++i) ask();

  // ---- u
  const int8_t* x = p.aq + (size_t)(tile.row + min(g, tile.rows - 1)) * p.K + 8 * t;
  const float* xs = p.asc + tile.row + min(2 * t, tile.rows - 1);
  const int second = 2 * t + 1 < tile.rows ? 1 : 0;
  for (int j0 = 0; j0 < rank; j0 += kFewRanks * 16) {
    float acc[kFewRanks][4] = {};
    uint2 v_next = make_uint2(0u, 0u);
    float s_next[2] = {};
    auto values = [&](int kb) {
      if (kb >= kb1) return;
      v_next = *reinterpret_cast<const uint2*>(x + kb * 32);
      s_next[0] = xs[(size_t)kb * p.Mp];
      s_next[1] = xs[(size_t)kb * p.Mp + second];
    };
    values(kb0);
    for (int kb = kb0; kb < kb1; kb += kWarps) {
      const uint4 v = eight_of<kBf16>(v_next);
      const float s0 = s_next[0], s1 = s_next[1];
      values(kb + kWarps);
#pragma unroll
      for (int i = 0; i < kFewRanks; ++i)
        if (j0 + i * 16 < rank) {
          uint4 r0, r1;
          take(r0, r1);
          float d[4] = {};
          mma32<kBf16>(d, r0, r1, v);
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
  const int ld = p.R + 8;
  const size_t piece = (size_t)kFewRows * ld;
  {
    const float f = make_pieces<kBf16>(s_u + warp * ld, piece, warp < tile.rows ? rank : 0, rank, [&](int j) {
      const float* from = s_all + j * 8 + warp;
      float u = 0.0f;
#pragma unroll 8
      for (int c = 0; c < p.cluster; ++c) u += from[(size_t)c * p.R * 8];
      return u;
    });
    if (lane == 0) s_factor[warp] = f;
  }
  __syncthreads();

  // ---- outputs
  const float f0 = tile.scale * s_factor[2 * t], f1 = tile.scale * s_factor[2 * t + 1];
  const bool has0 = 2 * t < tile.rows, has1 = second;
  const uint16_t* u = s_u + g * ld;
  const size_t first = (size_t)tile.row + 2 * t;
  const float* from = p.base ? p.base + first * p.ldb + nt0 * 16 + g : nullptr;
  float* to = p.C + first * p.ldc + nt0 * 16 + g;
  float next[4] = {};
  auto load_base = [&](int nt) {
    if (!from || nt >= nt1) return;
    const bool n0 = nt < whole || nt * 16 + g < p.N, n1 = nt < whole || nt * 16 + g + 8 < p.N;
    if (has0 && n0) next[0] = from[0];
    if (has0 && n1) next[2] = from[8];
    if (has1 && n0) next[1] = from[p.ldb];
    if (has1 && n1) next[3] = from[(size_t)p.ldb + 8];
    from += 16;
  };
  load_base(nt0);
  for (int nt = nt0; nt < nt1; ++nt, to += 16) {
    const float base[4] = {next[0], next[1], next[2], next[3]};
    load_base(nt + 1);
    float d[4] = {};
    for (int j = 0; j < rank; j += 32) {
      uint4 r0, r1;
      take(r0, r1);
      if (j + 32 <= rank) {
#pragma unroll
        for (int i = 0; i < kPieces<kBf16>; ++i) mma32<kBf16>(d, r0, r1, *reinterpret_cast<const uint4*>(u + i * piece + j + 8 * t));
      } else {  // sixteen more
#pragma unroll
        for (int i = 0; i < kPieces<kBf16>; ++i) {
          const uint2 v = *reinterpret_cast<const uint2*>(u + i * piece + j + 4 * t);
          mma<kBf16>(d, r0.x, r1.x, r0.y, r1.y, v.x, v.y);
        }
      }
    }
    const bool n0 = nt < whole || nt * 16 + g < p.N, n1 = nt < whole || nt * 16 + g + 8 < p.N;
    if (has0 && n0) to[0] = fmaf(f0, d[0], base[0]);
    if (has0 && n1) to[8] = fmaf(f0, d[2], base[2]);
    if (has1 && n0) to[p.ldc] = fmaf(f1, d[1], base[1]);
    if (has1 && n1) to[(size_t)p.ldc + 8] = fmaf(f1, d[3], base[3]);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------- up to 64 rows
constexpr int kRows = 64, kRowsCluster = 8, kOwn = kRows / kRowsCluster;  // a CTA joins the sums of kOwn rows
constexpr int kCols = 64;                                                  // outputs of a step of the second product
// u's pieces and B's tiles: rows of R rounded up to 32 values, in 16-byte chunks; where a row is a multiple of 128 bytes odd rows have the halves of
// their 128-byte lines changed over, so that two neighbouring rows' 64 bytes lie on different banks.  The same with A's tiles.
struct RowsPlan {
  int groups;                         // warps side by side on ranks in the first product, 32 ranks each; the others share its blocks of K
  int ld, swap;                       // a row's 16-bit values; what odd rows' chunk numbers are xored with
  int stages1, stages2;               // of asynchronous copies, in the first product and in the second
  uint32_t stage1, stage2;            // bytes: activations | their scales | A's tile; B's tile | base
  uint32_t first, all, total;         // where the stages (over them the partial sums) and the CTAs' sums are, behind the pieces
  RowsPlan(int R, bool bf16) {
    groups = R <= 32 ? 1 : R <= 64 ? 2 : R <= 128 ? 4 : 8;
    const int parts = kWarps / groups;
    ld = (R + 31) / 32 * 32;
    swap = ld % 64 ? 0 : 4;
    first = (bf16 ? 3 : 2) * kRows * ld * 2;
    stages1 = R <= 32 ? 2 : 3;
    stages2 = R <= 128 ? 3 : 2;
    stage1 = parts * (kRows * 32 + kRows * 4 + R * 64);
    stage2 = kCols * ld * 2 + kRows * kCols * 4;
    const uint32_t part = (uint32_t)parts * R * kRows * 4, sums = (uint32_t)kRowsCluster * R * kOwn * 4;
    const uint32_t early = (stages2 - 1) * stage2;  // (in use before the sums have been read)
    all = first + (part > early ? part : early);
    total = all + sums;
    if (total < first + stages1 * stage1) total = first + stages1 * stage1;
    if (total < first + stages2 * stage2) total = first + stages2 * stage2;
  }
};
template <int kN>
__device__ __forceinline__ void copies_there() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }
__device__ __forceinline__ void copies_there(int later) {
  if (later == 2) copies_there<2>();
  else if (later == 1) copies_there<1>();
  else copies_there<0>();
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// kRegs: the ranks are 64 at most, and a warp holds its rows' pieces in registers through the second product
template <bool kBf16, bool kVec, bool kRegs>
__global__ void __launch_bounds__(kThreads, 2) lora_rows_kernel(LoraArgs p, RowsPlan plan) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  __shared__ float s_factor[kRows];
  uint16_t* s_u = reinterpret_cast<uint16_t*>(smem);              // [piece][64][ld]
  float* s_part = reinterpret_cast<float*>(smem + plan.first);    // [K part][R][64 rows]
  float* s_all = reinterpret_cast<float*>(smem + plan.all);       // [CTA][R][kOwn]
  const int ld = plan.ld;
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
  const uint32_t stages_at = (uint32_t)__cvta_generic_to_shared(smem) + plan.first;

  // ---- u: a warp has 32 ranks x 64 rows, and every parts-th 32-block of the CTA's share of K; `parts` blocks per stage
  const int parts = kWarps / plan.groups, part = warp / plan.groups, j0 = warp % plan.groups * 32;
  {
    const int kb0 = share(p.K / 32, kRowsCluster, rank_of_cta), kb1 = share(p.K / 32, kRowsCluster, rank_of_cta + 1), steps = (kb1 - kb0 + parts - 1) / parts;
    const int row_log = __ffs(parts) + 1, swap = parts > 1 ? 4 : 0;  // a row of A's tile: 2^row_log chunks
    const uint32_t scales_at = parts * kRows * 32, a_at = scales_at + parts * kRows * 4;
    auto ask = [&](int step, int stage) {
      if (step < steps) {
        const uint32_t to = stages_at + stage * plan.stage1;
        const int kb = kb0 + step * parts, blocks = min(parts, kb1 - kb);
        for (int i = tid; i < blocks * kRows * 2; i += kThreads) {  // (rows past the tile's: the last one again, which nobody reads)
          const int r = min((i >> 1) & (kRows - 1), tile.rows - 1);
          copy16(to + i * 16, p.aq + (size_t)(tile.row + r) * p.K + (kb + (i >> 7)) * 32 + (i & 1) * 16);
        }
        for (int i = tid; i < blocks * kRows; i += kThreads)
          copy4(to + scales_at + i * 4, p.asc + (size_t)(kb + (i >> 6)) * p.Mp + tile.row + min(i & (kRows - 1), tile.rows - 1));
        for (int i = tid; i < rank << row_log; i += kThreads) {
          const int j = i >> row_log, c = i & ((1 << row_log) - 1);
          if (c < blocks * 4) copy16(to + a_at + ((j << row_log) + (c ^ (j & 1 ? swap : 0))) * 16, A + (size_t)j * p.K + kb * 32 + c * 8);
        }
      }
      copies_begun();
    };
    float acc[2][8][4] = {};
    const bool one = j0 < rank, two = j0 + 16 < rank;
    for (int i = 0; i < plan.stages1 - 1; ++i) ask(i, i);
    for (int step = 0, stage = 0; step < steps; ++step) {
      copies_there(plan.stages1 - 2);
      __syncthreads();
      ask(step + plan.stages1 - 1, stage == 0 ? plan.stages1 - 1 : stage - 1);
      const unsigned char* here = smem + plan.first + stage * plan.stage1;
      stage = stage + 1 == plan.stages1 ? 0 : stage + 1;
      if (!one || kb0 + step * parts + part >= kb1) continue;
      const uint4* a = reinterpret_cast<const uint4*>(here + a_at) + ((size_t)(j0 + g) << row_log) + ((part * 4) ^ (g & 1 ? swap : 0)) + t;
      uint4 r[2][2] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        r[0][h] = a[(8 * h) << row_log];
        if (two) r[1][h] = a[(16 + 8 * h) << row_log];
      }
      const uint2* x = reinterpret_cast<const uint2*>(here + part * kRows * 32) + g * 4 + t;
      const float2* xs = reinterpret_cast<const float2*>(here + scales_at + part * kRows * 4) + t;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i * 8 >= tile.rows) break;
        const uint4 c = eight_of<kBf16>(x[i * 32]);
        const float2 sc = xs[i * 4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float d[4] = {};
          mma32<kBf16>(d, r[m][0], r[m][1], c);
          acc[m][i][0] = fmaf(sc.x, d[0], acc[m][i][0]);
          acc[m][i][1] = fmaf(sc.y, d[1], acc[m][i][1]);
          acc[m][i][2] = fmaf(sc.x, d[2], acc[m][i][2]);
          acc[m][i][3] = fmaf(sc.y, d[3], acc[m][i][3]);
        }
      }
    }
    copies_there<0>();
    __syncthreads();  // (the partial sums go over the stages)
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

  // ---- steps of 64 outputs of the CTA's share: B's rows and the base come through stages, the first of them from here on
  const int steps_all = (p.N + kCols - 1) / kCols, step0 = share(steps_all, kRowsCluster, rank_of_cta), steps = share(steps_all, kRowsCluster, rank_of_cta + 1) - step0;
  const int m0 = (warp & 3) * 16, half = (warp >> 2) * 32;  // a warp has 16 rows and 32 of the 64 outputs
  const size_t row = tile.row + m0 + g;
  const bool has0 = m0 + g < tile.rows, has1 = m0 + g + 8 < tile.rows;
  const int b_row = tid >> 2, b_chunk = tid & 3, b_swap = b_row & 1 ? plan.swap : 0;  // four threads copy a row of B
  const uint32_t b_to = stages_at + b_row * ld * 2 + b_chunk * 16, base_to = stages_at + kCols * ld * 2 + tid * 16;
  const uint16_t* b_from = B + (size_t)(step0 * kCols + b_row) * p.R + b_chunk * 8;
  const float* base_from = p.base ? p.base + row * p.ldb + step0 * kCols + half + 4 * t : nullptr;
  const size_t eight = (size_t)8 * p.ldb;
  auto ask = [&](int step, int stage) {
    if (step < steps) {
      const uint32_t at = stage * plan.stage2;
      const int n0 = (step0 + step) * kCols;
      const bool whole = n0 + kCols <= p.N;
      const uint16_t* from = whole ? b_from + (size_t)step * kCols * p.R : B + (size_t)min(n0 + b_row, p.N - 1) * p.R + b_chunk * 8;
      for (int c = 0; c * 8 < rank; c += 4)
        if ((c + b_chunk) * 8 < rank) copy16(b_to + at + (c ^ b_swap) * 16, from + c * 8);
      if (base_from) {  // each lane what it will add: rows g and g + 8, four outputs of both of its warp's sixteens
        const float* of = base_from + (size_t)step * kCols;
        if (kVec && whole) {
          if (has0) {
            copy16(base_to + at, of);
            copy16(base_to + at + 2 * kThreads * 16, of + 16);
          }
          if (has1) {
            copy16(base_to + at + kThreads * 16, of + eight);
            copy16(base_to + at + 3 * kThreads * 16, of + eight + 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = n0 + half + (i >> 1) * 16 + 4 * t;
            if (!(i & 1 ? has1 : has0)) continue;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n + k < p.N) copy4(base_to + at + i * kThreads * 16 + k * 4, of + (i & 1 ? eight : 0) + (i >> 1) * 16 + k);
          }
        }
      }
    }
    copies_begun();
  };
  for (int i = 0; i < plan.stages2 - 1; ++i) ask(i, i);

  // ---- a warp per row of its CTA; the pieces go to every CTA
  const int padded = ld;
  const size_t piece = (size_t)kRows * ld;
  {
    static_assert(kOwn == kWarps, "a warp per row");
    const int own = rank_of_cta * kOwn + warp;
    const float f = make_pieces<kBf16>(s_u + own * ld, piece, own < tile.rows ? rank : 0, padded, [&](int j) {
      float u = s_all[(size_t)j * kOwn + warp];
#pragma unroll
      for (int c = 1; c < kRowsCluster; ++c) u += s_all[((size_t)c * p.R + j) * kOwn + warp];
      return u;
    }, (own & 1 ? plan.swap : 0) * 8);
    __syncwarp();
    for (int i = lane; i < kPieces<kBf16> * (padded / 8); i += 32) {
      const uint16_t* here = s_u + (i / (padded / 8)) * piece + own * ld + i % (padded / 8) * 8;
      const float4 v = *reinterpret_cast<const float4*>(here);
      for (int c = 0; c < kRowsCluster; ++c)
        if (c != rank_of_cta) remote_store(at_rank(here, c), v);
    }
    if (lane < kRowsCluster) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at_rank(&s_factor[own], lane)), "f"(f) : "memory");
  }
  cluster_arrive();
  cluster_wait();

  // ---- outputs
  const float f0 = tile.scale * s_factor[m0 + g], f1 = tile.scale * s_factor[m0 + g + 8];
  float *c0 = p.C + row * p.ldc + step0 * kCols + half + 4 * t, *c1 = c0 + 8 * (size_t)p.ldc;
  const int col = 4 * (g >> 1) + (g & 1);     // column g of the first instruction; of the second one: two further
  const int swap = g & 1 ? plan.swap : 0;     // (rows g + 8, columns two further: as odd as g)
  const uint16_t *u0 = s_u + (m0 + g) * ld + t * 8, *u1 = u0 + 8 * ld;
  uint4 held[kRegs ? 2 : 1][kPieces<kBf16>][2];
  if (kRegs) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int k = 0; k < kPieces<kBf16>; ++k) {
        held[kRegs ? j : 0][k][0] = 32 * j < ld ? *reinterpret_cast<const uint4*>(u0 + k * piece + (4 * j ^ swap) * 8) : make_uint4(0u, 0u, 0u, 0u);
        held[kRegs ? j : 0][k][1] = 32 * j < ld ? *reinterpret_cast<const uint4*>(u1 + k * piece + (4 * j ^ swap) * 8) : make_uint4(0u, 0u, 0u, 0u);
      }
  }
  for (int step = 0, stage = 0; step < steps; ++step) {
    copies_there(plan.stages2 - 2);
    __syncthreads();  // this stage has arrived for everybody, and everybody has done with the one before
    ask(step + plan.stages2 - 1, stage == 0 ? plan.stages2 - 1 : stage - 1);
    const unsigned char* here = smem + plan.first + stage * plan.stage2;
    stage = stage + 1 == plan.stages2 ? 0 : stage + 1;
    if (m0 >= tile.rows) continue;
    const uint16_t* b = reinterpret_cast<const uint16_t*>(here) + (half + col) * ld + t * 8;
    float d[2][2][4] = {};
    // 32 ranks of a tile: sixteen columns h, instruction i
    auto of_b = [&](int h, int i, int chunk) { return b + (16 * h + 2 * i) * ld + (chunk ^ swap) * 8; };
    if (kRegs) {
      // (B's columns between the adapter's rank and a multiple of 32 are what was there before: zeros by the pieces only if they are numbers, so sixteens
      // are taken by themselves)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (32 * j + 32 <= rank) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(of_b(h, i, 4 * j));
#pragma unroll
              for (int k = 0; k < kPieces<kBf16>; ++k) mma32<kBf16>(d[h][i], held[kRegs ? j : 0][k][0], held[kRegs ? j : 0][k][1], v);
            }
        }
      }
    }
    int j = kRegs ? rank & ~31 : 0;
    for (; j + 32 <= rank; j += 32) {
      uint4 v[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) v[h][i] = *reinterpret_cast<const uint4*>(of_b(h, i, j / 8));
#pragma unroll
      for (int k = 0; k < kPieces<kBf16>; ++k) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(u0 + k * piece + (j / 8 ^ swap) * 8), r1 = *reinterpret_cast<const uint4*>(u1 + k * piece + (j / 8 ^ swap) * 8);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) mma32<kBf16>(d[h][i], r0, r1, v[h][i]);
      }
    }
    if (j < rank) {  // sixteen more: a lane has four of them, in chunk t / 2 of the two
      const int at = (j / 8 ^ swap) * 8 + 4 * t - 8 * t;
#pragma unroll
      for (int k = 0; k < kPieces<kBf16>; ++k) {
        const uint2 r0 = *reinterpret_cast<const uint2*>(u0 + k * piece + at), r1 = *reinterpret_cast<const uint2*>(u1 + k * piece + at);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint2 v = *reinterpret_cast<const uint2*>(b + (16 * h + 2 * i) * ld + at);
            mma<kBf16>(d[h][i], r0.x, r1.x, r0.y, r1.y, v.x, v.y);
          }
      }
    }
    const float4* old = reinterpret_cast<const float4*>(here + kCols * ld * 2) + tid;
    const int n = (step0 + step) * kCols + half + 4 * t;
    const bool whole = (step0 + step + 1) * kCols <= p.N;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float4 o0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o1 = o0;
      if (p.base) {
        o0 = old[2 * h * kThreads];
        o1 = old[(2 * h + 1) * kThreads];
      }
      o0 = make_float4(fmaf(f0, d[h][0][0], o0.x), fmaf(f0, d[h][0][1], o0.y), fmaf(f0, d[h][1][0], o0.z), fmaf(f0, d[h][1][1], o0.w));
      o1 = make_float4(fmaf(f1, d[h][0][2], o1.x), fmaf(f1, d[h][0][3], o1.y), fmaf(f1, d[h][1][2], o1.z), fmaf(f1, d[h][1][3], o1.w));
      if (kVec && whole) {
        if (has0) *reinterpret_cast<float4*>(c0 + 16 * h) = o0;
        if (has1) *reinterpret_cast<float4*>(c1 + 16 * h) = o1;
      } else {
        const float v0[4] = {o0.x, o0.y, o0.z, o0.w}, v1[4] = {o1.x, o1.y, o1.z, o1.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (n + 16 * h + k < p.N) {
            if (has0) c0[16 * h + k] = v0[k];
            if (has1) c1[16 * h + k] = v1[k];
          }
      }
    }
    c0 += kCols;
    c1 += kCols;
  }
  copies_there<0>();
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
  static izb_device_once once[8];
  void (*const kernels[8])(LoraArgs, RowsPlan) = {lora_rows_kernel<false, false, false>, lora_rows_kernel<false, false, true>, lora_rows_kernel<false, true, false>, lora_rows_kernel<false, true, true>,
                                                  lora_rows_kernel<true, false, false>, lora_rows_kernel<true, false, true>, lora_rows_kernel<true, true, false>, lora_rows_kernel<true, true, true>};
  const int which = (bf16 ? 4 : 0) + (vec ? 2 : 0) + (R <= 64 ? 1 : 0);
  if (int rc = once[which].run(device, [&]() -> int {
        IZB_CUDA(cudaFuncSetAttribute(kernels[which], cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RowsPlan(R <= 64 ? 64 : kMaxRank, true).total));
        return IZB_OK;
      }))
    return rc;
  const RowsPlan plan(R, bf16);
  IZB_LAUNCH("lora_add", st, izb_launch_pdl_cluster(kernels[which], kRowsCluster, grid, kThreads, plan.total, st, p, plan));
  return IZB_OK;
}
