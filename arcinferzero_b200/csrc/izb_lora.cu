// Low-rank adapters of many requests beside a shared projection: the rows of a call come in segments, each with an adapter of its own
// or none,
//   u[t][j] = sum_k A[j][k] x[t][k],  x[t][k] = asc[k / 32][t] aq[t][k],      C[t][c_off + n] = base[t][n] + scale * sum_j B[n][j] u[t][j].
//
// Bound by bytes: the adapters' for decode rows, base in and outputs out for prompts (rank 64 over 17408 outputs: 64 operations per byte).  The work is on
// mma.sync with 16-bit operands: the int8 values are exact in them, so the first product is exact up to its f32 sums; u enters the second one in pieces that
// add up to 22 bits or more of it (f16: two, after a power of two per row that brings the row's largest value below 2^14; bf16: three).  (The tcgen05 path
// would want 128 rows of one adapter per tile and its accumulators back through registers for the base; the tensor pipe is 46 % busy at most.)
//
// Measured (us; floor by bytes): one row of 5120 -> 5120, rank 16: 5.0 (0.06); 64 requests of one row, 32 adapters of ranks 8 to 64, 5120 -> 17408: 29 (8.0); 64 of
// four rows, rank 32: 34 (9.2); 8192 rows, ranks 64 and 32, 5120 -> 17408: 265 (182; 245 in a graph of such calls alone), of which
// the second product 205 at 5.5 TB/s.  Off by, against 64 bits, of the norm of the adapters' part, in 2^-24: single rows 2; up to 8 rows, rank 16 / 64 / 256, f16 2 / 3 / 6 and
// bf16 2 / 4 / 10; prompts f16 3 / 4 / 12, bf16 2 / 5 / 15 -- a matrix instruction cuts its sums off, always towards zero, and the second product's are R / 16 per piece in a row.
//
// Two forms.  Decode rows (lora_few_kernel, up to 8 rows per segment on average): one launch and no memory for u.  A cluster of CTAs per tile of up to 8 rows
// of a segment, each with a share of K; the partial sums meet in distributed shared memory, and each CTA goes on with its share of the outputs.
// What bounds it is a chain: which rows, the adapter's first bytes, the exchange of sums (2 + 5 + 2 us), then B.  A call where every request has one row
// takes tiles of one row (lora_few_kernel<.., 1>): less shared memory, three CTAs per multiprocessor, the second product in plain f32.
// Prompts: tiles of up to 64 rows.  lora_inner_kernel makes u's pieces (a cluster per tile, a share of K each) and a list of the tiles; lora_outer_kernel
// deals out steps of 64 rows x 64 outputs in equal stretches.  (Both in one kernel, a cluster per tile, left the last of 3.5 rounds half empty and the
// memory idle during the first product: 312 us for 8192 x 5120 -> 17408 at rank 64.)  In the second product the order of columns within 16 outputs is chosen so
// that a lane has four neighbouring ones: 16-byte copies of the base and stores.
#include <cuda_bf16.h>

#include <type_traits>

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
__device__ __forceinline__ Tile find_tile(const LoraArgs& p, int tile, Tile* s_tile, int* s_sum, int* seen = nullptr) {  // `seen`: of a tile too many, how many there are
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_tile->rows = 0;
  const int asked = tile;
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
  if (seen) *seen = asked - tile;
  return *s_tile;
}

// ---------------------------------------------------------------------------------------------- operands
template <bool kBf16>
__device__ __forceinline__ float2 two_values(uint32_t w) {
  if (kBf16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {  // two IEEE operations in one instruction
  unsigned long long r;
  asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\tmov.b64 c, {%5, %6};\n\tfma.rn.f32x2 %0, a, b, c;\n\t}"
      : "=l"(r) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  float2 o;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(o.x), "=f"(o.y) : "l"(r));
  return o;
}
template <bool kBf16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 32 elements of the inner dimension in two instructions.  The order of the elements within the 32 is free: a lane's elements are 8t .. 8t+7, its column's as
// they lie in memory (16 bytes).  `lo`, `hi`: the row side's registers of the two instructions -- rows g and g + 8 alternate in them, which is why that side
// is always one that is made in registers or laid out for it, and the adapters are the column side: rows as they come would have to be moved together.
template <bool kBf16>
__device__ __forceinline__ void mma32(float (&d)[4], uint4 lo, uint4 hi, uint4 c) {
  mma<kBf16>(d, lo.x, lo.y, lo.z, lo.w, c.x, c.y);
  mma<kBf16>(d, hi.x, hi.y, hi.z, hi.w, c.z, c.w);
}
// Where element j of a row of `rank` is among such registers: the 16 bytes of a lane, as a number of 32-lane groups, and the 16-bit value in them.  (The last
// sixteen of a rank that is no multiple of 32 are one instruction's, four per lane.)
struct Place {
  int group, t, value;  // (value: 4 * register pair + half)
};
__device__ __forceinline__ Place place_of(int j, int rank) {
  const int chunk = j >> 5;
  if (chunk * 32 + 32 <= rank) return {chunk * 2 + ((j >> 2) & 1), (j & 31) >> 3, ((j >> 1) & 1) * 4 + (j & 1)};
  return {chunk * 2, (j & 15) >> 2, ((j >> 1) & 1) * 4 + (j & 1)};
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
// A warp makes the pieces of a row from its sums, put(piece, j, 16-bit value); the factor that the second product's result takes.  A row with a sum that is no
// finite number is NaN.
template <bool kBf16, class Sum, class Put>
__device__ __forceinline__ float make_pieces(int rank, Sum sum, Put put) {
  const int lane = threadIdx.x & 31;
  if (kBf16) {
    for (int j = lane; j < rank; j += 32) {
      float u = sum(j);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const __nv_bfloat16 h = __float2bfloat16_rn(u);
        put(i, j, __bfloat16_as_ushort(h));
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
    u[i] = 0.0f;
    if (i * 32 < rank && j < rank) u[i] = sum(j);
    most = max(most, __float_as_uint(u[i]) & 0x7FFFFFFFu);
  }
  most = __reduce_max_sync(0xFFFFFFFFu, most);
  const int ex = max((int)(most >> 23) - 127, -100);  // |u| < 2^(ex + 1)
  const bool none = most >= 0x7F800000u;
#pragma unroll
  for (int i = 0; i < kMaxRank / 32; ++i) {
    const int j = i * 32 + lane;
    if (i * 32 >= rank || j >= rank) break;
    const float v = none ? __uint_as_float(0x7FC00000u) : ldexpf(u[i], 13 - ex);
    const __half h = __float2half_rn(v);
    put(0, j, __half_as_ushort(h));
    put(1, j, __half_as_ushort(__float2half_rn(v - __half2float(h))));
  }
  return ldexpf(1.0f, ex - 13);
}

// ---------------------------------------------------------------------------------------------- asynchronous copies
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
// Pieces of an adapter (16 rows x 32 elements, 1 KB, and what the base has for them: 16 bytes per lane, of a single row 4) that a warp has asked for
template <int kRowsOf>
constexpr int kFewSlots = kRowsOf == 1 ? 5 : 6;
template <int kRowsOf>
constexpr int kFewSlot = kRowsOf == 1 ? 1152 : 1536;
template <int kRowsOf>
constexpr int kFewBlocks = kRowsOf == 1 ? 3 : 2;  // CTAs per multiprocessor
constexpr int kFewPart = kFewRanks * 16 + 8;  // a row of partial sums (the padding: rows on different banks)
// rings | partial sums of the warps | those of the CTAs | the pieces of u, two to an instruction
template <int kRowsOf>
static size_t few_smem(int R, int cluster) {
  return (size_t)kWarps * kFewSlots<kRowsOf> * kFewSlot<kRowsOf> + (size_t)kWarps * kRowsOf * kFewPart * 4 + (size_t)cluster * kRowsOf * (R + 8) * 4 + (size_t)2 * ((R + 31) / 32) * 1024;
}
// The adapter streams through a ring per warp: each lane copies what it will read itself (16 bytes of two of its rows), so that nobody waits for anybody, and
// the second product's first pieces are on their way while the first one's sums are exchanged.  The adapter's rows are the instruction's columns, tokens its
// rows: the upper eight rows are empty in the first product, and hold the second piece of u in the second one.
template <bool kBf16, int kRowsOf>
__global__ void __launch_bounds__(kThreads, kFewBlocks<kRowsOf>) lora_few_kernel(LoraArgs p) {
  constexpr int kSlots = kFewSlots<kRowsOf>, kSlot = kFewSlot<kRowsOf>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  __shared__ float s_factor[kRowsOf];
  float* s_part = reinterpret_cast<float*>(smem + kWarps * kSlots * kSlot);              // [warp][rows][kFewPart]
  float* s_all = s_part + kWarps * kRowsOf * kFewPart;                                    // [CTA][rows][R + 8]
  unsigned char* s_u = reinterpret_cast<unsigned char*>(s_all + (size_t)p.cluster * kRowsOf * (p.R + 8));  // [two pieces][groups of 32 lanes][16 bytes]
  const int rank_of_cta = blockIdx.x % p.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cluster_arrive();  // (waited for before anything is written to another CTA)
  pdl_launch_next();
  pdl_wait();
  const Tile tile = find_tile<kRowsOf>(p, blockIdx.x / p.cluster, &s_tile, s_sum);
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
  // (A single row is dealt with in f32 -- an instruction for eight rows would be an eighth of its own worth: two lanes on an output up to rank 16, else four, of
  // which each has 8 elements of a piece's 16, 32 or, beyond that, two times 8 of 64.)
  const bool single = kRowsOf == 1 || tile.rows == 1, split = single && rank > 32;
  const int lanes_log = rank <= 16 ? 1 : 2, lanes = 1 << lanes_log, unit = !single ? 16 : split ? 8 : 64 >> lanes_log;
  const int tiles = (p.N + unit - 1) / unit, nt0 = share(tiles, p.cluster * kWarps, rank_of_cta * kWarps + warp), nt1 = share(tiles, p.cluster * kWarps, rank_of_cta * kWarps + warp + 1);
  const int whole = p.N / unit;  // (a last tile may be cut off)

  // ---- the ring: pieces in the order in which they are used below
  unsigned char* ring = smem + warp * kSlots * kSlot + lane * 16;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  int ask_slot = 0, ask_j0 = kb0 < kb1 ? 0 : rank, ask_kb = kb0, ask_i = 0, ask_nt = nt0, ask_j = 0;
  const size_t eight_a = (size_t)8 * p.K;
  // of sixteen outputs a lane's columns are col and col + 2: it then has four neighbouring ones (see below)
  const int col = single ? lane >> lanes_log : 4 * (g >> 1) + (g & 1), col_step = !single ? 2 : split ? 0 : unit / 2;
  const size_t step_b = (size_t)col_step * p.R, unit_b = (size_t)unit * p.R;
  const uint16_t* ask_a = A + (size_t)g * p.K + kb0 * 32 + 8 * t;  // of rank tile 0 and ask_kb
  const uint16_t* ask_b = B + (size_t)(nt0 * unit + col) * p.R;    // of ask_nt
  // A lane's outputs: row g, four neighbouring ones of sixteen.  Of a single row: where the halves of a piece are two outputs, the sum over the lanes that share
  // them leaves the second one with those of the upper half.
  const bool upper = !split && lane & (lanes >> 1), mine_has = single ? (split ? (lane & 3) == 0 : (lane & ((lanes >> 1) - 1)) == 0) : g < tile.rows;
  const int out_at = single ? (upper ? col_step : 0) + col : 4 * t;
  const size_t out_row = (size_t)tile.row + (single ? 0 : min(g, tile.rows - 1));
  const bool vec = (((uintptr_t)p.C | (uintptr_t)p.base) & 15) == 0 && ((p.ldc | (p.base ? p.ldb : 0)) & 3) == 0;
  const float* ask_base = p.base + out_row * p.ldb + nt0 * unit + out_at;  // (not looked at without a base)
  float* to = p.C + out_row * p.ldc + nt0 * unit + out_at;
  auto ask = [&]() {
    const uint32_t to = ring_at + ask_slot * kSlot;
    ask_slot = ask_slot + 1 == kSlots ? 0 : ask_slot + 1;
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
      const uint16_t *from0 = ask_b + ask_j, *from1 = from0 + step_b;
      if (ask_nt >= whole) {
        from0 = B + (size_t)min(ask_nt * unit + col, p.N - 1) * p.R + ask_j;
        from1 = B + (size_t)min(ask_nt * unit + col + col_step, p.N - 1) * p.R + ask_j;
      }
      if (ask_j == 0 && p.base && mine_has) {  // what this lane will add
        const bool cut = ask_nt >= whole;
        const int n = ask_nt * unit + out_at;
        if (single) {
          if (!cut || n < p.N) copy4(to + 1024 - (kRowsOf == 1 ? lane * 12 : 0), ask_base);
        } else if (vec && !cut) {
          copy16(to + 1024, ask_base);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (n + k < p.N) copy4(to + 1024 + 4 * k, ask_base + k);
        }
      }
      if (single) {  // (past the rank: zeros)
        const int j0 = (lane & (lanes - 1)) * 8, j1 = split ? j0 + 32 : j0, bytes0 = ask_j + j0 < rank ? 16 : 0, bytes1 = ask_j + j1 < rank ? 16 : 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %3;\n\tcp.async.cg.shared.global [%0+512], [%2], 16, %4;" ::"r"(to), "l"(from0 + (bytes0 ? j0 : 0)),
                     "l"(from1 + (bytes1 ? j1 : 0)), "r"(bytes0), "r"(bytes1)
                     : "memory");
        ask_j += 64;
      } else if (ask_j + 32 <= rank) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n\tcp.async.cg.shared.global [%0+512], [%2], 16;" ::"r"(to), "l"(from0 + 8 * t), "l"(from1 + 8 * t) : "memory");
        ask_j += 32;
      } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;\n\tcp.async.ca.shared.global [%0+512], [%2], 8;" ::"r"(to), "l"(from0 + 4 * t), "l"(from1 + 4 * t) : "memory");
        ask_j += 32;
      }
      if (ask_j >= rank) {
        ask_j = 0;
        ++ask_nt;
        ask_b += unit_b;
        ask_base += unit;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int slot = 0;
  auto take = [&](uint4& r0, uint4& r1, float4& base) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
    r0 = *reinterpret_cast<const uint4*>(ring + slot * kSlot);
    r1 = *reinterpret_cast<const uint4*>(ring + slot * kSlot + 512);
    // (of an output's first piece)
    if (kRowsOf == 1) base.x = *reinterpret_cast<const float*>(ring + slot * kSlot + 1024 - lane * 12);
    else base = *reinterpret_cast<const float4*>(ring + slot * kSlot + 1024);
    slot = slot + 1 == kSlots ? 0 : slot + 1;
    ask();
  };
  const int8_t* x = p.aq + (size_t)(tile.row + min(g, tile.rows - 1)) * p.K + 8 * t;
  const float* xs = p.asc + tile.row + min(g, tile.rows - 1);
  uint2 v_next = make_uint2(0u, 0u);
  float s_next = 0.0f;
  auto values = [&](int kb) {
    if (kb >= kb1) return;
    v_next = *reinterpret_cast<const uint2*>(x + kb * 32);
    s_next = xs[(size_t)kb * p.Mp];
  };
  values(kb0);  // (ahead of what fills the queues to memory)
#pragma unroll
  for (int i = 0; i < kSlots; ++i) ask();

  // ---- u
  for (int j0 = 0; j0 < rank; j0 += kFewRanks * 16) {
    float acc[kFewRanks][4] = {};  // row g, ranks 2t, 2t + 1, 8 + 2t, 9 + 2t of the tile
    if (j0) values(kb0);
    for (int kb = kb0; kb < kb1; kb += kWarps) {
      const uint4 v = eight_of<kBf16>(v_next);
      const float s0 = s_next;
      values(kb + kWarps);
#pragma unroll
      for (int i = 0; i < kFewRanks; ++i)
        if (j0 + i * 16 < rank) {
          uint4 r[2];
          float4 none;
          take(r[0], r[1], none);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float d[4] = {};
            mma32<kBf16>(d, make_uint4(v.x, 0u, v.y, 0u), make_uint4(v.z, 0u, v.w, 0u), r[h]);
            acc[i][2 * h] = fmaf(s0, d[0], acc[i][2 * h]);
            acc[i][2 * h + 1] = fmaf(s0, d[1], acc[i][2 * h + 1]);
          }
        }
    }
#pragma unroll
    for (int i = 0; i < kFewRanks; ++i)
      if (j0 + i * 16 < rank && g < kRowsOf) {
        float* to = s_part + (warp * kRowsOf + g) * kFewPart + i * 16 + 2 * t;
        *reinterpret_cast<float2*>(to) = make_float2(acc[i][0], acc[i][1]);
        *reinterpret_cast<float2*>(to + 8) = make_float2(acc[i][2], acc[i][3]);
      }
    __syncthreads();
    if (j0 == 0) cluster_wait();  // every CTA has begun
    // the warps' sums, four values per thread, to every CTA
    const int row = tid >> 4, j = (tid & 15) * 4;
    if (row < tile.rows && j0 + j < rank) {
      const float* from = s_part + row * kFewPart + j;
      float4 v = *reinterpret_cast<const float4*>(from);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 b = *reinterpret_cast<const float4*>(from + w * kRowsOf * kFewPart);
        v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
      }
      const float* here = s_all + ((size_t)rank_of_cta * kRowsOf + row) * (p.R + 8) + j0 + j;
      for (int c = 0; c < p.cluster; ++c) remote_store(at_rank(here, c), v);
    }
    __syncthreads();
  }
  cluster_arrive();
  cluster_wait();
  // ---- a single row: its sums as they are, and outputs by lanes that share a row of B
  if (single) {
    float* s_f = reinterpret_cast<float*>(s_u);
    for (int j = tid; j < ((rank + 63) & ~63); j += kThreads) {
      float u = 0.0f;
      if (j < rank)
#pragma unroll 8
        for (int c = 0; c < p.cluster; ++c) u += s_all[(size_t)c * kRowsOf * (p.R + 8) + j];
      s_f[j] = u;
    }
    __syncthreads();
    const float* mine = s_f + (lane & (lanes - 1)) * 8;
    float2 u[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) u[h][e] = *reinterpret_cast<const float2*>(mine + (split ? 32 * h : 0) + 2 * e);
    int nt = nt0;
    auto sum_of = [&](const float2 (&v)[2]) {  // over the lanes that share an output (or two)
      const float a = v[0].x + v[0].y, b = v[1].x + v[1].y;
      if (split) {
        float y = a + b;
        y += __shfl_xor_sync(0xFFFFFFFFu, y, 2);
        return y + __shfl_xor_sync(0xFFFFFFFFu, y, 1);
      }
      const float y = (upper ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, upper ? a : b, lanes >> 1);
      return lanes == 4 ? y + __shfl_xor_sync(0xFFFFFFFFu, y, 1) : y;
    };
    auto add = [&](float2 (&v)[2], const uint4 (&r)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w[4] = {r[h].x, r[h].y, r[h].z, r[h].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h] = fma2(two_values<kBf16>(w[e]), u[h][e], v[h]);
      }
    };
    // Whole units of one piece each, which are nearly all there are: the ring's upkeep is a few additions (take() and ask() are four times as much)
    if (rank <= 64 && ask_nt < nt1) {
      const int j0 = (lane & (lanes - 1)) * 8, j1 = split ? j0 + 32 : j0, bytes0 = j0 < rank ? 16 : 0, bytes1 = j1 < rank ? 16 : 0;
      const uint16_t *from0 = ask_b + (bytes0 ? j0 : 0), *from1 = ask_b + step_b + (bytes1 ? j1 : 0);
      const float* base_from = ask_base;
      const bool with_base = p.base && mine_has;
      const int ask_end = min(nt1, whole);
      // (while what is asked for is whole, what is taken is)
      for (; ask_nt < ask_end; ++ask_nt, ++nt) {
        copies_there<kSlots - 1>();
        const unsigned char* here = ring + slot * kSlot;
        const uint4 r[2] = {*reinterpret_cast<const uint4*>(here), *reinterpret_cast<const uint4*>(here + 512)};
        const float base = with_base ? *reinterpret_cast<const float*>(here + 1024 - (kRowsOf == 1 ? lane * 12 : 0)) : 0.0f;
        const uint32_t at = ring_at + slot * kSlot;  // (the slot that has been read is the next one to fill)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %3;\n\tcp.async.cg.shared.global [%0+512], [%2], 16, %4;" ::"r"(at), "l"(from0), "l"(from1), "r"(bytes0), "r"(bytes1) : "memory");
        if (with_base) copy4(at + 1024 - (kRowsOf == 1 ? lane * 12 : 0), base_from);
        copies_begun();
        from0 += unit_b;
        from1 += unit_b;
        base_from += unit;
        slot = slot + 1 == kSlots ? 0 : slot + 1;
        float2 v[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        add(v, r);
        const float y = sum_of(v);
        if (mine_has) *to = fmaf(tile.scale, y, base);
        to += unit;
      }
      ask_slot = slot;
      ask_b += unit_b * (size_t)(nt - nt0);
      ask_base += (size_t)unit * (nt - nt0);
    }
    for (; nt < nt1; ++nt, to += unit) {
      float base = 0.0f;
      float2 v[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
      for (int j = 0; j < rank; j += 64) {
        uint4 r[2];
        float4 here;
        take(r[0], r[1], here);
        if (j == 0 && p.base) base = here.x;
        if (rank > 64) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) u[h][e] = *reinterpret_cast<const float2*>(mine + j + 32 * h + 2 * e);
        }
        add(v, r);
      }
      const float y = sum_of(v);
      if (mine_has && (nt < whole || nt * unit + out_at < p.N)) *to = fmaf(tile.scale, y, base);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    return;
  }
  if (kRowsOf == 1) return;
  // ---- the sums of the CTAs in order; a warp per row
  const int chunks = (p.R + 31) / 32;
  if (warp < tile.rows) {
    const float f = make_pieces<kBf16>(rank, [&](int j) {
      const float* from = s_all + warp * (p.R + 8) + j;
      float u = 0.0f;
#pragma unroll 8
      for (int c = 0; c < p.cluster; ++c) u += from[(size_t)c * kRowsOf * (p.R + 8)];
      return u;
    }, [&](int i, int j, uint16_t v) {
      const Place at = place_of(j, rank);
      *reinterpret_cast<uint16_t*>(s_u + ((size_t)(i >> 1) * 2 * chunks + at.group) * 512 + (warp * 4 + at.t) * 16 + (at.value + 2 * (i & 1)) * 2) = v;
    });
    if (lane == 0) s_factor[warp] = f;
  }
  __syncthreads();

  // ---- outputs
  const float f = mine_has ? tile.scale * s_factor[g] : 0.0f;
  const unsigned char* u = s_u + lane * 16;
  for (int nt = nt0; nt < nt1; ++nt, to += 16) {
    float4 base = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float d[2][4] = {};
    for (int j = 0; j < rank; j += 32) {
      uint4 r[2];
      float4 here;
      take(r[0], r[1], here);
      if (j == 0 && p.base) base = here;
#pragma unroll
      for (int i = 0; i < (kBf16 ? 2 : 1); ++i) {
        const unsigned char* of = u + ((size_t)i * 2 * chunks + j / 16) * 512;
        uint4 lo = *reinterpret_cast<const uint4*>(of), hi = *reinterpret_cast<const uint4*>(of + 512);
        if (i) lo.y = lo.w = hi.y = hi.w = 0u;  // (the third piece is alone)
        if (j + 32 <= rank) {
          mma32<kBf16>(d[0], lo, hi, r[0]);
          mma32<kBf16>(d[1], lo, hi, r[1]);
        } else {  // sixteen more
          mma<kBf16>(d[0], lo.x, lo.y, lo.z, lo.w, r[0].x, r[0].y);
          mma<kBf16>(d[1], lo.x, lo.y, lo.z, lo.w, r[1].x, r[1].y);
        }
      }
    }
    if (!mine_has) continue;
    const float4 y = make_float4(fmaf(f, d[0][0] + d[0][2], base.x), fmaf(f, d[0][1] + d[0][3], base.y), fmaf(f, d[1][0] + d[1][2], base.z), fmaf(f, d[1][1] + d[1][3], base.w));
    if (vec && nt < whole) {
      *reinterpret_cast<float4*>(to) = y;
    } else {
      const int left = p.N - nt * 16 - 4 * t;
      if (left > 0) to[0] = y.x;
      if (left > 1) to[1] = y.y;
      if (left > 2) to[2] = y.z;
      if (left > 3) to[3] = y.w;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------------------------- up to 64 rows
constexpr int kRows = 64;         // rows of a tile
constexpr int kCols = 64;         // outputs of a step of the second product
constexpr int kPitch = 72;        // floats of a step's row in shared memory where it starts anywhere (up to 17 chunks of 16 bytes)
// Where rows of base and outputs start: both on 16-byte boundaries; anywhere, but each row's two alike; anywhere
enum { kOnLines, kAlike, kAnywhere };
// A's and B's tiles: rows of whole 64 bytes in 16-byte chunks; where a row is a multiple of 128 bytes odd rows have the halves of their
// 128-byte lines changed over, so that two neighbouring rows' 64 bytes lie on different banks.
struct RowsPlan {
  int groups, parts;                  // warps by ranks (64 each) and by blocks of K in the first product; two more by rows (32 each)
  int ld, swap;                       // a row of B in 16-bit values (a multiple of 32); what odd rows' chunk numbers are xored with
  int stages2;                        // of asynchronous copies in the second product (three in the first)
  uint32_t stage1, stage2;            // bytes: activations | their scales | A's tile; B's tile | base
  uint32_t all, total1;               // first product: the CTAs' sums lie behind the stages and, over them, the warps' sums
  uint32_t pieces, total2;            // second product: u's pieces, then stages
  uint32_t at_tiles, at_factors, at_pieces;  // scratch: number of tiles | Tile each | 64 factors each | pieces each
  RowsPlan(int R, bool bf16, size_t tiles, int place = kOnLines) {
    groups = R <= 64 ? 1 : R <= 128 ? 2 : 4;
    parts = kWarps / 2 / groups;
    ld = (R + 31) / 32 * 32;
    swap = ld % 64 ? 0 : 4;
    stage1 = parts * (kRows * 32 + kRows * 4 + R * 64);
    const uint32_t part = (uint32_t)parts * kRows * (R + 8) * 4;
    all = part > 3 * stage1 ? part : 3 * stage1;
    total1 = all + (uint32_t)kRows * (R + 8) * 4;
    pieces = (bf16 ? 3 : 2) * kRows * ld * 2;
    stage2 = kCols * ld * 2 + kRows * (place == kAlike ? kPitch : kCols) * 4;
    const uint32_t half_sm = (228 << 10) / 2 - 1024;
    auto fits = [&](int stages, uint32_t room) { return pieces + stages * stage2 <= room; };
    stages2 = fits(3, half_sm) || (!fits(2, half_sm) && fits(3, kMost2)) ? 3 : 2;  // (two CTAs per multiprocessor before a third stage)
    total2 = pieces + stages2 * stage2;
    at_tiles = 16;
    at_factors = (uint32_t)(at_tiles + tiles * sizeof(Tile) + 15) / 16 * 16;
    at_pieces = (uint32_t)(at_factors + tiles * kRows * 4);
  }
  static constexpr int kMost2 = 227 << 10;   // total2 at most
  size_t scratch(size_t tiles) const { return at_pieces + tiles * pieces; }
};
// The first product: u's pieces, rows' factors and the tile's place, into scratch.
template <bool kBf16, int kParts>
__global__ void __launch_bounds__(kThreads, 2) lora_inner_kernel(LoraArgs p, RowsPlan plan, unsigned char* scratch) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Tile s_tile;
  __shared__ int s_sum[kWarps];
  float* s_part = reinterpret_cast<float*>(smem);              // [K part][64 rows][R + 8]
  float* s_all = reinterpret_cast<float*>(smem + plan.all);    // [CTA][rows that this CTA joins][R + 8]
  const int ldp = p.R + 8;
  const int index = blockIdx.x / p.cluster, rank_of_cta = blockIdx.x % p.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  cluster_arrive();
  pdl_wait();
  pdl_launch_next();
  int seen = 0;
  const Tile tile = find_tile<kRows>(p, index, &s_tile, s_sum, &seen);
  if (tid == 0 && rank_of_cta == 0) {
    if (tile.rows) reinterpret_cast<Tile*>(scratch + plan.at_tiles)[index] = tile;
    if (blockIdx.x + p.cluster == gridDim.x) *reinterpret_cast<int*>(scratch) = tile.rows ? index + 1 : seen;
  }
  if (!tile.rows || tile.rank == 0) {
    cluster_wait();
    return;
  }
  const uint16_t* A = p.A + (size_t)tile.adapter * p.R * p.K;
  const int rank = (tile.rank + 15) & ~15;

  // ---- a warp has 64 ranks x 32 rows, and every parts-th 32-block of the CTA's share of K; `parts` blocks per stage
  constexpr int parts = kParts;
  const int part = warp % parts, r0 = (warp / parts & 1) * 32, j0 = warp / (2 * parts) * 64;
  {
    const int kb0 = share(p.K / 32, p.cluster, rank_of_cta), kb1 = share(p.K / 32, p.cluster, rank_of_cta + 1), steps = (kb1 - kb0 + parts - 1) / parts;
    constexpr int row_log = parts == 4 ? 4 : parts == 2 ? 3 : 2, swap = parts > 1 ? 4 : 0;  // a row of A's tile: 2^row_log chunks
    const uint32_t stages_at = (uint32_t)__cvta_generic_to_shared(smem), scales_at = parts * kRows * 32, a_at = scales_at + parts * kRows * 4;
    // (rows past the tile's: the last one again, which nobody reads)
    const int8_t* x_from = p.aq + (size_t)(tile.row + min((tid >> 1) & (kRows - 1), tile.rows - 1)) * p.K + (kb0 + (tid >> 7)) * 32 + (tid & 1) * 16;
    const float* s_from = p.asc + (size_t)(kb0 + (tid >> 6)) * p.Mp + tile.row + min(tid & (kRows - 1), tile.rows - 1);
    const int a_c = tid & ((1 << row_log) - 1), a_j = tid >> row_log, a_step = kThreads >> row_log;
    const uint16_t* a_from = A + (size_t)a_j * p.K + kb0 * 32 + a_c * 8;
    const size_t a_rows = (size_t)a_step * p.K;
    const uint32_t a_to = a_at + ((a_j << row_log) + (a_c ^ (a_j & 1 ? swap : 0))) * 16;  // (a_step is even: the rows of a thread are all odd or all even)
    auto ask = [&](int step, int stage) {
      if (step < steps) {
        const uint32_t to = stages_at + stage * plan.stage1;
        const int blocks = min(parts, kb1 - kb0 - step * parts), k = step * parts * 32;
#pragma unroll
        for (int i = 0; i < parts * kRows * 2; i += kThreads)
          if (tid + i < blocks * kRows * 2) copy16(to + (tid + i) * 16, x_from + k + i / 4);
        if (tid < blocks * kRows) copy4(to + scales_at + tid * 4, s_from + (size_t)(step * parts) * p.Mp);
        if (a_c < blocks * 4) {
          const uint16_t* from = a_from + k;
          for (int j = a_j, i = 0; j < rank; j += a_step, ++i, from += a_rows) copy16(to + a_to + i * (kThreads * 16), from);
        }
      }
      copies_begun();
    };
    float acc[2][8][4] = {};  // rows 16 m + g, + 8, ranks 8 i + 2t, 2t + 1
    ask(0, 0);
    ask(1, 1);
    for (int step = 0, stage = 0; step < steps; ++step) {
      copies_there<1>();
      __syncthreads();
      ask(step + 2, stage == 0 ? 2 : stage - 1);
      const unsigned char* here = smem + stage * plan.stage1;
      stage = stage == 2 ? 0 : stage + 1;
      if (j0 >= rank || kb0 + step * parts + part >= kb1 || r0 >= tile.rows) continue;
      const uint2* x = reinterpret_cast<const uint2*>(here + part * kRows * 32) + (r0 + g) * 4 + t;
      const float* xs = reinterpret_cast<const float*>(here + scales_at + part * kRows * 4) + r0 + g;
      const uint4* a = reinterpret_cast<const uint4*>(here + a_at) + ((size_t)(j0 + g) << row_log) + ((part * 4) ^ (g & 1 ? swap : 0)) + t;
      uint4 lo[2], hi[2];
      float sc[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint4 v = eight_of<kBf16>(x[m * 64]), w = eight_of<kBf16>(x[m * 64 + 32]);
        lo[m] = make_uint4(v.x, w.x, v.y, w.y);
        hi[m] = make_uint4(v.z, w.z, v.w, w.w);
        sc[m][0] = xs[16 * m];
        sc[m][1] = xs[16 * m + 8];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (j0 + 8 * i >= rank) break;
        const uint4 c = a[(8 * i) << row_log];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float d[4] = {};
          mma32<kBf16>(d, lo[m], hi[m], c);
          acc[m][i][0] = fmaf(sc[m][0], d[0], acc[m][i][0]);
          acc[m][i][1] = fmaf(sc[m][0], d[1], acc[m][i][1]);
          acc[m][i][2] = fmaf(sc[m][1], d[2], acc[m][i][2]);
          acc[m][i][3] = fmaf(sc[m][1], d[3], acc[m][i][3]);
        }
      }
    }
    copies_there<0>();
    __syncthreads();  // (the partial sums go over the stages)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j0 + 8 * i < rank)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float* to = s_part + (size_t)(part * kRows + r0 + 16 * m + g) * ldp + j0 + 8 * i + 2 * t;
          *reinterpret_cast<float2*>(to) = make_float2(acc[m][i][0], acc[m][i][1]);
          *reinterpret_cast<float2*>(to + 8 * ldp) = make_float2(acc[m][i][2], acc[m][i][3]);
        }
  }
  __syncthreads();
  cluster_wait();  // every CTA has begun
  // the CTA's sums, four ranks per thread, to the CTA that joins these rows
  const int own = kRows / p.cluster;  // (4, 8, 16, 32 or 64)
  {
    const int row = tid >> 2;
    for (int j = (tid & 3) * 4; j < rank && row < tile.rows; j += 16) {
      const float* from = s_part + (size_t)row * ldp + j;
      float4 v = *reinterpret_cast<const float4*>(from);
      for (int w = 1; w < parts; ++w) {
        const float4 b = *reinterpret_cast<const float4*>(from + (size_t)w * kRows * ldp);
        v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
      }
      remote_store(at_rank(s_all + ((size_t)rank_of_cta * own + (row & (own - 1))) * ldp + j, row / own), v);
    }
  }
  cluster_arrive();
  cluster_wait();
  // ---- a warp per row of its CTA: the sums of the CTAs in order.  The pieces lie as the second product's instructions take them: [piece][16 rows][32 lanes' 16
  // bytes per instruction]
  unsigned char* u = scratch + plan.at_pieces + (size_t)index * plan.pieces;
  float* factors = reinterpret_cast<float*>(scratch + plan.at_factors) + (size_t)index * kRows;
  for (int i = warp; i < own; i += kWarps) {
    const int row = rank_of_cta * own + i;
    if (row >= tile.rows) break;
    const float f = make_pieces<kBf16>(rank, [&](int j) {
      const float* from = s_all + (size_t)i * ldp + j;
      float sum = 0.0f;
#pragma unroll 8
      for (int c = 0; c < p.cluster; ++c) sum += from[(size_t)c * own * ldp];
      return sum;
    }, [&](int k, int j, uint16_t v) {
      const Place at = place_of(j, rank);
      *reinterpret_cast<uint16_t*>(u + ((size_t)(k * 4 + (row >> 4)) * (plan.ld / 16) + at.group) * 512 + ((row & 7) * 4 + at.t) * 16 + (at.value + (row & 8 ? 2 : 0)) * 2) = v;
    });
    if (lane == 0) factors[row] = tile.scale * f;
  }
}

// The second product, base and outputs: steps of 64 rows x 64 outputs, an equal stretch of all of them for each CTA.
// kRegs: the ranks are 64 at most, and a warp holds its rows' pieces in registers
// kPlace: what base and outputs go through.  On boundaries a lane copies the 16 bytes that it adds to, and stores 16 bytes.  Where each row of the base starts as
// far from a boundary as the outputs' row, a step's 64 x 64 go through shared memory as they lie in memory, 16-byte chunks from boundary to boundary, both ways;
// a chunk is copied and stored by one thread, so that no barrier is needed for it to be filled again.  Else single values (6469 rows, 1024 -> 3416, rows of 3419:
// 126 us, through shared memory 104).
template <bool kBf16, int kPlace, bool kRegs>
__global__ void __launch_bounds__(kThreads, 2) lora_outer_kernel(LoraArgs p, RowsPlan plan, const unsigned char* scratch) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3, ld = plan.ld;
  const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(smem), stages_at = smem_at + plan.pieces;
  const bool in_place = p.base == p.C;
  constexpr bool kVec = kPlace == kOnLines;
  pdl_launch_next();
  pdl_wait();
  const int per = (p.N + kCols - 1) / kCols;
  const long long all = (long long)*reinterpret_cast<const int*>(scratch) * per;
  const long long begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
  if (begin >= end) return;
  const Tile* tiles = reinterpret_cast<const Tile*>(scratch + plan.at_tiles);

  // Column g of the first instruction, and how much further that of the second one is.  Where rows lie on 16-byte boundaries a lane has four neighbouring outputs;
  // else two and two, so that the four lanes of a row share 32 bytes at a time.
  const int col = kVec ? 4 * (g >> 1) + (g & 1) : g, col_step = kVec ? 2 : 8, out0 = kVec ? 4 * t : 2 * t;
  auto out_of = [&](int k) { return kVec ? k : (k >> 1) * 8 + (k & 1); };
  const int swap = g & 1 ? plan.swap : 0;     // (both columns are as odd as g)
  const int b_row = tid >> 2, b_chunk = tid & 3;  // four threads copy a row of B
  const uint32_t b_to = stages_at + (b_row * ld + (b_chunk ^ (b_row & 1 ? plan.swap : 0)) * 8) * 2, b_swap = b_row & 1 && plan.swap ? 0xFFFFFFC0u : 64u;  // (the next four chunks)
  const uint32_t base_to = stages_at + kCols * ld * 2 + (kPlace == kAlike ? (b_row * kPitch + b_chunk * 4) * 4 : tid * 16);
  uint4 held[kRegs ? 2 : 1][kPieces<kBf16>][2] = {};

  // A tile's steps in this CTA's stretch, one tile after the other
  int index = (int)(begin / per), step0 = (int)(begin % per);
  for (long long left = end - begin; left > 0; ++index, step0 = 0) {
    const Tile tile = tiles[index];
    // A warp has 16 rows and 32 of the 64 outputs; of a tile of 32 rows or fewer 16 outputs, so that all four tensor cores have work (42 segments of 9 rows,
    // 3840 -> 11281 at rank 128: 110 us against 129; 16 of 16, 5120 -> 17408 at rank 64: 32 against 38)
    const bool narrow = tile.rows <= 32;
    const int m0 = (narrow ? warp >> 2 : warp & 3) * 16, half = narrow ? (warp & 3) * 16 : (warp >> 2) * 32;
    auto of_u = [&](int k, int group) { return *reinterpret_cast<const uint4*>(smem + ((k * 4 + (m0 >> 4)) * (ld / 16) + group) * 512 + lane * 16); };
    const int steps = (int)min(left, (long long)(per - step0)), rank = (tile.rank + 15) & ~15;
    left -= steps;
    if (in_place && rank == 0) continue;
    __syncthreads();  // (everybody has done with the tile before)

    // ---- copies: a row of B per four threads, and for each lane what it will add: rows g and g + 8, four outputs of both of its warp's sixteens
    const int mine = (rank / 8 - b_chunk + 3) / 4;  // 16-byte chunks of the row for this thread
    const bool has0 = m0 + g < tile.rows, has1 = m0 + g + 8 < tile.rows;
    const uint16_t* b_from = p.B + ((size_t)(rank ? tile.adapter : 0) * p.N + step0 * kCols + b_row) * p.R + b_chunk * 8;
    const size_t row = tile.row + m0 + g;
    // (rows past the tile's: the last one again, which nobody stores)
    const float* from0 = p.base + (size_t)(tile.row + min(m0 + g, tile.rows - 1)) * p.ldb + step0 * kCols + half + out0;
    const float* from1 = p.base + (size_t)(tile.row + min(m0 + g + 8, tile.rows - 1)) * p.ldb + step0 * kCols + half + out0;
    // (kAlike: what this thread copies and stores, of row b_row the chunks b_chunk, b_chunk + 4, ...; chunk c holds the step's outputs 4c - shift .. 4c - shift + 3)
    const float* line_from = p.base + (size_t)(tile.row + min(b_row, tile.rows - 1)) * p.ldb;
    float* line_to = p.C + (size_t)(tile.row + min(b_row, tile.rows - 1)) * p.ldc;
    auto shift_of = [&](const float* at) { return (int)((uintptr_t)at >> 2) & 3; };
    const int shift = shift_of(line_to), chunks = b_row < tile.rows ? (kCols + shift + 3) / 4 : 0;
    auto store = [&](const unsigned char* stage, int n) {  // the step from output n on
      const float* from = reinterpret_cast<const float*>(stage + kCols * ld * 2) + b_row * kPitch;
#pragma unroll
      for (int j = 0; j < 5; ++j) {
        const int c = b_chunk + 4 * j, lo = 4 * c - shift;
        if (c >= chunks) break;
        const float4 v = *reinterpret_cast<const float4*>(from + 4 * c);
        float* to = line_to + n + lo;
        if (lo >= 0 && lo + 4 <= kCols && n + lo + 4 <= p.N) {
          *reinterpret_cast<float4*>(to) = v;
        } else {
          const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (lo + k >= 0 && lo + k < kCols && n + lo + k < p.N) to[k] = w[k];
        }
      }
    };
    int ask_n = step0 * kCols;         // the next step's first output
    int ask_left = steps;
    uint32_t ask_at = 0;               // its stage
    const uint32_t stages_end = plan.stages2 * plan.stage2;
    auto ask = [&]() {
      if (ask_left > 0) {
        --ask_left;
        if (ask_n + kCols <= p.N) {
          if (kRegs) {
            if (mine > 0) copy16(b_to + ask_at, b_from);
            if (mine > 1) copy16(b_to + ask_at + b_swap, b_from + 32);
          } else {
            for (int c = 0; c < mine; ++c) copy16(b_to + ask_at + (c >> 1) * 128 + (c & 1 ? b_swap : 0u), b_from + 32 * c);
          }
        } else {
          const uint16_t* from = p.B + ((size_t)(rank ? tile.adapter : 0) * p.N + min(ask_n + b_row, p.N - 1)) * p.R + b_chunk * 8;
          for (int c = 0; c < mine; ++c) copy16(b_to + ask_at + (c >> 1) * 128 + (c & 1 ? b_swap : 0u), from + 32 * c);
        }
        b_from += (size_t)kCols * p.R;
        if (p.base && (kPlace == kAlike || m0 < tile.rows)) {
          const uint32_t to = base_to + ask_at;
          if (kPlace == kAlike) {
#pragma unroll
            for (int j = 0; j < 5; ++j) {
              const int c = b_chunk + 4 * j, n = ask_n + 4 * c - shift;
              if (c >= chunks) break;
              if (n >= 0 && n + 4 <= p.N) {
                copy16(to + j * 64, line_from + n);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (n + k >= 0 && n + k < p.N) copy4(to + j * 64 + k * 4, line_from + n + k);
              }
            }
          } else if (kVec && ask_n + kCols <= p.N) {
            copy16(to, from0);
            copy16(to + kThreads * 16, from1);
            if (!narrow) {
              copy16(to + 2 * kThreads * 16, from0 + 16);
              copy16(to + 3 * kThreads * 16, from1 + 16);
            }
          } else {
            const int n = ask_n + half + out0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (n + out_of(k) < p.N) {
                copy4(to + k * 4, from0 + out_of(k));
                copy4(to + kThreads * 16 + k * 4, from1 + out_of(k));
              }
              if (!narrow && n + 16 + out_of(k) < p.N) {
                copy4(to + 2 * kThreads * 16 + k * 4, from0 + 16 + out_of(k));
                copy4(to + 3 * kThreads * 16 + k * 4, from1 + 16 + out_of(k));
              }
            }
          }
          from0 += kCols;
          from1 += kCols;
        }
        ask_n += kCols;
        ask_at += plan.stage2;
        if (ask_at == stages_end) ask_at = 0;
      }
      copies_begun();
    };
    // ---- u's pieces, then the first stages
    if (rank) {
      const unsigned char* from = scratch + plan.at_pieces + (size_t)index * plan.pieces;
      // (of each piece's sixteen rows what the rank fills)
      if (kRegs || rank + 16 > ld) {
        for (uint32_t k = tid * 16; k < plan.pieces; k += kThreads * 16) copy16(smem_at + k, from + k);
      } else {
        for (uint32_t k = tid * 16; k < plan.pieces; k += kThreads * 16)
          if (k % (ld * 32u) < rank * 32u) copy16(smem_at + k, from + k);
      }
      copies_begun();
    }
    for (int i = 0; i < plan.stages2 - 1; ++i) ask();
    float f0 = 0.0f, f1 = 0.0f;
    if (rank) {
      const float* factors = reinterpret_cast<const float*>(scratch + plan.at_factors) + (size_t)index * kRows + m0 + g;
      f0 = factors[0];
      f1 = factors[8];
      copies_there(plan.stages2 - 1);
      __syncthreads();
      if (kRegs) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (32 * j < ld)
#pragma unroll
            for (int k = 0; k < kPieces<kBf16>; ++k) {
              held[kRegs ? j : 0][k][0] = of_u(k, 2 * j);
              held[kRegs ? j : 0][k][1] = of_u(k, 2 * j + 1);
            }
      }
    }

    // ---- outputs
    const unsigned char *here = smem + plan.pieces, *stage = here;
    int at0 = 0, at1 = 0;  // (kAlike: where this lane's first outputs of rows g and g + 8 are in a stage)
    if (kPlace == kAlike) {
      const int r0 = m0 + g, r1 = m0 + g + 8;
      at0 = r0 * kPitch + half + out0 + shift_of(p.C + (size_t)(tile.row + r0) * p.ldc);
      at1 = r1 * kPitch + half + out0 + shift_of(p.C + (size_t)(tile.row + r1) * p.ldc);
    }
    float *c0 = p.C + row * p.ldc + step0 * kCols + half + out0, *c1 = c0 + 8 * (size_t)p.ldc;
    int n = step0 * kCols + half + out0;
    for (int i = 0; i < steps; ++i, n += kCols, c0 += kCols, c1 += kCols) {
      copies_there(plan.stages2 - 2);
      __syncthreads();  // this stage has arrived for everybody, and everybody has done with the one before
      if (kPlace == kAlike && i) store(stage, n - kCols - half - out0);
      stage = here;
      ask();
      const uint16_t* b = reinterpret_cast<const uint16_t*>(here) + (half + col) * ld + t * 8;
      const float4* old = reinterpret_cast<const float4*>(here + kCols * ld * 2) + tid;
      here += plan.stage2;
      if (here == smem + plan.pieces + stages_end) here = smem + plan.pieces;
      if (m0 >= tile.rows) continue;
      auto outputs = [&](auto sixteens) {
        constexpr int kH = decltype(sixteens)::value;
        float d[kH][2][4] = {};
        // chunks of 32 ranks of B's rows: sixteen outputs h, instruction q
        auto of_b = [&](int h, int q, int chunk) { return b + (16 * h + col_step * q) * ld + (chunk ^ swap) * 8; };
        if (kRegs) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (32 * j + 32 <= rank) {
#pragma unroll
              for (int h = 0; h < kH; ++h)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  const uint4 v = *reinterpret_cast<const uint4*>(of_b(h, q, 4 * j));
#pragma unroll
                  for (int k = 0; k < kPieces<kBf16>; ++k) mma32<kBf16>(d[h][q], held[kRegs ? j : 0][k][0], held[kRegs ? j : 0][k][1], v);
                }
            }
          }
        }
        int j = kRegs ? rank & ~31 : 0;
        if (!kRegs)
          for (; j + 32 <= rank; j += 32) {
            uint4 v[kH][2];
#pragma unroll
            for (int h = 0; h < kH; ++h)
#pragma unroll
              for (int q = 0; q < 2; ++q) v[h][q] = *reinterpret_cast<const uint4*>(of_b(h, q, j / 8));
#pragma unroll
            for (int k = 0; k < kPieces<kBf16>; ++k) {
              const uint4 r0 = of_u(k, j / 16), r1 = of_u(k, j / 16 + 1);
#pragma unroll
              for (int h = 0; h < kH; ++h)
#pragma unroll
                for (int q = 0; q < 2; ++q) mma32<kBf16>(d[h][q], r0, r1, v[h][q]);
            }
          }
        if (j < rank) {  // sixteen more: a lane has four of them, in chunk t / 2 of the two
          const int at = (j / 8 ^ swap) * 8 + 4 * t - 8 * t;
#pragma unroll
          for (int k = 0; k < kPieces<kBf16>; ++k) {
            const uint4 r = of_u(k, j / 16);
#pragma unroll
            for (int h = 0; h < kH; ++h)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const uint2 v = *reinterpret_cast<const uint2*>(b + (16 * h + col_step * q) * ld + at);
                mma<kBf16>(d[h][q], r.x, r.y, r.z, r.w, v.x, v.y);
              }
          }
        }
#pragma unroll
        for (int h = 0; h < kH; ++h) {
          float4 o0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o1 = o0;
          float *s0 = nullptr, *s1 = nullptr;
          if (kPlace == kAlike) {
            float* line = const_cast<float*>(reinterpret_cast<const float*>(stage + kCols * ld * 2)) + 16 * h;
            s0 = line + at0;
            s1 = line + at1;
            if (p.base) {
              o0 = make_float4(s0[out_of(0)], s0[out_of(1)], s0[out_of(2)], s0[out_of(3)]);
              o1 = make_float4(s1[out_of(0)], s1[out_of(1)], s1[out_of(2)], s1[out_of(3)]);
            }
          } else if (p.base) {
            o0 = old[2 * h * kThreads];
            o1 = old[(2 * h + 1) * kThreads];
          }
          if (rank) {
            o0 = make_float4(fmaf(f0, d[h][0][0], o0.x), fmaf(f0, d[h][0][1], o0.y), fmaf(f0, d[h][1][0], o0.z), fmaf(f0, d[h][1][1], o0.w));
            o1 = make_float4(fmaf(f1, d[h][0][2], o1.x), fmaf(f1, d[h][0][3], o1.y), fmaf(f1, d[h][1][2], o1.z), fmaf(f1, d[h][1][3], o1.w));
          }
          if (kPlace == kAlike) {
            const float v0[4] = {o0.x, o0.y, o0.z, o0.w}, v1[4] = {o1.x, o1.y, o1.z, o1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              s0[out_of(k)] = v0[k];
              s1[out_of(k)] = v1[k];
            }
          } else if (kVec && n - half - out0 + kCols <= p.N) {
            if (has0) *reinterpret_cast<float4*>(c0 + 16 * h) = o0;
            if (has1) *reinterpret_cast<float4*>(c1 + 16 * h) = o1;
          } else {
            const float v0[4] = {o0.x, o0.y, o0.z, o0.w}, v1[4] = {o1.x, o1.y, o1.z, o1.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (n + 16 * h + out_of(k) < p.N) {
                if (has0) c0[16 * h + out_of(k)] = v0[k];
                if (has1) c1[16 * h + out_of(k)] = v1[k];
              }
          }
        }
      };
      if (narrow) outputs(std::integral_constant<int, 1>());
      else outputs(std::integral_constant<int, 2>());
    }
    copies_there<0>();
    if (kPlace == kAlike) {
      __syncthreads();
      store(stage, n - kCols - half - out0);
    }
  }
}

constexpr int kMaxInner = 200 << 10;
// The host knows how many rows and segments there are, not which segments are long or empty.  Where they are unlike the form that the average picks costs: 64 rows
// of one request, 5120 -> 5120 at rank 64, 12 us alone and 20 beside 63 empty segments (as 64 single rows); 450 rows 19 alone and 54 with 63 single rows beside them.
bool few_rows(int T, int n_seg) { return T <= 8 * (int64_t)n_seg; }

}  // namespace

extern "C" size_t izb_lora_scratch(int dtype, int R, int T, int n_seg) {
  if (T < 1 || n_seg < 1 || R < 16 || R > kMaxRank || few_rows(T, n_seg)) return 0;
  const size_t tiles = (size_t)T / kRows + n_seg;
  return RowsPlan(R, dtype == IZB_BF16, tiles).scratch(tiles);
}

extern "C" int izb_lora_add(int dtype, const void* d_A, const void* d_B, int n_adapters, int R, const int32_t* d_ranks, const float* d_scales, int N, int K,
                            const int8_t* d_aq, const float* d_asc, int T, int Mp, const int32_t* d_seg, const int32_t* d_adapter, int n_seg,
                            const float* d_base, int ldb, float* d_C, int ldc, int c_off, void* d_scratch, void* stream) {
  if (!d_A || !d_B || !d_scales || !d_aq || !d_asc || !d_seg || !d_adapter || !d_C) IZB_FAIL(IZB_ERR_ARG, "lora_add: null pointer");
  if (dtype != IZB_F16 && dtype != IZB_BF16) IZB_FAIL(IZB_ERR_TYPE, "lora_add: adapters of type %d are not taken (IZB_F16, IZB_BF16)", dtype);
  if (n_adapters < 1 || R < 16 || R > kMaxRank || R % 16) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: %d adapters of rank %d (16..%d, a multiple of 16: pad with zeros)", n_adapters, R, kMaxRank);
  if (N < 1 || N > 1 << 28 || K < 256 || K > 1 << 28 || K % 256) IZB_FAIL(IZB_ERR_SHAPE, "lora_add: N=%d K=%d (K a multiple of 256, both 2^28 at most)", N, K);
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
  const bool bf16 = dtype == IZB_BF16, few = few_rows(T, n_seg), one = T <= n_seg;
  const int64_t tiles = (int64_t)T / (one ? 1 : few ? kFewRows : kRows) + n_seg;  // (at most)
  const int sms = izb_sm_count(device);
  // CTAs per tile.  Single rows: as many as leave all of them room at once (64 requests of 17408 x 5120, 4 / 5 / 6 / 8 CTAs: 34.7 / 31.8 / 29.0 / 32.5 us), 4 at
  // least and 16 at most.  Few rows: 16 while that leaves the multiprocessors two CTAs at most, else 8.  More rows: as many as fit at once, 16 at most, where
  // cuts of segments that are no multiple of 64 rows leave half a tile each (8 at most and a tile each before: 451 rows of 14592, rank 128, 50 us against 33; 2210
  // rows of 16128 in 46 segments, rank 16, 77 against 51).
  const int widest = R <= 128 ? 16 : 8;
  if (one) p.cluster = kFewBlocks<1> * sms / T > widest ? widest : kFewBlocks<1> * sms / T < 4 ? 4 : kFewBlocks<1> * sms / T;
  else p.cluster = few && n_seg * 16ll <= 2 * sms ? widest : 8;
  if (!few)
    for (p.cluster = widest; p.cluster > 1 && (T / kRows + (n_seg + 1ll) / 2) * p.cluster > 2 * sms;) p.cluster /= 2;
  if (tiles * p.cluster > 0x7FFFFFFF) IZB_FAIL(IZB_ERR_LIMIT, "lora_add: %d rows in %d segments", T, n_seg);
  const dim3 grid((unsigned)(tiles * p.cluster));
  if (few) {
    static izb_device_once once[4];
    void (*const kernels[4])(LoraArgs) = {lora_few_kernel<false, kFewRows>, lora_few_kernel<true, kFewRows>, lora_few_kernel<false, 1>, lora_few_kernel<true, 1>};
    const int which = (one ? 2 : 0) + bf16;
    if (int rc = once[which].run(device, [&]() -> int {
          IZB_CUDA(cudaFuncSetAttribute(kernels[which], cudaFuncAttributeMaxDynamicSharedMemorySize, 200 << 10));
          IZB_CUDA(cudaFuncSetAttribute(kernels[which], cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
          return IZB_OK;
        }))
      return rc;
    const size_t smem = one ? few_smem<1>(R, p.cluster) : few_smem<kFewRows>(R, p.cluster);
    IZB_LAUNCH("lora_add", st, izb_launch_pdl_cluster(kernels[which], p.cluster, grid, kThreads, smem, st, p));
    return IZB_OK;
  }
  if (!d_scratch || !izb_aligned(d_scratch, 16)) IZB_FAIL(IZB_ERR_ARG, "lora_add: %d rows in %d segments want %zu bytes of scratch, 16-byte aligned", T, n_seg, izb_lora_scratch(dtype, R, T, n_seg));
  if (RowsPlan(R, bf16, tiles).scratch(tiles) > 0xFFFFFFFFu) IZB_FAIL(IZB_ERR_LIMIT, "lora_add: %d rows in %d segments of rank %d", T, n_seg, R);
  const bool vec = izb_aligned(p.C, 16) && ldc % 4 == 0 && (!d_base || (izb_aligned(d_base, 16) && ldb % 4 == 0));
  const int place = vec ? kOnLines : !d_base || (((uintptr_t)p.C - (uintptr_t)d_base) % 16 == 0 && (ldc - (int64_t)ldb) % 4 == 0) ? kAlike : kAnywhere;
  const RowsPlan plan(R, bf16, tiles, place);
  static izb_device_once once[18];
  void (*const inners[6])(LoraArgs, RowsPlan, unsigned char*) = {lora_inner_kernel<false, 1>, lora_inner_kernel<false, 2>, lora_inner_kernel<false, 4>,
                                                                 lora_inner_kernel<true, 1>, lora_inner_kernel<true, 2>, lora_inner_kernel<true, 4>};
  const int which_inner = (bf16 ? 3 : 0) + plan.parts / 2;
  auto inner = inners[which_inner];
  void (*const outers[12])(LoraArgs, RowsPlan, const unsigned char*) = {
      lora_outer_kernel<false, kOnLines, false>, lora_outer_kernel<false, kOnLines, true>, lora_outer_kernel<false, kAlike, false>, lora_outer_kernel<false, kAlike, true>,
      lora_outer_kernel<false, kAnywhere, false>, lora_outer_kernel<false, kAnywhere, true>, lora_outer_kernel<true, kOnLines, false>, lora_outer_kernel<true, kOnLines, true>,
      lora_outer_kernel<true, kAlike, false>, lora_outer_kernel<true, kAlike, true>, lora_outer_kernel<true, kAnywhere, false>, lora_outer_kernel<true, kAnywhere, true>};
  const int which = (bf16 ? 6 : 0) + 2 * place + (R <= 64 ? 1 : 0);
  if (int rc = once[which].run(device, [&]() -> int {
        IZB_CUDA(cudaFuncSetAttribute(outers[which], cudaFuncAttributeMaxDynamicSharedMemorySize, RowsPlan::kMost2));
        return IZB_OK;
      }))
    return rc;
  if (int rc = once[12 + which_inner].run(device, [&]() -> int {
        IZB_CUDA(cudaFuncSetAttribute(inner, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxInner));
        IZB_CUDA(cudaFuncSetAttribute(inner, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        return IZB_OK;
      }))
    return rc;
  IZB_LAUNCH("lora_inner", st, izb_launch_pdl_cluster(inner, p.cluster, grid, kThreads, plan.total1, st, p, plan, (unsigned char*)d_scratch));
  // (two CTAs per multiprocessor; no more than there is work at most)
  const int64_t steps = tiles * ((N + kCols - 1) / kCols), outer_grid = steps < 2 * sms ? steps : 2 * sms;
  IZB_LAUNCH("lora_outer", st, izb_launch_pdl(outers[which], dim3((unsigned)outer_grid), kThreads, plan.total2, st, p, plan, (const unsigned char*)d_scratch));
  return IZB_OK;
}
