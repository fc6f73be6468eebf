// The whole mixture-of-experts block of a few tokens (a decode step's) in two kernels: routing, gate and up projections with SwiGLU, then the
// down projection with the weighted sum over a token's experts, the shared expert's output and the residual.
//   e_k, w_k as izb_moe_route;  g = x Wg_e^T, u = x Wu_e^T;  h = u * g / (1 + exp(-g));  out = x + sum_k w_k h_k Wd_e^T + sgate * sh
// The six-call path quantises h to int8 in between; here a block of 32 values of h is integers Q times a power of two, in three int8 digits
// (Q = 65536 d1 + 256 d2 + d3, |Q| <= 8355711), so that the down projection runs on the same integer matrix instruction and h is off by 2^-23 of its block's
// largest value, half a unit: about what a single f32 operation is off by.
//
// Bound by the bytes of the experts that the tokens reach, each read once.  Both kernels work on 16 weight rows x one superblock per warp (lane
// g = lane / 4, t = lane % 4 holds bytes 8t .. 8t+7 of each block of rows g and g + 8).  A warp has a ring of such pieces of its own in shared memory,
// filled by 16-byte asynchronous copies, and asks for the next piece as soon as it has one in registers, across the borders of experts and channels.
// Most experts have one or two tokens, for which an instruction with a token per column is mostly empty and a lane repeats a row's scales for all of
// its blocks.  So the columns are the eight blocks of the superblock instead: the B operand of block b's instruction has the token's values in
// column b and zeros beside them, eight instructions add up to the 16 x 8 block sums, and lane t scales blocks 2t and 2t + 1 of its two rows -- each
// scale is decoded by one lane, once.  What comes after is a sum over the quad.
//
// Routing is done by every CTA of the first kernel for itself (a warp per token; 2.6 us, with what follows from it, against a launch and its hand-over); one of
// them writes it out for the second kernel, which reads it behind its wait for the first one: what kernels before this call wrote is visible to it from
// there on only.
//
// Measured (us; the six calls / this; the floor by bytes), 128 experts of 768 over 2048, top 8, Q4_K: one token 26 / 16 (3.3), four 48 / 36, eight 88 / 57 (21),
// 16 156 / 91, 32 211 / 150 (45); 60 experts of 1280 over 4096, top 4, five tokens 100 / 58.  Many tokens per expert are where the block-per-column form has nothing
// to gain (it costs every token eight instructions): 8 experts, top 2, 32 tokens 47 / 57.  One token is latency: routing 2.6 us, first bytes of weights 2.4 in each kernel,
// barriers.  Eight tokens: the first kernel's loop runs at 4.1 TB/s, the second one's at 2.9, both near 48 % of the issue slots with 16 warps per multiprocessor:
// a superblock of gate and up takes about 560 instructions, of which decoding 6-bit scales is a fifth; the rest of the time is fixed latencies that 16 warps do
// not cover.  The first kernel's 128 registers leave 12 (Q4_K) and 20 bytes (Q8_0) of a thread in local memory.
// (Taken back: 24 warps per multiprocessor with gate and up one after the other and 80 registers, 55 -> 82 us; calling the routing and the epilogues once on
// zeros so that their code is in the cache, 18 -> 23; the first kernel's CTAs asking L2 for the second one's first pieces as they end, one token 17.1 -> 17.6, others 0 to 4 %
// slower.)
#include "izb_common.cuh"

namespace {

constexpr int kMaxTokens = 32, kMaxPairs = 512, kMaxExperts = 512, kMaxChoices = 32;
constexpr int kUpWarps = 8, kSplitK = 4;   // first kernel: two groups of 16 channels x four parts of K
constexpr int kDownWarps = 16;
constexpr int kGroup = 8;                  // tokens of an expert that are dealt with in one go
constexpr uint32_t kMagic = 0x4B400000u;  // 1.5 * 2^23: accumulators start there and are f32 numbers as they are (|sum| < 2^22)

struct MoeArgs {
  const uint8_t *wg, *wu, *wd;
  const int8_t* aq;
  const float *asc, *logits, *x, *sh;
  int8_t* hq;         // [T * NU][3][F]
  float *hs, *hsum;   // [T * NU][F / 32]: the power of two, the sum of the block's values
  uint32_t* routes;   // the routing, as write_routes leaves it
  float* out;
  int T, Mp, ldl, NE, NU, e0, n_mats, E, F, joined, splits, cluster;
  size_t gate_row, down_row;  // bytes of a row
};

// ---------------------------------------------------------------------------------------------- routing
struct Routed {
  float wt[kMaxPairs];
  short id[kMaxPairs];           // the expert's number in the stacks, -1: not here
  short list[kMaxPairs];         // experts with tokens, in increasing order, once per kGroup of them ...
  uint32_t group[kMaxPairs];     // ... and which those are
};
struct Routing : Routed {
  uint32_t tokens[kMaxExperts];  // of an expert
  int count[16];
};
// One warp: a token's choices in order, ties to the lower id (see izb_moe.cu); the weights' sum in choice order.
template <int kPer>
__device__ __forceinline__ void route_token(const MoeArgs& p, int token, Routing& s) {
  const int lane = threadIdx.x & 31;
  const float* row = p.logits + (size_t)token * p.ldl;
  uint32_t key[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    key[i] = 0u;
    if (i * 32 + lane < p.NE) {
      uint32_t u = __float_as_uint(__fadd_rn(row[i * 32 + lane], 0.0f));
      u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
      key[i] = u ? u : 1u;
    }
  }
  uint32_t best = 0u;
  int at = 0;
  auto rescan = [&]() {
    best = key[0];
    at = 0;
#pragma unroll
    for (int i = 1; i < kPer; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
  };
  rescan();
  uint32_t mine_key = 0u;
  int id = 0;
  for (int k = 0; k < p.NU; ++k) {
    const uint32_t win = __reduce_max_sync(0xFFFFFFFFu, best);
    const uint32_t who = __ballot_sync(0xFFFFFFFFu, best == win);
    // (one lane as a rule: the minimum over ids is only looked for where several hold the same logit)
    const int e = who & (who - 1) ? (int)__reduce_min_sync(0xFFFFFFFFu, best == win ? (uint32_t)(at * 32 + lane) : 0xFFFFu)
                                  : __shfl_sync(0xFFFFFFFFu, at * 32 + lane, __ffs(who) - 1);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i * 32 + lane == e) key[i] = 0u;
    if ((e & 31) == lane) rescan();
    if (lane == k) { mine_key = win; id = e; }
  }
  // p_k = exp(l_k - l_0), their sum in choice order
  const float l = __uint_as_float((mine_key & 0x80000000u) ? (mine_key & 0x7FFFFFFFu) : ~mine_key);
  const float mine = expf(l - __shfl_sync(0xFFFFFFFFu, l, 0));
  float denom = 0.0f;
  for (int k = 0; k < p.NU; ++k) denom += __shfl_sync(0xFFFFFFFFu, mine, k);
  if (lane < p.NU) {
    const int e = id - p.e0;
    const bool here = e >= 0 && e < p.n_mats;
    s.id[token * p.NU + lane] = (short)(here ? e : -1);
    s.wt[token * p.NU + lane] = __fdiv_rn(mine, denom);
    if (here) atomicOr(&s.tokens[e], 1u << token);
  }
}
// All tokens; the length of the list.  Every thread of the CTA calls it.
__device__ __forceinline__ int route_all(const MoeArgs& p, Routing& s) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kMaxExperts; i += blockDim.x) s.tokens[i] = 0u;
  __syncthreads();
  for (int t = warp; t < p.T; t += warps) {
    if (p.NE <= 128) route_token<4>(p, t, s);
    else route_token<kMaxExperts / 32>(p, t, s);
  }
  __syncthreads();
  const int blocks = (p.n_mats + 31) / 32;  // of 32 experts
  for (int i = warp; i < blocks; i += warps) {
    const int n = __reduce_add_sync(0xFFFFFFFFu, (__popc(s.tokens[i * 32 + lane]) + kGroup - 1) / kGroup);
    if (lane == 0) s.count[i] = n;
  }
  __syncthreads();
  int n = 0;
  for (int i = 0; i < blocks; ++i) {
    if (i % warps == warp) {
      uint32_t left = s.tokens[i * 32 + lane];
      const int mine = (__popc(left) + kGroup - 1) / kGroup;
      int before = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, before, o);
        if (lane >= o) before += v;
      }
      for (int j = n + before - mine; left; ++j) {
        uint32_t rest = left;
        for (int k = 0; k < kGroup; ++k) rest &= rest - 1;  // (0 stays 0)
        s.list[j] = (short)(i * 32 + lane);
        s.group[j] = left & ~rest;
        left = rest;
      }
    }
    n += s.count[i];
  }
  __syncthreads();
  return n;
}
// The routing of T * NU pairs in memory: the length of the list (and three words of nothing) | weights | experts | the list | its tokens.
__device__ __forceinline__ void write_routes(const MoeArgs& p, const Routed& s, int entries) {
  const int pairs = p.T * p.NU;
  if (threadIdx.x == 0) p.routes[0] = (uint32_t)entries;
  uint32_t* to = p.routes + 4;
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
    to[i] = __float_as_uint(s.wt[i]);
    to[pairs + i] = (uint32_t)s.id[i];
    if (i < entries) {
      to[2 * pairs + i] = (uint32_t)s.list[i];
      to[3 * pairs + i] = s.group[i];
    }
  }
}
// Every thread of the CTA calls it; the length of the list.
__device__ __forceinline__ int read_routes(const MoeArgs& p, Routed& s) {
  const int pairs = p.T * p.NU, entries = (int)p.routes[0];
  const uint32_t* from = p.routes + 4;
  for (int i = threadIdx.x; i < pairs; i += blockDim.x) {  // (behind the list's end: what is there, unused)
    const uint32_t wt = from[i], id = from[pairs + i], list = from[2 * pairs + i], group = from[3 * pairs + i];
    s.wt[i] = __uint_as_float(wt);
    s.id[i] = (short)id;
    s.list[i] = (short)list;
    s.group[i] = group;
  }
  __syncthreads();
  return entries;
}
// which of its choices expert `e` is for `token`, as a pair number
__device__ __forceinline__ int pair_of(const MoeArgs& p, const Routed& s, int token, int e) {
  const int lane = threadIdx.x & 31;
  return token * p.NU + __ffs(__ballot_sync(0xFFFFFFFFu, lane < p.NU && s.id[token * p.NU + min(lane, p.NU - 1)] == e)) - 1;
}

// ---------------------------------------------------------------------------------------------- 16 rows x one superblock
template <bool kUnsigned>
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kUnsigned)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// f32 pairs (blocks 2t and 2t + 1): two IEEE operations per instruction
typedef unsigned long long f2;
__device__ __forceinline__ f2 f2_of(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 f2_parts(f2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ f2 f2_add(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 f2_mul(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 f2_fma(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// two accumulators as the numbers they are
__device__ __forceinline__ f2 numbers(int a, int b) {
  return f2_add(f2_of(__int_as_float(a), __int_as_float(b)), f2_of(-__uint_as_float(kMagic), -__uint_as_float(kMagic)));
}
struct Scales {  // of rows g, g + 8 for blocks 2t, 2t + 1; mins with their sign changed
  f2 s[2], m[2];
};
template <int QT>
struct Raw;
template <>
struct Raw<IZB_Q4_K> {
  static constexpr int kBytes = 144, kPitch = 160;  // (40 words: four rows x eight words are on different banks)
  static constexpr bool kMin = true;
  uint2 q[2][4];
  uint4 h[2];
  __device__ __forceinline__ void load(const unsigned char* tile, int g, int t) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const unsigned char* row = tile + (g + 8 * r) * kPitch;
      h[r] = *reinterpret_cast<const uint4*>(row);
#pragma unroll
      for (int c = 0; c < 4; ++c) q[r][c] = *reinterpret_cast<const uint2*>(row + 16 + 32 * c + 8 * t);
    }
  }
  // block b's rows; high nibbles are multiplied where they are, as 16 q: their scale is a 16th
  __device__ __forceinline__ uint4 block(int b) const {
    const uint2 u = q[0][b >> 1], v = q[1][b >> 1];
    const uint32_t m = b & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
    return make_uint4(u.x & m, v.x & m, u.y & m, v.y & m);
  }
  __device__ __forceinline__ void scales(Scales& o, int t) const {
    const int sh = 16 * (t & 1);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t a = h[r].y >> sh, b = h[r].z >> sh, c = h[r].w >> sh;  // two blocks side by side
      const uint32_t sc = t < 2 ? a & 0x3F3Fu : (c & 0x0F0Fu) | ((a >> 2) & 0x3030u), mn = t < 2 ? b & 0x3F3Fu : ((c >> 4) & 0x0F0Fu) | ((b >> 2) & 0x3030u);
      // (a byte under the exponent of 2^23 is the number 2^23 + byte, and d * that - d * 2^23 is rounded once: no conversions)
      const float d = half_bits_to_float(h[r].x & 0xFFFFu), dm = -half_bits_to_float(h[r].x >> 16);
      const f2 dd = f2_of(d, d * 0.0625f), mm = f2_of(dm, dm), big = f2_of(-8388608.0f, -8388608.0f);
      o.s[r] = f2_fma(dd, f2_of(__uint_as_float(__byte_perm(sc, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(sc, 0x4B000000u, 0x7441))), f2_mul(dd, big));
      o.m[r] = f2_fma(mm, f2_of(__uint_as_float(__byte_perm(mn, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(mn, 0x4B000000u, 0x7441))), f2_mul(mm, big));
    }
  }
};
template <>
struct Raw<IZB_Q8_0> {
  static constexpr int kBytes = 272, kPitch = 288;
  static constexpr bool kMin = false;
  uint2 q[2][8];
  uint32_t h[2];
  __device__ __forceinline__ void load(const unsigned char* tile, int g, int t) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const unsigned char* row = tile + (g + 8 * r) * kPitch;
      h[r] = *reinterpret_cast<const uint32_t*>(row + 4 * t);
#pragma unroll
      for (int c = 0; c < 8; ++c) q[r][c] = *reinterpret_cast<const uint2*>(row + 16 + 32 * c + 8 * t);
    }
  }
  __device__ __forceinline__ uint4 block(int b) const { return make_uint4(q[0][b].x, q[1][b].x, q[0][b].y, q[1][b].y); }
  __device__ __forceinline__ void scales(Scales& o, int) const {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      o.s[r] = f2_of(half_bits_to_float(h[r] & 0xFFFFu), half_bits_to_float(h[r] >> 16));
    }
  }
};
// The sums of 16 rows x 8 blocks: kW pieces of weights against kX rows of values (one of the two is 1).  A block's operands are made once for all of them.
template <int kW, int kX, int QT>
__device__ __forceinline__ void dots(int (&d)[kW * kX][4], const Raw<QT>* const (&w)[kW], const uint2 (&x)[kX], int g) {
#pragma unroll
  for (int i = 0; i < kW * kX; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = (int)kMagic;
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    uint2 v[kX];
#pragma unroll
    for (int i = 0; i < kX; ++i) v[i] = make_uint2(g == b ? x[i].x : 0u, g == b ? x[i].y : 0u);
#pragma unroll
    for (int j = 0; j < kW; ++j) {
      const uint4 a = w[j]->block(b);
#pragma unroll
      for (int i = 0; i < kX; ++i) mma<Raw<QT>::kMin>(d[j * kX + i], a.x, a.y, a.z, a.w, v[i].x, v[i].y);
    }
  }
}

// A warp's copies of pieces into its ring.
template <int QT>
struct Copier {
  static constexpr int kRowChunks = Raw<QT>::kBytes / 16, kChunks = 16 * kRowChunks, kPer = (kChunks + 31) / 32, kTile = 16 * Raw<QT>::kPitch;
  uint32_t from[kPer], to[kPer];
  __device__ __forceinline__ Copier(size_t row_bytes, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int c = min(lane + 32 * i, kChunks - 1), row = c / kRowChunks, at = 16 * (c % kRowChunks);
      from[i] = (uint32_t)(row * row_bytes) + at;
      to[i] = row * Raw<QT>::kPitch + at;
    }
  }
  __device__ __forceinline__ void tile(uint32_t slot, const uint8_t* src, int lane) const {  // 16 rows from `src` on
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (32 * (i + 1) <= kChunks || lane + 32 * i < kChunks)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + to[i]), "l"(src + from[i]) : "memory");
  }
};
__device__ __forceinline__ void copies_begun() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the last kLater groups have arrived, for every lane of the warp
template <int kLater>
__device__ __forceinline__ void copies_there() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLater) : "memory");
  __syncwarp();
}

// ---------------------------------------------------------------------------------------------- gate, up, SwiGLU
// A CTA takes 32 channels of one expert at a time (one block of h); a warp 16 of them, gate and up, for every fourth superblock.
template <int QT>
struct Up {
  static constexpr int kSlots = QT == IZB_Q4_K ? 2 : 1, kSlot = 2 * Copier<QT>::kTile;
  static constexpr size_t kSums = 2 * kUpWarps * kGroup * 32 * sizeof(float), kSmem = kSums + (size_t)kUpWarps * kSlots * kSlot;
};
// The sums of a unit: a warp per token, channel f0 + lane.
__device__ __forceinline__ void up_epilogue(const MoeArgs& p, const Routed& s, const float (*sums)[kGroup][32], int entry, int f0, uint32_t tokens) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = p.F / 32, live = min(kSplitK, p.E / 256);
  for (int i = 0; i < warp; ++i) tokens &= tokens - 1;
  const int pair = pair_of(p, s, __ffs(tokens) - 1, s.list[entry]);
  float gate = 0.0f, up = 0.0f;
#pragma unroll
  for (int k = 0; k < kSplitK; ++k) {
    if (k >= live) break;
    const float* from = sums[(lane >> 4) * kSplitK + k][warp];
    gate += from[lane & 15];
    up += from[16 + (lane & 15)];
  }
  const float h = gate / (1.0f + expf(-gate)) * up;
  const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(h) & 0x7FFFFFFFu);  // (a NaN is above all numbers here)
  const int ex = max((int)(most >> 23), 1) - 127;                                           // |h| < 2^(ex + 1)
  const bool none = most >= 0x7F800000u;
  // a unit of 2^(ex - 22), or twice that where the largest value would need more than three digits hold: M / 2 (M its 24 bits, 2^23 .. 2^24) rounded is above 127 * 65793
  const int bits = (most & 0x7FFFFFu) <= 0x7EFEFEu ? 22 : 21, up1 = min(bits - ex, 100);
  const int Q = none ? 0 : __float2int_rn(h * __int_as_float((up1 + 127) << 23) * __int_as_float((bits - ex - up1 + 127) << 23));
  const int d3 = (int8_t)Q, q1 = (Q - d3) >> 8, d2 = (int8_t)q1, d1 = (q1 - d2) >> 8;
  const int sum = __reduce_add_sync(0xFFFFFFFFu, Q);
  int8_t* hq = p.hq + (size_t)pair * 3 * p.F + f0 + lane;
  hq[0] = (int8_t)d1;
  hq[p.F] = (int8_t)d2;
  hq[2 * p.F] = (int8_t)d3;
  if (lane == 0) {
    const float unit_of = none ? __int_as_float(0x7FC00000) : ldexpf(1.0f, ex - bits);
    p.hs[(size_t)pair * per + f0 / 32] = unit_of;
    p.hsum[(size_t)pair * per + f0 / 32] = unit_of * (float)sum;
  }
}
template <int QT>
__global__ void __launch_bounds__(kUpWarps * 32, 2) moe_layer_up_kernel(MoeArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Routing s;
  constexpr int kSlots = Up<QT>::kSlots, kSlot = Up<QT>::kSlot;
  auto s_sum = reinterpret_cast<float(*)[kUpWarps][kGroup][32]>(smem);  // [two units][..][..][gate row, up row of the warp]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, half = warp / kSplitK, part = warp % kSplitK;
  unsigned char* ring = smem + Up<QT>::kSums + (size_t)warp * kSlots * kSlot;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const Copier<QT> copier(p.gate_row, lane);
  pdl_wait();
  pdl_launch_next();
  const int sbs = p.E / 256, entries = route_all(p, s);
  if (blockIdx.x == 0) write_routes(p, s, entries);

  // A unit is an entry of the list and a block of 32 channels; a CTA takes every gridDim.x-th.
  struct Unit {
    int entry, f0;
  };
  auto next = [&](Unit& u, int by) {
    u.f0 += 32 * by;
    while (u.f0 >= p.F) {
      u.f0 -= p.F;
      ++u.entry;
    }
  };
  Unit asked = {0, 0};  // what is asked for next
  next(asked, blockIdx.x);
  Unit unit = asked;
  int ask_sb = part, ask_slot = 0;
  const uint8_t *ask_g = nullptr, *ask_u = nullptr;
  const size_t expert_rows = (size_t)p.F * (p.joined ? 2 : 1);
  auto open = [&]() {
    if (asked.entry >= entries) return;
    const size_t first = s.list[asked.entry] * expert_rows + (p.joined ? 2 * asked.f0 : asked.f0) + 16 * half;
    ask_g = p.wg + first * p.gate_row + part * Raw<QT>::kBytes;
    ask_u = p.joined ? ask_g + 32 * p.gate_row : p.wu + first * p.gate_row + part * Raw<QT>::kBytes;
  };
  auto ask = [&]() {
    if (asked.entry < entries) {
      copier.tile(ring_at + ask_slot * kSlot, ask_g, lane);
      copier.tile(ring_at + ask_slot * kSlot + Copier<QT>::kTile, ask_u, lane);
      ask_g += kSplitK * Raw<QT>::kBytes;
      ask_u += kSplitK * Raw<QT>::kBytes;
      ask_sb += kSplitK;
      if (ask_sb >= sbs) {
        ask_sb = part;
        next(asked, gridDim.x);
        open();
      }
    }
    copies_begun();
    ask_slot = ask_slot + 1 == kSlots ? 0 : ask_slot + 1;
  };
  if (part >= sbs) asked.entry = entries;  // (a short K: nothing for this warp)
  open();
#pragma unroll
  for (int i = 0; i < kSlots; ++i) ask();

  for (int buf = 0, slot = 0; unit.entry < entries; next(unit, gridDim.x), buf ^= 1) {
    const uint32_t tokens = s.group[unit.entry];
    for (int sb = part; sb < sbs; sb += kSplitK) {
      const int8_t* aq = p.aq + (sb * 256 + g * 32 + 8 * t);
      const float* asc = p.asc + (size_t)(sb * 8 + 2 * t) * p.Mp;
      auto values = [&](int token) { return *reinterpret_cast<const uint2*>(aq + token * p.E); };  // (32 rows of at most 2^24 values)
      auto scale = [&](int token, int i) { return asc[i * p.Mp + token]; };
      uint32_t left = tokens;
      int token = __ffs(left) - 1;
      uint2 x = values(token);
      float xs[2] = {scale(token, 0), scale(token, 1)};
      Raw<QT> wg, wu;
      copies_there<kSlots - 1>();
      wg.load(ring + slot * kSlot, g, t);
      wu.load(ring + slot * kSlot + Copier<QT>::kTile, g, t);
      slot = slot + 1 == kSlots ? 0 : slot + 1;
      __syncwarp();  // (all lanes have theirs before the slot is filled again)
      ask();
      Scales cg, cu;
      wg.scales(cg, t);
      wu.scales(cu, t);
      for (int i = 0; left; ++i) {
        left &= left - 1;
        const uint2 x_now = x;
        const float s0 = xs[0], s1 = xs[1];
        if (left) {
          token = __ffs(left) - 1;
          x = values(token);
          xs[0] = scale(token, 0);
          xs[1] = scale(token, 1);
        }
        int d[2][4];
        const Raw<QT>* const both_weights[2] = {&wg, &wu};
        const uint2 values_now[1] = {x_now};
        dots(d, both_weights, values_now, g);
        const f2 ss = f2_of(s0, s1);
        f2 sums = 0;
        if (Raw<QT>::kMin) {
          int sum = __dp4a((int)x_now.x, 0x01010101, __dp4a((int)x_now.y, 0x01010101, 0));  // of block g
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
          sums = f2_mul(f2_of((float)__shfl_sync(0xFFFFFFFFu, sum, 8 * t), (float)__shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4)), ss);
        }
        float v[4];  // gate row g, g + 8, up row g, g + 8
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const Scales& c = r < 2 ? cg : cu;
          f2 q = f2_mul(f2_mul(numbers(d[r >> 1][2 * (r & 1)], d[r >> 1][2 * (r & 1) + 1]), c.s[r & 1]), ss);
          if (Raw<QT>::kMin) q = f2_fma(c.m[r & 1], sums, q);
          const float2 both = f2_parts(q);
          v[r] = both.x + both.y;
        }
        // the quad's sums: lane t keeps v[t]
        const bool odd = t & 1, high = t & 2;
        const float a = (odd ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? v[0] : v[1], 1);
        const float b = (odd ? v[3] : v[2]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2] : v[3], 1);
        const float c = (high ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, high ? a : b, 2);
        float* to = &s_sum[buf][warp][i][(t >> 1) * 16 + (t & 1) * 8 + g];
        *to = sb == part ? c : *to + c;
      }
    }
    // One barrier per unit: the sums of the unit before last have been read before a warp comes to the barrier of the last one.
    __syncthreads();
    if (warp < __popc(tokens)) up_epilogue(p, s, s_sum[buf], unit.entry, unit.f0, tokens);
  }
}

// ---------------------------------------------------------------------------------------------- down, combine
// A CTA takes 16 outputs of all tokens; its warps the experts, each in `splits` parts of F (by F alone, so that a token's sums do not depend on
// which others the call has).  Where there are few outputs a cluster of CTAs takes 16 of them, each its share of the experts: their sums go to the first
// one's shared memory, the last step of each straight from registers (us
// without / with: 25 tokens, 512 outputs, F 768, 6 experts, top 5 59 / 46; 31 tokens, 768 outputs, F 512, 19 experts, top 6 53 / 45).
template <int QT>
struct Down {
  static constexpr int kSlots = QT == IZB_Q4_K ? 3 : 2, kSlot = Copier<QT>::kTile;
  static size_t smem(int warps, size_t pairs, int splits) { return pairs * splits * 16 * sizeof(float) + (size_t)warps * kSlots * kSlot; }
};
// 16 outputs of all tokens.  `base`: what a thread adds in its first output of the CTA's first 16, asked for ahead.
__device__ __forceinline__ void down_combine(const MoeArgs& p, const Routed& s, const float* s_y, int n0, bool ahead, float base) {
  const int splits_log = p.splits - 1;
  for (int i = threadIdx.x; i < p.T * 16; i += blockDim.x) {
    const int token = i >> 4, at = token * p.E + n0 + (i & 15), pr0 = token * p.NU;
    if (p.x && (!ahead || i >= (int)blockDim.x)) base = p.x[at];
    float v = 0.0f;
#pragma unroll 4
    for (int k = 0; k < p.NU; ++k) {
      const float* y = s_y + ((pr0 + k) << splits_log) * 16 + (i & 15);
      const float sum = splits_log ? y[0] + y[16] : y[0], next = fmaf(s.wt[pr0 + k], sum, v);
      if (s.id[pr0 + k] >= 0) v = next;
    }
    if (p.sh) v = fmaf(p.sh[at], 1.0f / (1.0f + expf(-p.logits[(size_t)token * p.ldl + p.NE])), v);
    p.out[at] = p.x ? base + v : v;
  }
}
template <int QT, bool kCluster>
__global__ void __launch_bounds__(kDownWarps * 32, 1) moe_layer_down_kernel(MoeArgs p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Routed s;
  constexpr int kSlots = Down<QT>::kSlots, kSlot = Down<QT>::kSlot;
  float* s_y = reinterpret_cast<float*>(smem);  // [T * NU][splits][16]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* ring = smem + (size_t)p.T * p.NU * p.splits * 16 * sizeof(float) + (size_t)warp * kSlots * kSlot;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const Copier<QT> copier(p.down_row, lane);
  pdl_launch_next();
  int rank = 0, tile0 = blockIdx.x, tiles = gridDim.x;
  if (kCluster) asm("mov.u32 %0, %%cluster_ctarank;\n\tmov.u32 %1, %%clusterid.x;\n\tmov.u32 %2, %%nclusterid.x;" : "=r"(rank), "=r"(tile0), "=r"(tiles));
  tile0 *= 16;
  tiles *= 16;
  const int cluster = kCluster ? p.cluster : 1, stride = warps * cluster;
  if (kCluster) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // (waited for before anything is written to another CTA)
  const int splits_log = p.splits - 1, stride_log = __ffs(stride) - 1, sbs = p.F / 256, per = p.F / 32;  // (one or two splits)
  pdl_wait();
  const int items = read_routes(p, s) << splits_log;

  // what the combine adds to
  float base = 0.0f;
  if (p.x) base = p.x[min((int)threadIdx.x >> 4, p.T - 1) * p.E + tile0 + (threadIdx.x & 15)];

  // A place in a warp's work: 16 outputs, an item (an expert's tokens and a part of F: parts of unlike lengths go round among the warps), a superblock.
  struct Place {
    int n0, item, sb, end, k;
  };
  auto open = [&](Place& w) {
    while (w.item >= items && w.n0 < p.E) {
      w.n0 += tiles;
      w.item = warp * cluster + rank;
      if (w.item >= items) w.n0 = p.E;  // (fewer items than warps)
    }
    w.k = (w.item + (w.item >> stride_log)) & splits_log;
    w.sb = w.k ? sbs >> 1 : 0;
    w.end = w.k || !splits_log ? sbs : sbs >> 1;
  };
  auto step = [&](Place& w) {
    if (++w.sb == w.end) {
      w.item += stride;
      open(w);
    }
  };
  Place asked = {tile0, warp * cluster + rank, 0, 0, 0};
  if (asked.item >= items) asked.n0 = p.E;
  open(asked);
  Place now = asked;
  int ask_slot = 0;
  auto ask = [&]() {
    if (asked.n0 < p.E) {
      copier.tile(ring_at + ask_slot * kSlot, p.wd + ((size_t)s.list[asked.item >> splits_log] * p.E + asked.n0) * p.down_row + (size_t)asked.sb * Raw<QT>::kBytes, lane);
      step(asked);
    }
    copies_begun();
    ask_slot = ask_slot + 1 == kSlots ? 0 : ask_slot + 1;
  };
#pragma unroll
  for (int i = 0; i < kSlots; ++i) ask();
  if (kCluster) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");

  uint2 x[3];
  f2 hs, hm;
  int pair = 0;
  auto values = [&](const Place& w, int token) {
    pair = pair_of(p, s, token, s.list[w.item >> splits_log]);
    const int8_t* hq = p.hq + (pair * 3 * p.F + w.sb * 256) + (g * 32 + 8 * t);  // (512 pairs of at most 2^20 values)
    x[0] = *reinterpret_cast<const uint2*>(hq);
    x[1] = *reinterpret_cast<const uint2*>(hq + p.F);
    x[2] = *reinterpret_cast<const uint2*>(hq + 2 * p.F);
    const int at = pair * per + w.sb * 8 + 2 * t;
    hs = *reinterpret_cast<const f2*>(p.hs + at);
    if (Raw<QT>::kMin) hm = *reinterpret_cast<const f2*>(p.hsum + at);
  };
  if (now.n0 < p.E) values(now, __ffs(s.group[now.item >> splits_log]) - 1);
  for (int n0 = tile0, slot = 0; n0 < p.E; n0 += tiles) {
    while (now.n0 == n0) {
      const Place here = now;
      step(now);
      Raw<QT> w;
      copies_there<kSlots - 1>();
      w.load(ring + slot * kSlot, g, t);
      slot = slot + 1 == kSlots ? 0 : slot + 1;
      __syncwarp();
      ask();
      Scales c;
      w.scales(c, t);
      uint32_t left = s.group[here.item >> splits_log];
      const bool first = here.sb == (here.k ? sbs >> 1 : 0);
      while (left) {
        left &= left - 1;
        int d[3][4];
        const Raw<QT>* const weights[1] = {&w};
        dots(d, weights, x, g);
        const f2 hs_now = hs, hm_now = hm;
        const int pair_now = pair;
        if (left) values(here, __ffs(left) - 1);
        else if (now.n0 < p.E) values(now, __ffs(s.group[now.item >> splits_log]) - 1);
        float v[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          f2 q = f2_fma(numbers(d[1][2 * r], d[1][2 * r + 1]), f2_of(256.0f, 256.0f), numbers(d[2][2 * r], d[2][2 * r + 1]));
          q = f2_fma(numbers(d[0][2 * r], d[0][2 * r + 1]), f2_of(65536.0f, 65536.0f), q);
          q = f2_mul(f2_mul(q, c.s[r]), hs_now);
          if (Raw<QT>::kMin) q = f2_fma(c.m[r], hm_now, q);
          const float2 both = f2_parts(q);
          v[r] = both.x + both.y;
        }
        float a = (t & 1 ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, t & 1 ? v[0] : v[1], 1);
        a += __shfl_xor_sync(0xFFFFFFFFu, a, 2);
        if (t < 2) {
          float* to = s_y + ((pair_now << splits_log) + here.k) * 16 + t * 8 + g;
          if (!first) a += *to;
          if (kCluster && here.sb + 1 == here.end) {
            uint32_t there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(to)));
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(a) : "memory");
          } else {
            *to = a;
          }
        }
      }
    }
    if (kCluster) {  // (of one round)
      asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
      if (rank) break;
    } else {
      __syncthreads();
    }
    down_combine(p, s, s_y, n0, n0 == tile0, base);
    __syncthreads();
  }
}

bool takes(const izb_weight* w) { return w->type == IZB_Q4_K || w->type == IZB_Q8_0; }

}  // namespace

extern "C" size_t izb_moe_layer_scratch(int T, int NU, int F) {
  // three digits of every value of h, a scale and a sum per 32 of them; the routing
  return T < 1 || NU < 1 || F < 1 ? 0 : (size_t)T * NU * ((size_t)F * 3 + (size_t)F / 32 * 8 + 16) + 16;
}

extern "C" int izb_moe_layer(const izb_weight* wg, const izb_weight* wu, const izb_weight* wd, const int8_t* d_aq, const float* d_asc, int T, int Mp,
                             const float* d_logits, int ldl, int NE, int NU, int e0, const float* d_sh, const float* d_x, float* d_out, void* d_scratch,
                             void* stream) {
  if (!wg || !wd || !d_aq || !d_asc || !d_logits || !d_out) IZB_FAIL(IZB_ERR_ARG, "moe_layer: null pointer");
  if (!wu && !wg->gu32) IZB_FAIL(IZB_ERR_ARG, "moe_layer: no up projection (wu = NULL is for a stack of izb_weight_create_gateup)");
  if (wu && wg->gu32) IZB_FAIL(IZB_ERR_ARG, "moe_layer: an interleaved gate | up stack and an up projection beside it");
  if (!takes(wg) || (wu && !takes(wu)) || !takes(wd)) IZB_FAIL(IZB_ERR_TYPE, "moe_layer: expert stacks of Q4_K, Q8_0 and Q4_0 are taken");
  const int F = wg->gu32 ? wg->N / 2 : wg->N, E = wg->K;
  if (wu && (wu->type != wg->type || wu->N != wg->N || wu->K != wg->K || wu->n_mats != wg->n_mats || wu->gu32)) IZB_FAIL(IZB_ERR_SHAPE, "moe_layer: gate and up stacks differ");
  if (wd->gu32 || wd->N != E || wd->K != F || wd->n_mats != wg->n_mats)
    IZB_FAIL(IZB_ERR_SHAPE, "moe_layer: a down stack of %d x [%d, %d] for %d experts of %d channels over %d", wd->n_mats, wd->N, wd->K, wg->n_mats, F, E);
  if (T < 1 || NU < 1 || NE < NU || NE > kMaxExperts || NU > kMaxChoices || Mp % 16 || Mp < T || ldl < NE + (d_sh ? 1 : 0))
    IZB_FAIL(IZB_ERR_SHAPE, "moe_layer: T=%d Mp=%d NE=%d NU=%d ldl=%d (NE <= %d, NU <= %d, ldl >= NE, + 1 with a shared expert)", T, Mp, NE, NU, ldl, kMaxExperts, kMaxChoices);
  if (E > 1 << 20 || F > 1 << 20) IZB_FAIL(IZB_ERR_LIMIT, "moe_layer: %d channels over %d (2^20 at most)", F, E);
  if (T > kMaxTokens || T * NU > kMaxPairs)
    IZB_FAIL(IZB_ERR_LIMIT, "moe_layer: %d tokens x %d experts (up to %d tokens and %d pairs: izb_moe_route, _sort, _gateup, _down and _combine take more)", T, NU, kMaxTokens, kMaxPairs);
  if (!d_scratch) IZB_FAIL(IZB_ERR_ARG, "moe_layer: no scratch");
  if (e0 < 0 || e0 > NE - wg->n_mats) IZB_FAIL(IZB_ERR_SHAPE, "moe_layer: %d experts from %d on, of %d", wg->n_mats, e0, NE);
  if (!izb_aligned(d_aq, 16) || !izb_aligned(d_scratch, 16)) IZB_FAIL(IZB_ERR_ALIGN, "moe_layer: aq and scratch must be 16-byte aligned");
  if (!izb_aligned(d_asc, 4) || !izb_aligned(d_logits, 4) || !izb_aligned(d_out, 4) || !izb_aligned(d_x, 4) || !izb_aligned(d_sh, 4))
    IZB_FAIL(IZB_ERR_ALIGN, "moe_layer: f32 pointers must be 4-byte aligned");
  if (izb_overlap_in_part(d_x, E, d_out, E, T, E) || izb_overlap_in_part(d_sh, E, d_out, E, T, E)) IZB_FAIL(IZB_ERR_ARG, "moe_layer: x or sh overlaps out in part");
  if ((wu && wu->device != wg->device) || wd->device != wg->device) IZB_FAIL(IZB_ERR_ARG, "moe_layer: the stacks live on different devices");
  if (int rc = izb_require_device(wg->device, "moe_layer")) return rc;
  MoeArgs p = {};
  p.wg = wg->raw; p.wu = wu ? wu->raw : nullptr; p.wd = wd->raw;
  p.aq = d_aq; p.asc = d_asc; p.logits = d_logits; p.x = d_x; p.sh = d_sh;
  const size_t pairs = (size_t)T * NU;
  p.hq = (int8_t*)d_scratch; p.hs = (float*)((int8_t*)d_scratch + pairs * 3 * F); p.hsum = p.hs + pairs * (F / 32);
  p.routes = (uint32_t*)(p.hsum + pairs * (F / 32));
  p.out = d_out;
  p.T = T; p.Mp = Mp; p.ldl = ldl; p.NE = NE; p.NU = NU; p.e0 = e0; p.n_mats = wg->n_mats; p.E = E; p.F = F;
  p.joined = wg->gu32; p.gate_row = wg->row_bytes; p.down_row = wd->row_bytes;
  p.splits = F >= 512 ? 2 : 1;
  const int sms = izb_sm_count(wg->device), units = (int)(pairs < (size_t)wg->n_mats ? pairs : wg->n_mats) * (F / 32);
  const int up_grid = units < 2 * sms ? units : 2 * sms;
  // the second kernel: a CTA of 16 warps per multiprocessor, or two of 8 where one round of the former does not do
  const int tiles = E / 16, down_warps = tiles <= sms ? kDownWarps : kDownWarps / 2, most = tiles <= sms ? sms : 2 * sms;
  // (a cluster per 16 outputs while there is a multiprocessor for each CTA and more items, about, than warps: with 14 of them for 32 23 us came to 27)
  const size_t groups = pairs < wg->n_mats + pairs / kGroup ? pairs : wg->n_mats + pairs / kGroup;
  p.cluster = 1;
  while (p.cluster < 8 && tiles * p.cluster * 2 <= sms && groups * p.splits > (size_t)down_warps * p.cluster) p.cluster *= 2;
  const int down_grid = tiles < most ? tiles * p.cluster : most;
  cudaStream_t st = (cudaStream_t)stream;
  const bool up4 = wg->type == IZB_Q4_K, down4 = wd->type == IZB_Q4_K;
  const size_t up_smem = up4 ? Up<IZB_Q4_K>::kSmem : Up<IZB_Q8_0>::kSmem;
  const size_t down_smem = down4 ? Down<IZB_Q4_K>::smem(down_warps, pairs, p.splits) : Down<IZB_Q8_0>::smem(down_warps, pairs, p.splits);
  IZB_SMEM_OPTIN(moe_layer_up_kernel<IZB_Q4_K>, Up<IZB_Q4_K>::kSmem, wg->device);
  IZB_SMEM_OPTIN(moe_layer_up_kernel<IZB_Q8_0>, Up<IZB_Q8_0>::kSmem, wg->device);
  IZB_SMEM_OPTIN((moe_layer_down_kernel<IZB_Q4_K, false>), Down<IZB_Q4_K>::smem(kDownWarps, kMaxPairs, 2), wg->device);
  IZB_SMEM_OPTIN((moe_layer_down_kernel<IZB_Q4_K, true>), Down<IZB_Q4_K>::smem(kDownWarps, kMaxPairs, 2), wg->device);
  IZB_SMEM_OPTIN((moe_layer_down_kernel<IZB_Q8_0, false>), Down<IZB_Q8_0>::smem(kDownWarps, kMaxPairs, 2), wg->device);
  IZB_SMEM_OPTIN((moe_layer_down_kernel<IZB_Q8_0, true>), Down<IZB_Q8_0>::smem(kDownWarps, kMaxPairs, 2), wg->device);
  auto up = up4 ? moe_layer_up_kernel<IZB_Q4_K> : moe_layer_up_kernel<IZB_Q8_0>;
  const bool shared = p.cluster > 1;
  auto down = down4 ? (shared ? moe_layer_down_kernel<IZB_Q4_K, true> : moe_layer_down_kernel<IZB_Q4_K, false>)
                    : (shared ? moe_layer_down_kernel<IZB_Q8_0, true> : moe_layer_down_kernel<IZB_Q8_0, false>);
  IZB_LAUNCH("moe_layer_up", st, izb_launch_pdl(up, up_grid, kUpWarps * 32, up_smem, st, p));
  IZB_LAUNCH("moe_layer_down", st, izb_launch_pdl_cluster(down, p.cluster, dim3(down_grid), down_warps * 32, down_smem, st, p));
  return IZB_OK;
}
