// The whole mixture-of-experts block of a few tokens (a decode step's) in two kernels: routing, gate and up projections with SwiGLU, then the
// down projection with the weighted sum over a token's experts, the shared expert's output and the residual.
//   e_k, w_k as izb_moe_route;  g = x Wg_e^T, u = x Wu_e^T;  h = u * g / (1 + exp(-g));  out = x + sum_k w_k h_k Wd_e^T + sgate * sh
// The six-call path quantises h to int8 in between; here a block of 32 values of h is 23-bit integers Q times a power of two, in three int8 digits
// (Q = 65536 d1 + 256 d2 + d3), so that the down projection runs on the same integer matrix instruction and h is off by 2^-22 of its block's largest value.
//
// Bound by the bytes of the experts that the tokens reach, each read once.  Both kernels work on 16 weight rows x one superblock per warp, straight
// from global memory into the instruction's registers (lane g = lane / 4, t = lane % 4 holds bytes 8t .. 8t+7 of each block of rows g and g + 8).
// Most experts have one or two tokens, for which an instruction with a token per column is mostly empty and a lane repeats a row's scales for all of
// its blocks.  So the columns are the eight blocks of the superblock instead: the B operand of block b's instruction has the token's values in
// column b and zeros beside them, eight instructions add up to the 16 x 8 block sums, and lane t scales blocks 2t and 2t + 1 of its two rows -- each
// scale is decoded by one lane, once.  What comes after is a sum over the quad.
//
// Routing is done by every CTA for itself (a warp per token, a microsecond less than a launch).  The first kernel lets the second one in behind its own
// wait for the kernel before: what was written before this call is then visible to the second kernel from its start, and it routes and asks for its first
// weights while the first kernel still runs.
#include "izb_common.cuh"

namespace {

constexpr int kMaxTokens = 32, kMaxPairs = 512, kMaxExperts = 512, kMaxChoices = 32;
constexpr int kUpWarps = 8, kSplitK = 4;  // first kernel: two groups of 16 channels x four parts of K
constexpr int kDownWarps = 16;
constexpr uint32_t kMagic = 0x4B400000u;  // 1.5 * 2^23: accumulators start there and are f32 numbers as they are (|sum| < 2^22)

struct MoeArgs {
  const uint8_t *wg, *wu, *wd;
  const int8_t* aq;
  const float *asc, *logits, *x, *sh;
  int8_t* hq;         // [T * NU][3][F]
  float *hs, *hsum;   // [T * NU][F / 32]: the power of two, the sum of the block's values
  float* out;
  int T, Mp, ldl, NE, NU, e0, n_mats, E, F, joined, splits;
  size_t gate_row, down_row;  // bytes of a row
};

// ---------------------------------------------------------------------------------------------- routing
struct Routed {
  float wt[kMaxPairs];
  short id[kMaxPairs];           // the expert's number in the stacks, -1: not here
  uint32_t tokens[kMaxExperts];  // of an expert
  short list[kMaxExperts];       // experts with tokens, in increasing order
  int count[17];
};
// One warp: a token's choices in order, ties to the lower id (see izb_moe.cu); the weights' sum in choice order.
template <int kPer>
__device__ __forceinline__ void route_token(const MoeArgs& p, int token, Routed& s) {
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
  float top = 0.0f, denom = 0.0f, mine = 0.0f;
  int id = 0;
  for (int k = 0; k < p.NU; ++k) {
    const uint32_t win = __reduce_max_sync(0xFFFFFFFFu, best);
    const int e = (int)__reduce_min_sync(0xFFFFFFFFu, best == win ? (uint32_t)(at * 32 + lane) : 0xFFFFu);
    if ((e & 31) == lane) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i == (e >> 5)) key[i] = 0u;
      rescan();
    }
    const float l = __uint_as_float((win & 0x80000000u) ? (win & 0x7FFFFFFFu) : ~win);
    if (k == 0) top = l;
    const float q = expf(l - top);
    denom += q;
    if (lane == k) { mine = q; id = e; }
  }
  if (lane < p.NU) {
    const int e = id - p.e0;
    const bool here = e >= 0 && e < p.n_mats;
    s.id[token * p.NU + lane] = (short)(here ? e : -1);
    s.wt[token * p.NU + lane] = __fdiv_rn(mine, denom);
    if (here) atomicOr(&s.tokens[e], 1u << token);
  }
}
// All tokens; the number of experts that have any.  Every thread of the CTA calls it.
__device__ int route_all(const MoeArgs& p, Routed& s) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kMaxExperts; i += blockDim.x) s.tokens[i] = 0u;
  __syncthreads();
  for (int t = warp; t < p.T; t += warps) {
    if (p.NE <= 128) route_token<4>(p, t, s);
    else route_token<kMaxExperts / 32>(p, t, s);
  }
  __syncthreads();
  const int groups = (p.n_mats + 31) / 32;  // of 32 experts
  for (int i = warp; i < groups; i += warps) {
    const uint32_t has = __ballot_sync(0xFFFFFFFFu, s.tokens[i * 32 + lane] != 0u);
    if (lane == 0) s.count[i] = __popc(has);
  }
  __syncthreads();
  int n = 0;
  for (int i = 0; i < groups; ++i) {
    if ((i % warps) == warp) {
      const bool has = s.tokens[i * 32 + lane] != 0u;
      const uint32_t all = __ballot_sync(0xFFFFFFFFu, has);
      if (has) s.list[n + __popc(all & ((1u << lane) - 1u))] = (short)(i * 32 + lane);
    }
    n += s.count[i];
  }
  __syncthreads();
  return n;
}
// which of its choices expert `e` is for `token`, as a pair number
__device__ __forceinline__ int pair_of(const MoeArgs& p, const Routed& s, int token, int e) {
  const int lane = threadIdx.x & 31;
  return token * p.NU + __ffs(__ballot_sync(0xFFFFFFFFu, lane < p.NU && s.id[token * p.NU + min(lane, p.NU - 1)] == e)) - 1;
}

// ---------------------------------------------------------------------------------------------- 16 rows x one superblock
__device__ __forceinline__ uint2 ldg_stream_v2(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
template <bool kUnsigned>
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kUnsigned)
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
struct Scales {  // of rows g, g + 8 and blocks 2t, 2t + 1
  float s[2][2], m[2][2];
};
template <int QT>
struct Raw;
template <>
struct Raw<IZB_Q4_K> {
  static constexpr int kBytes = 144;
  static constexpr bool kMin = true;
  uint2 q[2][4];
  uint4 h[2];
  __device__ __forceinline__ void load(const uint8_t* r0, const uint8_t* r1, int t) {
    h[0] = ldg_stream_v4(r0);
    h[1] = ldg_stream_v4(r1);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      q[0][c] = ldg_stream_v2(r0 + 16 + 32 * c + 8 * t);
      q[1][c] = ldg_stream_v2(r1 + 16 + 32 * c + 8 * t);
    }
  }
  // high nibbles are multiplied where they are, as 16 q: their scale is a 16th
  __device__ __forceinline__ void dots(int (&d)[4], uint2 x, int g) const {
    d[0] = d[1] = d[2] = d[3] = (int)kMagic;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint2 u = q[0][b >> 1], v = q[1][b >> 1];
      const uint32_t m = b & 1 ? 0xF0F0F0F0u : 0x0F0F0F0Fu;
      mma<true>(d, u.x & m, v.x & m, u.y & m, v.y & m, g == b ? x.x : 0u, g == b ? x.y : 0u);
    }
  }
  __device__ __forceinline__ void scales(Scales& o, int t) const {
    const int sh = 16 * (t & 1);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint32_t a = h[r].y >> sh, b = h[r].z >> sh, c = h[r].w >> sh;  // two blocks side by side
      const uint32_t sc = t < 2 ? a & 0x3F3Fu : (c & 0x0F0Fu) | ((a >> 2) & 0x3030u), mn = t < 2 ? b & 0x3F3Fu : ((c >> 4) & 0x0F0Fu) | ((b >> 2) & 0x3030u);
      const float d = half_bits_to_float(h[r].x & 0xFFFFu), dm = half_bits_to_float(h[r].x >> 16);
      o.s[r][0] = d * (float)(sc & 0xFFu);
      o.s[r][1] = d * 0.0625f * (float)(sc >> 8);
      o.m[r][0] = dm * (float)(mn & 0xFFu);
      o.m[r][1] = dm * (float)(mn >> 8);
    }
  }
};
template <>
struct Raw<IZB_Q8_0> {
  static constexpr int kBytes = 272;
  static constexpr bool kMin = false;
  uint2 q[2][8];
  uint32_t h[2];
  __device__ __forceinline__ void load(const uint8_t* r0, const uint8_t* r1, int t) {
    h[0] = __ldg(reinterpret_cast<const uint32_t*>(r0) + t);
    h[1] = __ldg(reinterpret_cast<const uint32_t*>(r1) + t);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      q[0][c] = ldg_stream_v2(r0 + 16 + 32 * c + 8 * t);
      q[1][c] = ldg_stream_v2(r1 + 16 + 32 * c + 8 * t);
    }
  }
  __device__ __forceinline__ void dots(int (&d)[4], uint2 x, int g) const {
    d[0] = d[1] = d[2] = d[3] = (int)kMagic;
#pragma unroll
    for (int b = 0; b < 8; ++b) mma<false>(d, q[0][b].x, q[1][b].x, q[0][b].y, q[1][b].y, g == b ? x.x : 0u, g == b ? x.y : 0u);
  }
  __device__ __forceinline__ void scales(Scales& o, int) const {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      o.s[r][0] = half_bits_to_float(h[r] & 0xFFFFu);
      o.s[r][1] = half_bits_to_float(h[r] >> 16);
    }
  }
};
__device__ __forceinline__ float number(int d) { return __int_as_float(d) - __uint_as_float(kMagic); }

// ---------------------------------------------------------------------------------------------- gate, up, SwiGLU
// A CTA takes 32 channels of one expert at a time (one block of h); a warp 16 of them, gate and up, for every fourth superblock.
template <int QT>
__global__ void __launch_bounds__(kUpWarps * 32, 2) moe_layer_up_kernel(MoeArgs p) {
  __shared__ Routed s;
  __shared__ float s_sum[kUpWarps][kMaxTokens][32];  // [..][gate row, up row of the warp]
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, half = warp / kSplitK, part = warp % kSplitK;
  pdl_wait();
  pdl_launch_next();
  const int n_exp = route_all(p, s), per = p.F / 32, sbs = p.E / 256;
  for (int unit = blockIdx.x; unit < n_exp * per; unit += gridDim.x) {
    const int e = s.list[unit / per], f0 = unit % per * 32;
    const uint32_t tokens = s.tokens[e];
    const size_t first = (size_t)e * p.F * (p.joined ? 2 : 1) + (p.joined ? 2 * f0 : f0) + 16 * half + g;
    const uint8_t* rg = p.wg + first * p.gate_row;
    const uint8_t* ru = p.joined ? rg + 32 * p.gate_row : p.wu + first * p.gate_row;
    for (int sb = part; sb < sbs; sb += kSplitK) {
      Raw<QT> wg, wu;
      const size_t at = (size_t)sb * Raw<QT>::kBytes;
      wg.load(rg + at, rg + 8 * p.gate_row + at, t);
      wu.load(ru + at, ru + 8 * p.gate_row + at, t);
      uint32_t left = tokens;
      auto values = [&](int token) { return *reinterpret_cast<const uint2*>(p.aq + (size_t)token * p.E + sb * 256 + g * 32 + 8 * t); };
      auto scale = [&](int token, int i) { return p.asc[(size_t)(sb * 8 + 2 * t + i) * p.Mp + token]; };
      int token = __ffs(left) - 1;
      uint2 x = values(token);
      float xs[2] = {scale(token, 0), scale(token, 1)};
      Scales cg, cu;
      wg.scales(cg, t);
      wu.scales(cu, t);
      for (int slot = 0; left; ++slot) {
        left &= left - 1;
        const uint2 x_now = x;
        const float s0 = xs[0], s1 = xs[1];
        if (left) {
          token = __ffs(left) - 1;
          x = values(token);
          xs[0] = scale(token, 0);
          xs[1] = scale(token, 1);
        }
        int dg[4], du[4];
        wg.dots(dg, x_now, g);
        wu.dots(du, x_now, g);
        float v[4];  // gate row g, g + 8, up row g, g + 8
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          v[r] = fmaf(number(dg[2 * r]) * cg.s[r][0], s0, number(dg[2 * r + 1]) * cg.s[r][1] * s1);
          v[2 + r] = fmaf(number(du[2 * r]) * cu.s[r][0], s0, number(du[2 * r + 1]) * cu.s[r][1] * s1);
        }
        if (Raw<QT>::kMin) {
          int sum = __dp4a((int)x_now.x, 0x01010101, __dp4a((int)x_now.y, 0x01010101, 0));  // of block g
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
          sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
          const float x0 = (float)__shfl_sync(0xFFFFFFFFu, sum, 8 * t) * s0, x1 = (float)__shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4) * s1;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            v[r] = fmaf(-cg.m[r][0], x0, fmaf(-cg.m[r][1], x1, v[r]));
            v[2 + r] = fmaf(-cu.m[r][0], x0, fmaf(-cu.m[r][1], x1, v[2 + r]));
          }
        }
        // the quad's sums: lane t keeps v[t]
        const bool odd = t & 1, high = t & 2;
        const float a = (odd ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? v[0] : v[1], 1);
        const float b = (odd ? v[3] : v[2]) + __shfl_xor_sync(0xFFFFFFFFu, odd ? v[2] : v[3], 1);
        const float c = (high ? b : a) + __shfl_xor_sync(0xFFFFFFFFu, high ? a : b, 2);
        float* to = &s_sum[warp][slot][(t >> 1) * 16 + (t & 1) * 8 + g];
        *to = sb == part ? c : *to + c;
      }
    }
    __syncthreads();
    // a warp per token: channel f0 + lane
    const int n_tok = __popc(tokens), live = min(kSplitK, sbs);
    for (int slot = warp; slot < n_tok; slot += kUpWarps) {
      uint32_t left = tokens;
      for (int i = 0; i < slot; ++i) left &= left - 1;
      const int pair = pair_of(p, s, __ffs(left) - 1, e);
      float gate = 0.0f, up = 0.0f;
      for (int k = 0; k < live; ++k) {
        const float* from = s_sum[(lane >> 4) * kSplitK + k][slot];
        gate += from[lane & 15];
        up += from[16 + (lane & 15)];
      }
      const float h = gate / (1.0f + expf(-gate)) * up;
      const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(h) & 0x7FFFFFFFu);  // (a NaN is above all numbers here)
      const int ex = max((int)(most >> 23), 1) - 127;                                           // |h| < 2^(ex + 1)
      const bool none = most >= 0x7F800000u;
      const int up1 = min(21 - ex, 100);
      const int Q = none ? 0 : __float2int_rn(h * __int_as_float((up1 + 127) << 23) * __int_as_float((21 - ex - up1 + 127) << 23));
      const int d3 = (int8_t)Q, q1 = (Q - d3) >> 8, d2 = (int8_t)q1, d1 = (q1 - d2) >> 8;
      int8_t* hq = p.hq + (size_t)pair * 3 * p.F + f0 + lane;
      hq[0] = (int8_t)d1;
      hq[p.F] = (int8_t)d2;
      hq[2 * p.F] = (int8_t)d3;
      const int sum = __reduce_add_sync(0xFFFFFFFFu, Q);
      if (lane == 0) {
        const float unit_of = none ? __int_as_float(0x7FC00000) : ldexpf(1.0f, ex - 21);
        p.hs[(size_t)pair * per + f0 / 32] = unit_of;
        p.hsum[(size_t)pair * per + f0 / 32] = unit_of * (float)sum;
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------- down, combine
// A CTA takes 16 outputs of all tokens; its warps the experts, each in `splits` parts of F (by F alone, so that a token's sums do not depend on
// which others the call has).
template <int QT>
__global__ void __launch_bounds__(kDownWarps * 32, 1) moe_layer_down_kernel(MoeArgs p) {
  extern __shared__ float s_y[];  // [T * NU][splits][16]
  __shared__ Routed s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3;
  pdl_launch_next();
  const int n_exp = route_all(p, s), sbs = p.F / 256, per = p.F / 32, items = n_exp * p.splits;
  bool waited = false;
  for (int n0 = blockIdx.x * 16; n0 < p.E; n0 += gridDim.x * 16) {
    Raw<QT> w, next;
    int item = warp, sb = 0, end = 0;
    const uint8_t* row = nullptr;
    auto open = [&]() {  // the item's first superblock and rows
      if (item >= items) return;
      const int k = item % p.splits;
      sb = sbs * k / p.splits;
      end = sbs * (k + 1) / p.splits;
      row = p.wd + ((size_t)s.list[item / p.splits] * p.E + n0 + g) * p.down_row;
    };
    auto fetch = [&](Raw<QT>& to) { to.load(row + (size_t)sb * Raw<QT>::kBytes, row + 8 * p.down_row + (size_t)sb * Raw<QT>::kBytes, t); };
    open();
    if (item < items) fetch(w);
    if (!waited) {
      pdl_wait();
      waited = true;
    }
    while (item < items) {
      const int e = s.list[item / p.splits], k = item % p.splits, now = sb, start = sbs * k / p.splits;
      uint32_t left = s.tokens[e];
      if (++sb == end) {
        item += warps;
        open();
      }
      if (item < items) fetch(next);
      int pair = pair_of(p, s, __ffs(left) - 1, e);
      uint2 x[3];
      float2 hs, hm;
      auto values = [&]() {
#pragma unroll
        for (int d = 0; d < 3; ++d) x[d] = *reinterpret_cast<const uint2*>(p.hq + ((size_t)pair * 3 + d) * p.F + now * 256 + g * 32 + 8 * t);
        hs = *reinterpret_cast<const float2*>(p.hs + (size_t)pair * per + now * 8 + 2 * t);
        if (Raw<QT>::kMin) hm = *reinterpret_cast<const float2*>(p.hsum + (size_t)pair * per + now * 8 + 2 * t);
      };
      values();
      Scales c;
      w.scales(c, t);
      while (left) {
        left &= left - 1;
        int d1[4], d2[4], d3[4];
        w.dots(d1, x[0], g);
        w.dots(d2, x[1], g);
        w.dots(d3, x[2], g);
        const float2 hs_now = hs, hm_now = hm;
        const int pair_now = pair;
        if (left) {
          pair = pair_of(p, s, __ffs(left) - 1, e);
          values();
        }
        float v[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float q[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) q[i] = fmaf(number(d1[2 * r + i]), 65536.0f, fmaf(number(d2[2 * r + i]), 256.0f, number(d3[2 * r + i]))) * c.s[r][i];
          v[r] = fmaf(q[0], hs_now.x, q[1] * hs_now.y);
          if (Raw<QT>::kMin) v[r] = fmaf(-c.m[r][0], hm_now.x, fmaf(-c.m[r][1], hm_now.y, v[r]));
        }
        float a = (t & 1 ? v[1] : v[0]) + __shfl_xor_sync(0xFFFFFFFFu, t & 1 ? v[0] : v[1], 1);
        a += __shfl_xor_sync(0xFFFFFFFFu, a, 2);
        if (t < 2) {
          float* to = s_y + ((size_t)pair_now * p.splits + k) * 16 + t * 8 + g;
          *to = now == start ? a : *to + a;
        }
      }
      w = next;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.T * 16; i += blockDim.x) {
      const int token = i >> 4, n = n0 + (i & 15);
      float v = 0.0f;
      for (int k = 0; k < p.NU; ++k) {
        const int pair = token * p.NU + k;
        if (s.id[pair] < 0) continue;
        float y = s_y[(size_t)pair * p.splits * 16 + (i & 15)];
        for (int j = 1; j < p.splits; ++j) y += s_y[((size_t)pair * p.splits + j) * 16 + (i & 15)];
        v = fmaf(s.wt[pair], y, v);
      }
      const size_t at = (size_t)token * p.E + n;
      if (p.sh) v = fmaf(p.sh[at], 1.0f / (1.0f + expf(-p.logits[(size_t)token * p.ldl + p.NE])), v);
      p.out[at] = p.x ? p.x[at] + v : v;
    }
    __syncthreads();
  }
  if (!waited) pdl_wait();
}

bool takes(const izb_weight* w) { return w->type == IZB_Q4_K || w->type == IZB_Q8_0; }

}  // namespace

extern "C" size_t izb_moe_layer_scratch(int T, int NU, int F) {
  // three digits of every value of h, a scale and a sum per 32 of them
  return T < 1 || NU < 1 || F < 1 ? 0 : (size_t)T * NU * ((size_t)F * 3 + (size_t)F / 32 * 8);
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
  if (T > kMaxTokens || T * NU > kMaxPairs)
    IZB_FAIL(IZB_ERR_LIMIT, "moe_layer: %d tokens x %d experts (up to %d tokens and %d pairs: izb_moe_route, _sort, _gateup, _down and _combine take more)", T, NU, kMaxTokens, kMaxPairs);
  if (!d_scratch) IZB_FAIL(IZB_ERR_ARG, "moe_layer: no scratch");
  if (e0 < 0 || e0 + wg->n_mats > NE) IZB_FAIL(IZB_ERR_SHAPE, "moe_layer: experts [%d, %d) of %d", e0, e0 + wg->n_mats, NE);
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
  p.out = d_out;
  p.T = T; p.Mp = Mp; p.ldl = ldl; p.NE = NE; p.NU = NU; p.e0 = e0; p.n_mats = wg->n_mats; p.E = E; p.F = F;
  p.joined = wg->gu32; p.gate_row = wg->row_bytes; p.down_row = wd->row_bytes;
  p.splits = F >= 512 ? 2 : 1;
  const int sms = izb_sm_count(wg->device), units = (int)(pairs < (size_t)wg->n_mats ? pairs : wg->n_mats) * (F / 32);
  const int up_grid = units < 2 * sms ? units : 2 * sms;
  // the second kernel: a CTA of 16 warps per multiprocessor, or two of 8 where one round of the former does not do
  const int tiles = E / 16, down_warps = tiles <= sms ? kDownWarps : kDownWarps / 2, most = tiles <= sms ? sms : 2 * sms;
  const int down_grid = tiles < most ? tiles : most;
  const size_t smem = pairs * p.splits * 16 * sizeof(float);
  cudaStream_t st = (cudaStream_t)stream;
  auto up = wg->type == IZB_Q4_K ? moe_layer_up_kernel<IZB_Q4_K> : moe_layer_up_kernel<IZB_Q8_0>;
  auto down = wd->type == IZB_Q4_K ? moe_layer_down_kernel<IZB_Q4_K> : moe_layer_down_kernel<IZB_Q8_0>;
  constexpr size_t kMaxSmem = (size_t)kMaxPairs * 2 * 16 * sizeof(float);
  IZB_SMEM_OPTIN(moe_layer_down_kernel<IZB_Q4_K>, kMaxSmem, wd->device);
  IZB_SMEM_OPTIN(moe_layer_down_kernel<IZB_Q8_0>, kMaxSmem, wd->device);
  IZB_LAUNCH("moe_layer_up", st, izb_launch_pdl(up, up_grid, kUpWarps * 32, 0, st, p));
  IZB_LAUNCH("moe_layer_down", st, izb_launch_pdl(down, down_grid, down_warps * 32, smem, st, p));
  return IZB_OK;
}
