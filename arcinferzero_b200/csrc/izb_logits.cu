// The rules of each request on its row of the output head's logits: penalties for tokens that the row's history holds, a list of
// biases, a grammar mask, the temperature; and of the outcome the best token and log(sum(exp)).
//
//   c[v] = how often v stands in the row's history;  per token, in this order, each operation rounded once:
//   c > 0:          l = l > 0 ? l / repetition : l * repetition,  l = l - (frequency * c + presence)
//   v in the list:  l = l + bias
//   mask bit 0:     l = -inf
//   temperature>0:  l = l / temperature
//
// Every logit is read once and written once: bound by those bytes, and with rules on by instruction issue (256 rows of 128256: 48 to 54 us without rules for
// 40 us of bytes, 85 with all of them at 70 % of the issue slots).  A row is split over a cluster of CTAs, each with a stretch of the vocabulary, so
// that a single row has 16 multiprocessors at work; what is joined at the end is one (maximum, index, sum) per CTA, through distributed shared memory,
// in the order of the stretches.  A CTA first asks for the row's history, then for its logits (three 16-byte copies per thread in flight, into a ring; loads
// into as many registers share scoreboards and wait for one another, 84 against 67 us), then counts: one word of shared memory per token of a window of the
// stretch, the count of the history in its lower half and the number of the bias in the upper one.  Every CTA of a row reads the row's whole history, since
// most of it belongs to others: handing tokens on through distributed shared memory would save less than the cluster-wide barrier costs.  Rows with more than
// 65535 of either take two words per token and half the window at a time.
// (Taken back: a bitmap of the tokens that the rules touch, and counts for those alone, numbered by its running sum.  The pass over the others is then
// free of rules, but the steps before it wait for memory one after the other: 64 rows that stay in L2 55 us against 36.  Counts of 16 bits, two to a word, with biases
// marked and looked up in their list or in a table in shared memory: 71 and 41 against 41, 256 rows 88 against 84.  The touched tokens of a lane one by one instead of its
// four together: 93 against 85 for 256 rows, by the registers it takes.)
#include <math.h>

#include "izb_common.cuh"

namespace {

constexpr int kThreads = 512, kBatch = 3;  // groups of four tokens that a thread has in flight
constexpr int kRing = (kBatch + 1) * kThreads * 16;
constexpr int kWords = 19456;              // counting words of a CTA at most (two CTAs per multiprocessor)
constexpr int kEarly = 8;                  // history tokens that a thread keeps in registers (4096 in all; the rest is read for every window)
constexpr int kMaxCluster = 16;
constexpr float kBig = 3.4028234e38f;

struct LogitsArgs {
  const float* in;
  float* out;
  const float* params;
  const int32_t *hist, *hist_off, *bias_ids, *bias_off, *mask_row;
  const float* bias;
  const uint32_t* mask;
  int32_t* best;
  float* logz;
  int ldl, ldo, V, n_hist, n_bias, mask_words, n_masks, cluster, words;
};

// exp(d) of a difference to the maximum (d <= 0, or a NaN)
__device__ __forceinline__ float exp_of(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
  return r;
}

// l / t, correctly rounded, with y the correctly rounded 1 / t (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990: a quotient within one unit of the last place and its exactly computed remainder give the rounded one; the first step here brings it that
// near).  Where an intermediate could leave the normal range, and for zeros and what is no number, the division itself.
__device__ __forceinline__ bool plain_size(float v) { return (__float_as_uint(v) & 0x7FFFFFFFu) - (67u << 23) < (120u << 23); }  // 2^-60 .. 2^60
__device__ __forceinline__ float quotient(float l, float t, float y) {
  float q = __fmul_rn(l, y);
  q = __fmaf_rn(__fmaf_rn(-t, q, l), y, q);
  return __fmaf_rn(__fmaf_rn(-t, q, l), y, q);
}

struct Top {  // largest value, its lowest index, sum of exp(l - m); m itself may be infinite, what is subtracted is the largest finite number then
  float m, s;
  int at;
};
__device__ __forceinline__ float finite(float m) { return fminf(fmaxf(m, -kBig), kBig); }
__device__ __forceinline__ Top top_join(Top a, Top b) {
  const bool of_b = b.m > a.m || (b.m == a.m && b.at < a.at);
  const float m = of_b ? b.m : a.m;
  // (a sum whose maximum is m stays as it is: it may be infinite)
  const float s = (a.m == m ? a.s : a.s * exp_of(finite(a.m) - finite(m))) + (b.m == m ? b.s : b.s * exp_of(finite(b.m) - finite(m)));
  return {m, s, of_b ? b.at : a.at};
}

__global__ void __launch_bounds__(kThreads, 2) logits_process_kernel(LogitsArgs p) {
  extern __shared__ __align__(16) uint32_t s_word[];
  __shared__ Top s_top[kThreads / 32], s_cta[kMaxCluster];
  const int r = blockIdx.x / p.cluster, rank = blockIdx.x % p.cluster, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");  // (waited for before anything is written to another CTA)
  pdl_launch_next();
  pdl_wait();
  const float* in = p.in + (size_t)r * p.ldl;
  float* out = p.out + (size_t)r * p.ldo;
  // Groups of four tokens on the input's 16-byte boundaries: group g holds tokens 4g - shift ..; where the output has the same phase it is stored so too.
  const int shift = (int)((uintptr_t)in >> 2) & 3;
  const bool same = ((int)((uintptr_t)out >> 2) & 3) == shift;
  const int groups = (p.V + shift + 3) >> 2, per = (groups + p.cluster - 1) / p.cluster, g0 = min(rank * per, groups), g1 = min(g0 + per, groups);
  float rep = 1.0f, pres = 0.0f, freq = 0.0f, temp = 0.0f;
  if (p.params) {
    const float* q = p.params + 4 * (size_t)r;
    rep = q[0]; pres = q[1]; freq = q[2]; temp = q[3];
  }
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  if (p.hist) { h0 = min(max(p.hist_off[r], 0), p.n_hist); h1 = min(max(p.hist_off[r + 1], h0), p.n_hist); }
  if (p.bias_ids) { b0 = min(max(p.bias_off[r], 0), p.n_bias); b1 = min(max(p.bias_off[r + 1], b0), p.n_bias); }
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int m = p.mask_row ? p.mask_row[r] : r;
    if (m >= 0 && m < p.n_masks) mask = p.mask + (size_t)m * p.mask_words;
  }
  // (what the first steps wait for is asked for ahead of what fills the queues to memory, and kept for every window)
  int early[kEarly];
#pragma unroll
  for (int j = 0; j < kEarly; ++j) early[j] = h0 + tid + j * kThreads < h1 ? p.hist[h0 + tid + j * kThreads] : -1;
  const int early_bias = b0 + tid < b1 ? p.bias_ids[b0 + tid] : -1;
  const bool counted = h1 > h0 || b1 > b0, wide = h1 - h0 > 65535 || b1 - b0 > 65535, logz = p.logz != nullptr;
  const int window = p.words ? (wide ? p.words / 2 : p.words) / 4 : groups;  // groups at a time
  uint32_t* s_bias = s_word + 4 * window;                 // (wide: the numbers of the biases)

  const int i0 = (shift + 3) >> 2, inner = ((p.V + shift) >> 2) - i0;  // groups i0 .. i0 + inner - 1 lie in the row as a whole
  const bool scaled = temp > 0.0f, fast = plain_size(temp);
  const float inv = __frcp_rn(temp);

  // A thread's groups g, g + kThreads, ... come through a ring of its own slots of shared memory, kBatch ahead.
  float4* ring = reinterpret_cast<float4*>(s_word + p.words) + tid;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  auto ask = [&](int g, int slot, int end) {
    if (g < end && (unsigned)(g - i0) < (unsigned)inner)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring_at + slot * (kThreads * 16)), "l"(in + (4 * g - shift)) : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Top top = {-INFINITY, 0.0f, 0x7FFFFFFF};
  float f = -kBig;  // top.m as a finite number
  auto one = [&](float x, uint32_t c, uint32_t b) {
    if (c) {
      x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      x = __fsub_rn(x, __fadd_rn(__fmul_rn(freq, (float)c), pres));
    }
    return b ? __fadd_rn(x, p.bias[b0 + b - 1]) : x;
  };
  for (int w0 = g0; w0 < g1; w0 += window) {
    const int w1 = min(w0 + window, g1);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) ask(w0 + tid + j * kThreads, j, w1);
    if (counted) {
      const int first = 4 * w0 - shift, n = 4 * (w1 - w0);  // word i counts token first + i
      if (w0 > g0) __syncthreads();
      for (int i = tid; i < w1 - w0; i += kThreads) {
        reinterpret_cast<uint4*>(s_word)[i] = make_uint4(0u, 0u, 0u, 0u);
        if (wide) reinterpret_cast<uint4*>(s_bias)[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      __syncthreads();
      auto bias_at = [&](int v, int i) {  // the last entry of a token counts
        const uint32_t at = (uint32_t)v - (uint32_t)first;
        if (v >= 0 && v < p.V && at < (uint32_t)n) atomicMax((wide ? s_bias : s_word) + at, (uint32_t)(i - b0 + 1) << (wide ? 0 : 16));
      };
      if (b1 > b0) {
        bias_at(early_bias, b0 + tid);
        for (int i = b0 + tid + kThreads; i < b1; i += kThreads) bias_at(p.bias_ids[i], i);
        __syncthreads();
      }
      auto count = [&](int v) {
        const uint32_t at = (uint32_t)v - (uint32_t)first;
        if (v >= 0 && v < p.V && at < (uint32_t)n) atomicAdd(s_word + at, 1u);
      };
#pragma unroll
      for (int j = 0; j < kEarly; ++j) count(early[j]);
#pragma unroll 1
      for (int i = h0 + tid + kEarly * kThreads; i < h1; i += 4 * kThreads) {
        int v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j * kThreads < h1 ? p.hist[i + j * kThreads] : -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) count(v[j]);
      }
      __syncthreads();
    }
    for (int g = w0 + tid, slot = 0; g < w1; g += kThreads) {
      const int v = 4 * g - shift;
      const bool whole = (unsigned)(g - i0) < (unsigned)inner;
      ask(g + kBatch * kThreads, slot == 0 ? kBatch : slot - 1, w1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kBatch) : "memory");
      float4 x = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      if (whole) {
        x = ring[slot * kThreads];
      } else {
        if (v >= 0 && v < p.V) x.x = in[v];
        if (v + 1 >= 0 && v + 1 < p.V) x.y = in[v + 1];
        if (v + 2 >= 0 && v + 2 < p.V) x.z = in[v + 2];
        if (v + 3 < p.V) x.w = in[v + 3];
      }
      slot = slot == kBatch ? 0 : slot + 1;
      if (counted) {
        const uint4 c = reinterpret_cast<const uint4*>(s_word)[g - w0];
        if (wide) {
          const uint4 b = reinterpret_cast<const uint4*>(s_bias)[g - w0];
          x = make_float4(one(x.x, c.x, b.x), one(x.y, c.y, b.y), one(x.z, c.z, b.z), one(x.w, c.w, b.w));
        } else if (c.x | c.y | c.z | c.w) {
          x = make_float4(one(x.x, c.x & 0xFFFFu, c.x >> 16), one(x.y, c.y & 0xFFFFu, c.y >> 16), one(x.z, c.z & 0xFFFFu, c.z >> 16), one(x.w, c.w & 0xFFFFu, c.w >> 16));
        }
      }
      if (scaled) {  // (before the mask, which leaves nothing of what it takes either way: few logits are infinite here)
        if (fast && plain_size(x.x) && plain_size(x.y) && plain_size(x.z) && plain_size(x.w))
          x = make_float4(quotient(x.x, temp, inv), quotient(x.y, temp, inv), quotient(x.z, temp, inv), quotient(x.w, temp, inv));
        else
          x = make_float4(__fdiv_rn(x.x, temp), __fdiv_rn(x.y, temp), __fdiv_rn(x.z, temp), __fdiv_rn(x.w, temp));
      }
      if (mask) {  // bits of tokens v .. v + 3 (they may lie in two words)
        const int at = max(v, 0) >> 5;
        const uint32_t lo = mask[at], hi = mask[min(at + 1, p.mask_words - 1)];
        const uint32_t bits = v >= 0 ? __funnelshift_r(lo, hi, v & 31) : lo << -v;
        if (!(bits & 1)) x.x = -INFINITY;
        if (!(bits & 2)) x.y = -INFINITY;
        if (!(bits & 4)) x.z = -INFINITY;
        if (!(bits & 8)) x.w = -INFINITY;
      }
      if (whole && same) {
        *reinterpret_cast<float4*>(out + v) = x;
      } else {  // (what is outside the row counts as -inf)
        if (v >= 0 && v < p.V) out[v] = x.x; else x.x = -INFINITY;
        if (v + 1 >= 0 && v + 1 < p.V) out[v + 1] = x.y; else x.y = -INFINITY;
        if (v + 2 >= 0 && v + 2 < p.V) out[v + 2] = x.z; else x.z = -INFINITY;
        if (v + 3 < p.V) out[v + 3] = x.w; else x.w = -INFINITY;
      }
      const float m = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));  // (fmaxf passes NaN by)
      if (m > top.m) {
        top.m = m;
        top.at = x.x == m ? v : x.y == m ? v + 1 : x.z == m ? v + 2 : v + 3;
        top.s *= exp_of(f - finite(m));
        f = finite(m);
      }
      if (logz) top.s += (exp_of(x.x - f) + exp_of(x.y - f)) + (exp_of(x.z - f) + exp_of(x.w - f));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // over the warp, the CTA's warps, the row's CTAs: lane by lane each time
  auto join = [&](int lanes) {
#pragma unroll 1
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      const Top b = {__shfl_xor_sync(0xFFFFFFFFu, top.m, o), __shfl_xor_sync(0xFFFFFFFFu, top.s, o), __shfl_xor_sync(0xFFFFFFFFu, top.at, o)};
      top = top_join(top, b);
    }
  };
  join(32);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  if (p.cluster > 1) asm volatile("barrier.cluster.wait;" ::: "memory");  // every CTA of the row has begun
  if (warp == 0) {
    top = s_top[lane & (kThreads / 32 - 1)];
    join(kThreads / 32);
    if (p.cluster > 1 && lane == 0) {  // into the first CTA's shared memory
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&s_cta[rank])));
      asm volatile("st.shared::cluster.f32 [%0], %1;\n\tst.shared::cluster.f32 [%0+4], %2;\n\tst.shared::cluster.s32 [%0+8], %3;" ::"r"(to), "f"(top.m), "f"(top.s), "r"(top.at)
                   : "memory");
    }
  }
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  if (rank == 0 && warp == 0) {
    if (p.cluster > 1) {
      top = s_cta[lane & (p.cluster - 1)];  // (a power of two)
      join(p.cluster);
    }
    if (lane == 0) {
      if (p.best) p.best[r] = top.at == 0x7FFFFFFF ? 0 : top.at;
      if (logz) p.logz[r] = logf(top.s) + top.m;
    }
  }
}

}  // namespace

extern "C" int izb_logits_process(const float* d_logits, int ldl, float* d_out, int ldo, int rows, int V, const float* d_params, const int32_t* d_hist,
                                  const int32_t* d_hist_off, int n_hist, const int32_t* d_bias_ids, const float* d_bias, const int32_t* d_bias_off, int n_bias,
                                  const uint32_t* d_mask, int mask_words, int n_masks, const int32_t* d_mask_row, int32_t* d_best, float* d_logz, void* stream) {
  if (!d_logits || !d_out) IZB_FAIL(IZB_ERR_ARG, "logits_process: null pointer");
  if (rows < 1 || V < 1 || V > 1 << 30 || (rows > 1 && (ldl < V || ldo < V))) IZB_FAIL(IZB_ERR_SHAPE, "logits_process: rows=%d V=%d ldl=%d ldo=%d (ldl, ldo >= V)", rows, V, ldl, ldo);
  if (n_hist < 0 || (n_hist && (!d_hist || !d_hist_off)) || n_bias < 0 || (n_bias && (!d_bias_ids || !d_bias || !d_bias_off)))
    IZB_FAIL(IZB_ERR_ARG, "logits_process: %d history tokens, %d biases and a null pointer among their arrays", n_hist, n_bias);
  if (n_hist > 1 << 30 || n_bias > 1 << 30) IZB_FAIL(IZB_ERR_LIMIT, "logits_process: %d history tokens, %d biases (2^30 at most)", n_hist, n_bias);
  if (n_hist && !d_params) IZB_FAIL(IZB_ERR_ARG, "logits_process: a history without the penalties' parameters");
  if (d_mask && (mask_words < 0 || (int64_t)mask_words * 32 < V || n_masks < 1 || (!d_mask_row && n_masks < rows)))
    IZB_FAIL(IZB_ERR_SHAPE, "logits_process: %d masks of %d words for %d rows of %d tokens", n_masks, mask_words, rows, V);
  if (d_mask_row && !d_mask) IZB_FAIL(IZB_ERR_ARG, "logits_process: rows of a mask that is not there");
  if (izb_overlap_in_part(d_logits, ldl, d_out, ldo, rows, V)) IZB_FAIL(IZB_ERR_ARG, "logits_process: the output overlaps the logits in part");
  if (!izb_aligned(d_logits, 4) || !izb_aligned(d_out, 4)) IZB_FAIL(IZB_ERR_ALIGN, "logits_process: logits and out must be 4-byte aligned");
  LogitsArgs p = {};
  p.in = d_logits; p.out = d_out; p.params = d_params;
  if (n_hist) { p.hist = d_hist; p.hist_off = d_hist_off; }
  if (n_bias) { p.bias_ids = d_bias_ids; p.bias = d_bias; p.bias_off = d_bias_off; }
  p.mask = d_mask; p.mask_row = d_mask_row;
  p.best = d_best; p.logz = d_logz;
  p.ldl = ldl; p.ldo = ldo; p.V = V; p.n_hist = n_hist; p.n_bias = n_bias; p.mask_words = mask_words; p.n_masks = n_masks;
  // How many CTAs share a row: 16 while that leaves the multiprocessors two CTAs at most, else 4 (64 rows of 151936, CTAs per row 2 / 4 / 8: 63 / 38 / 44 us;
  // 256 rows of 128256: 86 / 86 / 102; without rules 24 / 16 / 21 and 50 / 54 / 69), and no more than give every thread a group.
  int device = 0;
  IZB_CUDA(cudaGetDevice(&device));
  const int groups = V / 4 + 2;
  int cluster = (int64_t)rows * 16 <= 2 * izb_sm_count(device) ? 16 : 4;
  while (cluster > 1 && groups < cluster / 2 * kThreads) cluster /= 2;
  if ((int64_t)rows * cluster > 0x7FFFFFFF) IZB_FAIL(IZB_ERR_LIMIT, "logits_process: %d rows", rows);
  p.cluster = cluster;
  const int need = ((groups + cluster - 1) / cluster) * 4;
  p.words = ((need < kWords ? need : kWords) + 7) / 8 * 8;
  if (!n_hist && !n_bias) p.words = 0;
  const size_t smem = (size_t)p.words * 4 + kRing;
  cudaStream_t st = (cudaStream_t)stream;
  IZB_SMEM_OPTIN(logits_process_kernel, kWords * 4 + kRing, device);
  static izb_device_once sixteen;
  if (int rc = sixteen.run(device, [&]() -> int {
        IZB_CUDA(cudaFuncSetAttribute(logits_process_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        return IZB_OK;
      }))
    return rc;
  IZB_LAUNCH("logits_process", st, izb_launch_pdl_cluster(logits_process_kernel, cluster, dim3(rows * cluster), kThreads, smem, st, p));
  return IZB_OK;
}
