// The whole mixture-of-experts block of a few tokens (a decode step's) in two kernels: routing, gate and up projections with SwiGLU, then the
// down projection with the weighted sum over a token's experts, the shared expert's output and the residual.
//   e_k, w_k as izb_moe_route;  g = x Wg_e^T, u = x Wu_e^T;  h = u * g / (1 + exp(-g));  out = x + sum_k w_k h_k Wd_e^T + sgate * sh
// The six-call path quantises h to int8 in between; here it stays in f32.
#include "izb_common.cuh"

namespace {

constexpr int kWarps = 8, kMaxTokens = 32, kMaxPairs = 512, kMaxExperts = 512, kMaxChoices = 32;

struct MoeArgs {
  const uint8_t *wg, *wu, *wd;
  const int8_t* aq;
  const float *asc, *logits, *x, *sh;
  float *h, *out;
  int T, Mp, ldl, NE, NU, e0, n_mats, E, F;
  int joined;                          // gate and up rows alternate in groups of 32 in wg
  size_t gate_row, down_row;           // bytes of a row
};

// One warp: the choices of a token, in order; s_id and s_wt get NU entries (ties go to the lower id; the weights' sum in choice order).
__device__ void route_token(const float* row, int NE, int NU, int* s_id, float* s_wt) {
  const int lane = threadIdx.x & 31;
  uint32_t key[kMaxExperts / 32];
#pragma unroll
  for (int i = 0; i < kMaxExperts / 32; ++i) {
    key[i] = 0u;
    if (i * 32 + lane < NE) {
      uint32_t u = __float_as_uint(__fadd_rn(row[i * 32 + lane], 0.0f));
      u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
      key[i] = u ? u : 1u;
    }
  }
  float top = 0.0f, denom = 0.0f, mine = 0.0f;
  int id = 0;
  for (int k = 0; k < NU; ++k) {
    uint32_t best = 0u;
    int at = 0;
#pragma unroll
    for (int i = 0; i < kMaxExperts / 32; ++i)
      if (key[i] > best) { best = key[i]; at = i * 32 + lane; }
    const uint32_t win = __reduce_max_sync(0xFFFFFFFFu, best);
    const int e = (int)__reduce_min_sync(0xFFFFFFFFu, best == win ? (uint32_t)at : 0xFFFFu);
#pragma unroll
    for (int i = 0; i < kMaxExperts / 32; ++i)
      if (i * 32 + lane == e) key[i] = 0u;
    const float l = __uint_as_float((win & 0x80000000u) ? (win & 0x7FFFFFFFu) : ~win);
    if (k == 0) top = l;
    const float p = expf(l - top);
    denom += p;
    if (lane == k) { mine = p; id = e; }
  }
  if (lane < NU) { s_id[lane] = id; s_wt[lane] = __fdiv_rn(mine, denom); }
}

// weight `k` of a row in the device form
template <int QT>
__device__ __forceinline__ float weight_at(const uint8_t* row, int k) {
  const uint8_t* sb = row + (size_t)(k >> 8) * (QT == IZB_Q4_K ? 144 : 272);
  const int j = (k >> 5) & 7, l = k & 31;
  if (QT == IZB_Q8_0) return half_bits_to_float(reinterpret_cast<const uint16_t*>(sb)[j]) * (float)(int8_t)sb[16 + 32 * j + l];
  const uint32_t* w = reinterpret_cast<const uint32_t*>(sb);
  const uint32_t s[3] = {w[1], w[2], w[3]};
  int sc, mn;
  q4k_scale_min(s, j, sc, mn);
  const int b = sb[16 + 32 * (j >> 1) + l], q = (j & 1) ? b >> 4 : b & 15;
  return half_bits_to_float(w[0] & 0xFFFF) * sc * q - half_bits_to_float(w[0] >> 16) * mn;
}

template <int QT>
__global__ void __launch_bounds__(kWarps * 32) moe_layer_up_kernel(MoeArgs p) {
  __shared__ int s_id[kMaxChoices];
  __shared__ float s_wt[kMaxChoices];
  const int t = blockIdx.y / p.NU, k = blockIdx.y % p.NU, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) route_token(p.logits + (size_t)t * p.ldl, p.NE, p.NU, s_id, s_wt);
  __syncthreads();
  const int e = s_id[k] - p.e0, f = blockIdx.x * kWarps + warp;
  if (e < 0 || e >= p.n_mats) return;
  const size_t rows = p.joined ? 2 * (size_t)p.F : p.F, g_row = (size_t)e * rows + (p.joined ? (f >> 5) * 64 + (f & 31) : f);
  const uint8_t *rg = p.wg + g_row * p.gate_row, *ru = p.joined ? rg + 32 * p.gate_row : p.wu + g_row * p.gate_row;
  float g = 0.0f, u = 0.0f;
  for (int i = lane; i < p.E; i += 32) {
    const float x = (float)p.aq[(size_t)t * p.E + i] * p.asc[(size_t)(i >> 5) * p.Mp + t];
    g += weight_at<QT>(rg, i) * x;
    u += weight_at<QT>(ru, i) * x;
  }
  g = warp_sum(g);
  u = warp_sum(u);
  if (lane == 0) p.h[(size_t)blockIdx.y * p.F + f] = g / (1.0f + expf(-g)) * u;
}

template <int QT>
__global__ void __launch_bounds__(kWarps * 32) moe_layer_down_kernel(MoeArgs p) {
  __shared__ int s_id[kMaxChoices];
  __shared__ float s_wt[kMaxChoices];
  const int t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockIdx.x * kWarps + warp;
  if (warp == 0) route_token(p.logits + (size_t)t * p.ldl, p.NE, p.NU, s_id, s_wt);
  __syncthreads();
  float v = 0.0f;
  for (int k = 0; k < p.NU; ++k) {
    const int e = s_id[k] - p.e0;
    if (e < 0 || e >= p.n_mats) continue;
    const uint8_t* row = p.wd + ((size_t)e * p.E + n) * p.down_row;
    const float* h = p.h + (size_t)(t * p.NU + k) * p.F;
    float y = 0.0f;
    for (int i = lane; i < p.F; i += 32) y += weight_at<QT>(row, i) * h[i];
    v += s_wt[k] * warp_sum(y);
  }
  if (lane == 0) {
    const size_t at = (size_t)t * p.E + n;
    if (p.sh) v += p.sh[at] / (1.0f + expf(-p.logits[(size_t)t * p.ldl + p.NE]));
    p.out[at] = p.x ? p.x[at] + v : v;
  }
}

bool takes(const izb_weight* w) { return w->type == IZB_Q4_K || w->type == IZB_Q8_0; }

}  // namespace

extern "C" size_t izb_moe_layer_scratch(int T, int NU, int F) {
  return T < 1 || NU < 1 || F < 1 ? 0 : (size_t)T * NU * F * 4;
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
  p.h = (float*)d_scratch; p.out = d_out;
  p.T = T; p.Mp = Mp; p.ldl = ldl; p.NE = NE; p.NU = NU; p.e0 = e0; p.n_mats = wg->n_mats; p.E = E; p.F = F;
  p.joined = wg->gu32; p.gate_row = wg->row_bytes; p.down_row = wd->row_bytes;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 up(F / kWarps, T * NU), down(E / kWarps, T);
  if (wg->type == IZB_Q4_K)
    IZB_LAUNCH("moe_layer_up", st, moe_layer_up_kernel<IZB_Q4_K><<<up, kWarps * 32, 0, st>>>(p));
  else
    IZB_LAUNCH("moe_layer_up", st, moe_layer_up_kernel<IZB_Q8_0><<<up, kWarps * 32, 0, st>>>(p));
  if (wd->type == IZB_Q4_K)
    IZB_LAUNCH("moe_layer_down", st, moe_layer_down_kernel<IZB_Q4_K><<<down, kWarps * 32, 0, st>>>(p));
  else
    IZB_LAUNCH("moe_layer_down", st, moe_layer_down_kernel<IZB_Q8_0><<<down, kWarps * 32, 0, st>>>(p));
  return IZB_OK;
}
