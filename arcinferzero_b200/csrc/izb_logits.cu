// The rules of each request on its row of the output head's logits: penalties for tokens that the row's history holds, a list of
// biases, a grammar mask, the temperature; and of the outcome the best token and log(sum(exp)).
//
//   c[v] = how often v stands in the row's history;  per token, in this order, each operation rounded once:
//   c > 0:          l = l > 0 ? l / repetition : l * repetition,  l = l - (frequency * c + presence)
//   v in the list:  l = l + bias
//   mask bit 0:     l = -inf
//   temperature>0:  l = l / temperature
#include <math.h>

#include "izb_common.cuh"

namespace {

constexpr int kThreads = 512, kChunk = 4096;

struct LogitsArgs {
  const float* in;
  float* out;
  const float* params;
  const int32_t *hist, *hist_off, *bias_ids, *bias_off, *mask_row;
  const float* bias;
  const uint32_t* mask;
  int32_t* best;
  float* logz;
  int ldl, ldo, V, n_hist, n_bias, mask_words, n_masks;
};

struct Top {  // largest value, its lowest index, sum of exp(l - m)
  float m, s;
  int at;
};
__device__ __forceinline__ Top top_join(Top a, Top b) {
  const bool of_b = b.m > a.m || (b.m == a.m && b.at < a.at);
  const float m = of_b ? b.m : a.m;
  // (a sum whose maximum is m stays as it is, infinite or not)
  const float s = (a.m == m ? a.s : a.s * expf(a.m - m)) + (b.m == m ? b.s : b.s * expf(b.m - m));
  return {m, s, of_b ? b.at : a.at};
}

__global__ void __launch_bounds__(kThreads) logits_process_kernel(LogitsArgs p) {
  __shared__ int s_count[kChunk], s_bias[kChunk];
  __shared__ Top s_top[kThreads / 32];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* in = p.in + (size_t)r * p.ldl;
  float* out = p.out + (size_t)r * p.ldo;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f, temp = 0.0f;
  if (p.params) { rep = p.params[4 * r]; pres = p.params[4 * r + 1]; freq = p.params[4 * r + 2]; temp = p.params[4 * r + 3]; }
  int h0 = 0, h1 = 0, b0 = 0, b1 = 0;
  if (p.hist && p.params) { h0 = min(max(p.hist_off[r], 0), p.n_hist); h1 = min(max(p.hist_off[r + 1], h0), p.n_hist); }
  if (p.bias_ids) { b0 = min(max(p.bias_off[r], 0), p.n_bias); b1 = min(max(p.bias_off[r + 1], b0), p.n_bias); }
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int m = p.mask_row ? p.mask_row[r] : r;
    if (m >= 0 && m < p.n_masks) mask = p.mask + (size_t)m * p.mask_words;
  }
  Top top = {-INFINITY, 0.0f, 0x7FFFFFFF};
  for (int v0 = 0; v0 < p.V; v0 += kChunk) {
    const int n = min(kChunk, p.V - v0);
    for (int i = tid; i < n; i += kThreads) s_count[i] = s_bias[i] = 0;
    __syncthreads();
    for (int i = h0 + tid; i < h1; i += kThreads) {
      const uint32_t v = (uint32_t)p.hist[i] - (uint32_t)v0;  // (tokens outside the vocabulary fall outside every chunk)
      if (p.hist[i] >= 0 && v < (uint32_t)n) atomicAdd(&s_count[v], 1);
    }
    for (int i = b0 + tid; i < b1; i += kThreads) {  // the last entry of a token counts
      const uint32_t v = (uint32_t)p.bias_ids[i] - (uint32_t)v0;
      if (p.bias_ids[i] >= 0 && v < (uint32_t)n) atomicMax(&s_bias[v], i - b0 + 1);
    }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const int v = v0 + i, c = s_count[i], b = s_bias[i];
      float l = in[v];
      if (c > 0) {
        l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        l = __fsub_rn(l, __fadd_rn(__fmul_rn(freq, (float)c), pres));
      }
      if (b) l = __fadd_rn(l, p.bias[b0 + b - 1]);
      if (mask && !(mask[v >> 5] >> (v & 31) & 1)) l = -INFINITY;
      if (temp > 0.0f) l = __fdiv_rn(l, temp);
      out[v] = l;
      if (l > top.m) {
        top.s = top.s * expf(top.m - l) + 1.0f;
        top.m = l;
        top.at = v;
      } else if (l == top.m) {
        top.s += l > -INFINITY ? 1.0f : 0.0f;
      } else {
        top.s += expf(l - top.m);
      }
    }
    __syncthreads();
  }
  for (int o = 16; o > 0; o >>= 1) {
    const Top b = {__shfl_xor_sync(0xFFFFFFFFu, top.m, o), __shfl_xor_sync(0xFFFFFFFFu, top.s, o), __shfl_xor_sync(0xFFFFFFFFu, top.at, o)};
    top = top_join(top, b);
  }
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; ++w) top = top_join(top, s_top[w]);
    if (p.best) p.best[r] = top.at == 0x7FFFFFFF ? 0 : top.at;
    if (p.logz) p.logz[r] = logf(top.s) + top.m;
  }
}

}  // namespace

extern "C" int izb_logits_process(const float* d_logits, int ldl, float* d_out, int ldo, int rows, int V, const float* d_params, const int32_t* d_hist,
                                  const int32_t* d_hist_off, int n_hist, const int32_t* d_bias_ids, const float* d_bias, const int32_t* d_bias_off, int n_bias,
                                  const uint32_t* d_mask, int mask_words, int n_masks, const int32_t* d_mask_row, int32_t* d_best, float* d_logz, void* stream) {
  if (!d_logits || !d_out) IZB_FAIL(IZB_ERR_ARG, "logits_process: null pointer");
  if (rows < 1 || V < 1 || (rows > 1 && (ldl < V || ldo < V))) IZB_FAIL(IZB_ERR_SHAPE, "logits_process: rows=%d V=%d ldl=%d ldo=%d (ldl, ldo >= V)", rows, V, ldl, ldo);
  if (n_hist < 0 || (n_hist && (!d_hist || !d_hist_off)) || n_bias < 0 || (n_bias && (!d_bias_ids || !d_bias || !d_bias_off)))
    IZB_FAIL(IZB_ERR_ARG, "logits_process: %d history tokens, %d biases and a null pointer among their arrays", n_hist, n_bias);
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
  cudaStream_t st = (cudaStream_t)stream;
  IZB_LAUNCH("logits_process", st, logits_process_kernel<<<rows, kThreads, 0, st>>>(p));
  return IZB_OK;
}
