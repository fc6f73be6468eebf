// Low-rank adapters of many requests beside a shared projection: the rows of a call come in segments, each with an adapter of its own
// or none,
//   u[t][j] = sum_k A[j][k] x[t][k],  x[t][k] = asc[k / 32][t] aq[t][k],      C[t][c_off + n] = base[t][n] + scale * sum_j B[n][j] u[t][j].
#include <cuda_bf16.h>

#include "izb_common.cuh"

namespace {

constexpr int kThreads = 256, kRows = 8, kMaxRank = 256;

struct LoraArgs {
  const uint16_t *A, *B;
  const int32_t *ranks, *seg, *adapter;
  const float *scales, *asc, *base;
  const int8_t* aq;
  float* C;
  int n_ad, R, N, K, T, Mp, n_seg, ldb, ldc, c_off;
};

template <bool kBf16>
__device__ __forceinline__ float value(uint16_t v) {
  return kBf16 ? __uint_as_float((uint32_t)v << 16) : __half2float(__ushort_as_half(v));
}

// one CTA per up to kRows rows of a segment
template <bool kBf16>
__global__ void __launch_bounds__(kThreads) lora_kernel(LoraArgs p) {
  __shared__ float s_u[kMaxRank][kRows];
  __shared__ int s_at[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    int tile = blockIdx.x;
    s_at[2] = 0;
    for (int s = 0; s < p.n_seg; ++s) {
      const int lo = min(max(p.seg[s], 0), p.T), hi = min(max(p.seg[s + 1], lo), p.T), n = (hi - lo + kRows - 1) / kRows;
      if (tile < n) {
        s_at[0] = s;
        s_at[1] = lo + tile * kRows;
        s_at[2] = min(kRows, hi - s_at[1]);
        break;
      }
      tile -= n;
    }
  }
  __syncthreads();
  const int t0 = s_at[1], rows = s_at[2];
  if (!rows) return;
  const int a = p.adapter[s_at[0]];
  const bool with = a >= 0 && a < p.n_ad;
  const int rank = with ? min(max(p.ranks ? p.ranks[a] : p.R, 0), p.R) : 0;
  for (int j = warp; j < rank; j += kThreads / 32) {
    const uint16_t* row = p.A + ((size_t)a * p.R + j) * p.K;
    for (int t = 0; t < rows; ++t) {
      float u = 0.0f;
      for (int k = lane; k < p.K; k += 32) u += value<kBf16>(row[k]) * ((float)p.aq[(size_t)(t0 + t) * p.K + k] * p.asc[(size_t)(k >> 5) * p.Mp + t0 + t]);
      u = warp_sum(u);
      if (lane == 0) s_u[j][t] = u;
    }
  }
  __syncthreads();
  const float scale = with ? p.scales[a] : 0.0f;
  for (int n = tid; n < p.N; n += kThreads)
    for (int t = 0; t < rows; ++t) {
      float y = 0.0f;
      for (int j = 0; j < rank; ++j) y += value<kBf16>(p.B[((size_t)a * p.N + n) * p.R + j]) * s_u[j][t];
      const float b = p.base ? p.base[(size_t)(t0 + t) * p.ldb + n] : 0.0f;
      p.C[(size_t)(t0 + t) * p.ldc + p.c_off + n] = with ? b + scale * y : b;
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
  const int64_t tiles = (int64_t)T / kRows + n_seg;
  if (tiles > 0x7FFFFFFF) IZB_FAIL(IZB_ERR_LIMIT, "lora_add: %d rows in %d segments", T, n_seg);
  LoraArgs p = {(const uint16_t*)d_A, (const uint16_t*)d_B, d_ranks, d_seg, d_adapter, d_scales, d_asc, d_base, d_aq, d_C, n_adapters, R, N, K, T, Mp, n_seg, ldb, ldc, c_off};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == IZB_BF16)
    IZB_LAUNCH("lora_add", st, lora_kernel<true><<<(unsigned)tiles, kThreads, 0, st>>>(p));
  else
    IZB_LAUNCH("lora_add", st, lora_kernel<false><<<(unsigned)tiles, kThreads, 0, st>>>(p));
  return IZB_OK;
}
