// Small program over the C++ mirror (engine.hpp): one FFN block of a dense layer as the reference's layer_ffn issues it
// (zero/engine_qwen.h:419-452): quantise -> gate (store) -> up (fused SwiGLU store mode) -> quantise -> down (add to
// the residual).  Prints a checksum; the GPU test compares it with the same sequence through the Python binding.
// Then what a server of many requests adds to a step -- adapters, the expert block of a few rows, rules on logits -- through the mirror and
// through the C calls themselves, which must agree bit for bit.
// usage: engine_demo <rows> <hidden> <ffn> <seed>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>

#include "engine.hpp"

static std::vector<uint8_t> random_q4k(int N, int K, uint32_t seed) {
  std::mt19937 rng(seed);
  std::vector<uint8_t> w((size_t)N * (K / 256) * 144);
  for (auto& b : w) b = (uint8_t)rng();
  for (size_t sb = 0; sb < w.size() / 144; ++sb) {  // fp16 d, dmin in a sane range: 0x1C00..0x2000 = 0.0039..0.0078
    const uint16_t d = (uint16_t)(0x1C00 + rng() % 0x400), m = (uint16_t)(0x1C00 + rng() % 0x400);
    memcpy(&w[sb * 144], &d, 2);
    memcpy(&w[sb * 144 + 2], &m, 2);
  }
  return w;
}

// device copies that live until the end of the program
template <class V>
static V* on_device(const std::vector<V>& v) {
  V* d = nullptr;
  if (cudaMalloc(&d, v.size() * sizeof(V)) != cudaSuccess || cudaMemcpy(d, v.data(), v.size() * sizeof(V), cudaMemcpyHostToDevice) != cudaSuccess)
    throw std::runtime_error("engine_demo: out of device memory");
  return d;
}
static bool equal_on_device(const float* a, const float* b, size_t n) {
  std::vector<float> x(n), y(n);
  cudaMemcpy(x.data(), a, n * 4, cudaMemcpyDeviceToHost);
  cudaMemcpy(y.data(), b, n * 4, cudaMemcpyDeviceToHost);
  bool any = false;
  for (float v : x) any = any || (v != 0.0f && v == v);
  return any && memcmp(x.data(), y.data(), n * 4) == 0;
}

// One step of `T` rows of E values, F channels per expert.
static bool request_operators(izb::Engine& eng, int T, int E, int F, uint32_t seed) {
  std::mt19937 rng(seed);
  std::normal_distribution<float> nd(0.0f, 1.0f);
  auto normal = [&](size_t n) { std::vector<float> v(n); for (auto& x : v) x = nd(rng); return v; };
  const int Mp = izb::Engine::pad_rows(T), NE = 6, NU = 2, R = 16, V = 1003;
  float* x = on_device(normal((size_t)T * E));
  int8_t* aq = on_device(std::vector<int8_t>((size_t)Mp * E));
  float* asc = on_device(std::vector<float>((size_t)Mp * (E / 32)));
  izb::check(izb_quantize_act(x, E, T, Mp, E, aq, asc, nullptr, nullptr), "quantize_act");
  eng.set_rows(T);
  eng.quant_rows(x, E, E, Mp);
  bool same = true;

  // adapters: all rows one request's, then a request per row
  std::vector<uint16_t> a((size_t)2 * R * E), b((size_t)2 * F * R);
  for (auto* w : {&a, &b})
    for (auto& h : *w) h = (uint16_t)((rng() & 0x8000) | (0x2400 + rng() % 0x800));  // f16 of 0.016 .. 0.06
  izb::Engine::Adapters ad;
  ad.dtype = IZB_F16; ad.n = 2; ad.R = R; ad.N = F; ad.K = E;
  ad.A = on_device(a); ad.B = on_device(b); ad.scales = on_device(std::vector<float>{0.5f, 2.0f});
  std::vector<int32_t> rows(T + 1), which(T);
  for (int t = 0; t <= T; ++t) rows[t] = t;
  for (int t = 0; t < T; ++t) which[t] = t % 3 - 1;
  const std::vector<float> c0 = normal((size_t)T * (F + 4));
  for (int n_seg : {1, T}) {
    const int32_t *seg = on_device(n_seg == 1 ? std::vector<int32_t>{0, T} : rows), *adapter = on_device(n_seg == 1 ? std::vector<int32_t>{1} : which);
    float *c1 = on_device(c0), *c2 = on_device(c0);
    void* scratch = on_device(std::vector<uint8_t>(eng.lora_scratch(ad, n_seg) + 16));
    eng.lora_add(ad, seg, adapter, n_seg, c1, F + 4, 4, scratch);
    izb::check(izb_lora_add(ad.dtype, ad.A, ad.B, ad.n, R, nullptr, ad.scales, F, E, aq, asc, T, Mp, seg, adapter, n_seg, c2 + 4, F + 4, c2, F + 4, 4, scratch, nullptr), "lora_add");
    same = same && equal_on_device(c1, c2, c0.size());
  }

  // the expert block: whole and in place, then experts [2, 6) alone
  const int Td = T < 32 ? T : 32, Mpd = izb::Engine::pad_rows(Td);
  const auto g = random_q4k(NE * F, E, seed + 1), u = random_q4k(NE * F, E, seed + 2), d = random_q4k(NE * E, F, seed + 3);
  izb::GpuWeight gu = eng.make_weight_gateup(IZB_Q4_K, g.data(), u.data(), F, E, NE), down = eng.make_weight(IZB_Q4_K, d.data(), E, F, NE);
  const size_t of_gu = g.size() / NE, of_d = d.size() / NE;
  izb::GpuWeight g2 = eng.make_weight(IZB_Q4_K, g.data() + 2 * of_gu, F, E, NE - 2), u2 = eng.make_weight(IZB_Q4_K, u.data() + 2 * of_gu, F, E, NE - 2),
                 d2 = eng.make_weight(IZB_Q4_K, d.data() + 2 * of_d, E, F, NE - 2);
  const float *logits = on_device(normal((size_t)Td * (NE + 1))), *sh = on_device(normal((size_t)Td * E));
  const std::vector<float> r0 = normal((size_t)Td * E);
  float *r1 = on_device(r0), *r2 = on_device(r0), *p1 = on_device(r0), *p2 = on_device(r0);
  izb::check(izb_quantize_act(x, E, Td, Mpd, E, aq, asc, nullptr, nullptr), "quantize_act");
  eng.set_rows(Td);
  eng.quant_rows(x, E, E, Mpd);
  void* scratch = on_device(std::vector<uint8_t>(eng.moe_scratch(NU, F)));
  eng.moe_layer(gu, nullptr, down, logits, NE + 1, NE, NU, sh, r1, scratch);
  izb::check(izb_moe_layer(gu.h, nullptr, down.h, aq, asc, Td, Mpd, logits, NE + 1, NE, NU, 0, sh, r2, r2, scratch, nullptr), "moe_layer");
  same = same && equal_on_device(r1, r2, r0.size());
  eng.moe_layer(g2, &u2, d2, logits, NE + 1, NE, NU, nullptr, nullptr, scratch, 2, p1);
  izb::check(izb_moe_layer(g2.h, u2.h, d2.h, aq, asc, Td, Mpd, logits, NE + 1, NE, NU, 2, nullptr, nullptr, p2, scratch, nullptr), "moe_layer");
  same = same && equal_on_device(p1, p2, r0.size());

  // rules on logits: penalties, a bias per row, a mask for the first row
  const std::vector<float> l0 = normal((size_t)Td * V);
  std::vector<float> params, bias(Td, 1.5f);
  std::vector<int32_t> hist, off(Td + 1), ids(Td), mask_row(Td, -1);
  for (int t = 0; t < Td; ++t) {
    params.insert(params.end(), {1.25f, 0.5f, 0.25f, 0.75f});
    for (int i = 0; i < 3; ++i) hist.push_back((int32_t)(rng() % V));
    ids[t] = (int32_t)(rng() % V);
    off[t + 1] = t + 1;
  }
  std::vector<int32_t> hist_off(off);
  for (auto& v : hist_off) v *= 3;
  mask_row[0] = 0;
  izb::Engine::LogitRules r;
  r.params = on_device(params); r.hist = on_device(hist); r.hist_off = on_device(hist_off); r.n_hist = 3 * Td;
  r.bias_ids = on_device(ids); r.bias = on_device(bias); r.bias_off = on_device(off); r.n_bias = Td;
  r.mask = on_device(std::vector<uint32_t>((V + 31) / 32, 0xAAAAAAAAu)); r.mask_words = (V + 31) / 32; r.n_masks = 1; r.mask_row = on_device(mask_row);
  float *l1 = on_device(l0), *l2 = on_device(l0), *z1 = on_device(std::vector<float>(Td)), *z2 = on_device(std::vector<float>(Td));
  int32_t *b1 = on_device(std::vector<int32_t>(Td)), *b2 = on_device(std::vector<int32_t>(Td));
  eng.logits_process(l1, V, V, r, b1, z1);
  izb::check(izb_logits_process(l2, V, l2, V, Td, V, r.params, r.hist, r.hist_off, 3 * Td, r.bias_ids, r.bias, r.bias_off, Td, r.mask, r.mask_words, 1, r.mask_row, b2, z2, nullptr),
             "logits_process");
  same = same && equal_on_device(l1, l2, l0.size()) && equal_on_device(z1, z2, Td) && !equal_on_device(l1, on_device(l0), l0.size());
  return same;
}

int main(int argc, char** argv) {
  const int T = argc > 1 ? atoi(argv[1]) : 40, E = argc > 2 ? atoi(argv[2]) : 512, F = argc > 3 ? atoi(argv[3]) : 1024;
  const uint32_t seed = argc > 4 ? (uint32_t)atoi(argv[4]) : 1;
  try {
    izb::Engine eng(0);
    const auto wg = random_q4k(F, E, seed), wu = random_q4k(F, E, seed + 1), wd = random_q4k(E, F, seed + 2);
    izb::GpuWeight Wg = eng.make_weight(IZB_Q4_K, wg.data(), F, E), Wu = eng.make_weight(IZB_Q4_K, wu.data(), F, E),
                   Wd = eng.make_weight(IZB_Q4_K, wd.data(), E, F);
    const int Mp = izb::Engine::pad_rows(T);
    eng.alloc_buffers(Mp, F > E ? F : E);
    std::mt19937 rng(seed + 3);
    std::normal_distribution<float> nd(0.0f, 1.0f);
    std::vector<float> x((size_t)T * E);
    for (auto& v : x) v = nd(rng);
    float *dx, *dh, *dres;
    cudaMalloc(&dx, x.size() * 4);
    cudaMalloc(&dh, (size_t)Mp * F * 4);
    cudaMalloc(&dres, (size_t)Mp * E * 4);
    cudaMemcpy(dx, x.data(), x.size() * 4, cudaMemcpyHostToDevice);
    cudaMemset(dres, 0, (size_t)Mp * E * 4);
    eng.set_rows(T);
    eng.quant_rows(dx, E, E, Mp);
    eng.matmul("gemm_gate", Wg, Mp, dh, F, 0, 0);
    eng.matmul("gemm_up", Wu, Mp, dh, F, 0, 2);      // h = up * silu(gate)
    eng.quant_rows(dh, F, F, Mp);
    eng.matmul("gemm_down", Wd, Mp, dres, E, 0, 1);  // residual += h Wd^T
    std::vector<float> out((size_t)T * E);
    cudaMemcpy(out.data(), dres, out.size() * 4, cudaMemcpyDeviceToHost);
    double sum = 0, sq = 0;
    for (float v : out) { sum += v; sq += (double)v * v; }
    printf("rows %d hidden %d ffn %d checksum %.6e l2 %.6e\n", T, E, F, sum, sq);
    // a bad shape must throw before anything is launched
    bool threw = false;
    try { eng.matmul("bad", Wg, Mp, dres, E, 0, 0); } catch (const std::runtime_error&) { threw = true; }  // Wg.K = E, rows hold F
    printf("shape error raised: %s\n", threw ? "yes" : "no");
    cudaFree(dx); cudaFree(dh); cudaFree(dres);
    const bool same = request_operators(eng, T, E, F, seed + 4);
    printf("request operators equal the C calls: %s\n", same ? "yes" : "no");
    return threw && same ? 0 : 2;
  } catch (const std::exception& e) {
    fprintf(stderr, "engine_demo: %s\n", e.what());
    return 1;
  }
}
