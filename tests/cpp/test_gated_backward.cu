// test_gated_backward.cu — the C++ backward pass of the gated product takes the
// layouts that its forward pass takes: views, and transpose() views of weights
// stored N x K.
// Run: test_gated_backward cpu | gpu | all
#include <cmath>
#include <vector>

#include "choreo-ir/choreo-ir.hpp"
#include "mini_test.hpp"

using namespace choreo_ir;

namespace {
using bf16 = bfloat16_t;
}

TEST(gpu_gated_backward, TransposedWeightsAndViews) {
  initialize();
  const int M = 70, N = 96, K = 80;
  auto X = host_tensor<bf16>::random({M, K}, -1, 1, 1);
  auto Wg = host_tensor<bf16>::random({K, N}, -0.2f, 0.2f, 2);
  auto Wu = host_tensor<bf16>::random({K, N}, -0.2f, 0.2f, 3);
  auto dH = host_tensor<bf16>::random({M, N}, -1, 1, 4);
  auto WgT = host_tensor<bf16>::zeros({N, K}), WuT = host_tensor<bf16>::zeros({N, K});
  for (int k = 0; k < K; ++k)
    for (int j = 0; j < N; ++j) {
      WgT(j, k) = Wg(k, j);
      WuT(j, k) = Wu(k, j);
    }
  auto Xd = X.to_device(), Wgd = Wg.to_device(), Wud = Wu.to_device(), dHd = dH.to_device();
  auto WgTd = WgT.to_device(), WuTd = WuT.to_device();
  compute::GatedFfnConfig cfg;
  cfg.synchronize = true;
  auto run = [&](bool trans, bool keep, std::vector<float>& dx, std::vector<float>& dwg, std::vector<float>& dwu) {
    auto dX = device_tensor<bf16>::zeros({M, K});
    auto dWg = trans ? device_tensor<float>::zeros({N, K}) : device_tensor<float>::zeros({K, N});
    auto dWu = trans ? device_tensor<float>::zeros({N, K}) : device_tensor<float>::zeros({K, N});
    auto G = device_tensor<bf16>::zeros({M, N}), U = device_tensor<bf16>::zeros({M, N}), H = device_tensor<bf16>::zeros({M, N});
    compute::GatedFfnGrads<bf16, float> out;
    out.dX = &dX;
    out.dWg = &dWg;
    out.dWu = &dWu;
    if (keep) {
      compute::gated_ffn(Xd, Wgd, Wud, H, cfg, &G, &U);
      out.gate = &G;
      out.up = &U;
    }
    if (trans)
      compute::gated_ffn_backward(dHd.view(), Xd.view(), WgTd.transpose(), WuTd.transpose(), out, cfg);
    else
      compute::gated_ffn_backward(dHd, Xd, Wgd, Wud, out, cfg);
    auto a = dX.to_host();
    auto b = dWg.to_host(), c = dWu.to_host();
    for (int i = 0; i < M * K; ++i) dx.push_back(to_float(a.data()[i]));
    for (int k = 0; k < K; ++k)
      for (int j = 0; j < N; ++j) {
        dwg.push_back(trans ? b(j, k) : b(k, j));
        dwu.push_back(trans ? c(j, k) : c(k, j));
      }
  };
  for (bool keep : {false, true}) {
    std::vector<float> want[3], got[3];
    run(false, keep, want[0], want[1], want[2]);
    run(true, keep, got[0], got[1], got[2]);
    // the sums run in the same order in either layout
    for (int i = 0; i < 3; ++i) {
      double norm = 0;
      EXPECT_EQ(want[i].size(), got[i].size());
      for (size_t e = 0; e < want[i].size(); ++e) {
        EXPECT_EQ(want[i][e], got[i][e]);
        norm += std::abs(want[i][e]);
      }
      EXPECT_TRUE(norm > 0.0);
    }
  }
  finalize();
}

TEST(cpu_gated_backward, Contracts) {
  const Layout x({4, 8}), w({8, 6}), wt({6, 8}), h({4, 6});
  auto* p = reinterpret_cast<bf16*>(0x1000);
  const TensorView<bf16> X(p, x), W(p, w), WT(p, wt), dH(p, h), short_dH(p, x);
  compute::GatedFfnGrads<bf16, bf16> out;
  EXPECT_THROW(compute::gated_ffn_backward(short_dH, X, W, W, out), compute::ValidationError);
  EXPECT_THROW(compute::gated_ffn_backward(dH, X, WT, WT, out), compute::ValidationError);             // N x K, no view
  EXPECT_THROW(compute::gated_ffn_backward(dH, X, W, WT.transpose(), out), compute::ValidationError);  // two layouts
  auto host = host_tensor<bf16>::zeros({8, 6});
  out.dWg = out.dWu = &host;
  EXPECT_THROW(compute::gated_ffn_backward(dH, X, W, W, out), compute::ValidationError);   // host memory
}

int main(int argc, char** argv) { return mini_main(argc, argv); }
