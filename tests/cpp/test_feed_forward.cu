// test_feed_forward.cu — the C++ API of the gated feed-forward product, its
// backward pass, the block quantiser and the block-scaled product, against
// double loops on the host.
// Run: test_feed_forward cpu | gpu | all
#include <cmath>
#include <vector>

#include "choreo-ir/choreo-ir.hpp"
#include "mini_test.hpp"

using namespace choreo_ir;

namespace {
using bf16 = bfloat16_t;

double silu(double g) { return g / (1 + std::exp(-g)); }
double silu_slope(double g) {
  const double s = 1 / (1 + std::exp(-g));
  return s * (1 + g * (1 - s));
}

// Relative 2-norm distance.
template <typename T>
double distance(const Tensor<T>& dev, const std::vector<double>& want) {
  auto h = dev.to_host();
  double off = 0, norm = 0;
  for (size_t i = 0; i < want.size(); ++i) {
    const double d = static_cast<double>(to_float(h.data()[i])) - want[i];
    off += d * d;
    norm += want[i] * want[i];
  }
  return std::sqrt(off / norm);
}
}  // namespace

TEST(gpu_feed_forward, ForwardAndBackward) {
  initialize();
  const int M = 70, N = 96, K = 80;
  auto X = host_tensor<bf16>::random({M, K}, -1, 1, 1);
  auto Wg = host_tensor<bf16>::random({K, N}, -0.2f, 0.2f, 2);
  auto Wu = host_tensor<bf16>::random({K, N}, -0.2f, 0.2f, 3);
  auto dH = host_tensor<bf16>::random({M, N}, -1, 1, 4);
  std::vector<double> g(M * N), u(M * N), h(M * N), dg(M * N), du(M * N), dx(M * K), dwg(K * N), dwu(K * N);
  for (int i = 0; i < M; ++i)
    for (int j = 0; j < N; ++j) {
      double a = 0, b = 0;
      for (int k = 0; k < K; ++k) {
        a += double(to_float(X(i, k))) * to_float(Wg(k, j));
        b += double(to_float(X(i, k))) * to_float(Wu(k, j));
      }
      const double d = to_float(dH(i, j));
      g[i * N + j] = a;
      u[i * N + j] = b;
      h[i * N + j] = silu(a) * b;
      dg[i * N + j] = d * b * silu_slope(a);
      du[i * N + j] = d * silu(a);
    }
  for (int i = 0; i < M; ++i)
    for (int k = 0; k < K; ++k)
      for (int j = 0; j < N; ++j) {
        dx[i * K + k] += dg[i * N + j] * to_float(Wg(k, j)) + du[i * N + j] * to_float(Wu(k, j));
        dwg[k * N + j] += dg[i * N + j] * to_float(X(i, k));
        dwu[k * N + j] += du[i * N + j] * to_float(X(i, k));
      }
  auto Xd = X.to_device(), Wgd = Wg.to_device(), Wud = Wu.to_device(), dHd = dH.to_device();
  // bf16 stores round by 2^-8 at most; the gradients' operands dG and dU once more
  auto H = compute::gated_ffn(Xd, Wgd, Wud);
  EXPECT_LE(distance(H, h), 0.004);
  auto G = device_tensor<bf16>::zeros({M, N}), U = device_tensor<bf16>::zeros({M, N});
  auto H2 = device_tensor<bf16>::zeros({M, N});
  compute::gated_ffn(Xd, Wgd, Wud, H2, compute::GatedFfnConfig(), &G, &U);
  EXPECT_LE(distance(G, g), 0.004);
  EXPECT_LE(distance(U, u), 0.004);
  // the weights as transpose views of N x K storage give the same bits
  auto WgT = host_tensor<bf16>::zeros({N, K}), WuT = host_tensor<bf16>::zeros({N, K});
  for (int k = 0; k < K; ++k)
    for (int j = 0; j < N; ++j) {
      WgT(j, k) = Wg(k, j);
      WuT(j, k) = Wu(k, j);
    }
  auto WgTd = WgT.to_device(), WuTd = WuT.to_device();
  auto H3 = device_tensor<bf16>::zeros({M, N});
  compute::gated_ffn(Xd.view(), WgTd.transpose(), WuTd.transpose(), H3.view());
  auto a = H.to_host(), b = H2.to_host(), c = H3.to_host();
  for (index_t i = 0; i < a.numel(); ++i) {
    EXPECT_EQ(to_float(a.data()[i]), to_float(b.data()[i]));
    EXPECT_EQ(to_float(a.data()[i]), to_float(c.data()[i]));
  }
  for (bool keep : {false, true}) {
    auto dX = device_tensor<bf16>::zeros({M, K}), Hb = device_tensor<bf16>::zeros({M, N});
    auto dWg = device_tensor<float>::zeros({K, N}), dWu = device_tensor<float>::zeros({K, N});
    compute::GatedFfnGrads<bf16, float> out;
    out.dX = &dX;
    out.dWg = &dWg;
    out.dWu = &dWu;
    out.H = &Hb;
    if (keep) {
      out.gate = &G;
      out.up = &U;
    }
    out.accumulate = true;  // onto zeros
    compute::GatedFfnConfig cfg;
    cfg.synchronize = true;
    compute::gated_ffn_backward(dHd, Xd, Wgd, Wud, out, cfg);
    EXPECT_LE(distance(dX, dx), 0.01);
    EXPECT_LE(distance(dWg, dwg), 0.01);
    EXPECT_LE(distance(dWu, dwu), 0.01);
    EXPECT_LE(distance(Hb, h), 0.01);
  }
  finalize();
}

TEST(gpu_feed_forward, QuantizeAndProduct) {
  initialize();
  const int M = 40, N = 150, K = 300;
  auto A = host_tensor<bf16>::random({M, K}, -1, 1, 5);
  auto B = host_tensor<float>::random({K, N}, -0.2f, 0.2f, 6);  // stored K x N: quantised transposed
  auto D = host_tensor<float>::random({M, N}, -1, 1, 7);
  std::vector<double> want(M * N);
  for (int i = 0; i < M; ++i)
    for (int j = 0; j < N; ++j) {
      double s = 0;
      for (int k = 0; k < K; ++k) s += double(to_float(A(i, k))) * B(k, j);
      want[i * N + j] = s + D(i, j);
    }
  auto Ad = A.to_device();
  auto Bd = B.to_device();
  auto Dd = D.to_device();
  auto qa = compute::quantize_block(Ad);
  for (index_t block : {1, 128}) {
    auto qb = compute::quantize_block(Bd, block, /*transpose=*/true);
    EXPECT_EQ(qb.rows, N);
    EXPECT_EQ(qb.cols, K);
    auto C = device_tensor<float>::zeros({M, N});
    compute::GEMMConfig cfg;
    cfg.synchronize = true;
    compute::gemm_block_scaled(qa, qb, C, 1.0f, 1.0f, &Dd, cfg);
    // two e4m3 roundings, 2^-4 at most and about 0.026 in the mean square each
    EXPECT_LE(distance(C, want), 0.06);
  }
  finalize();
}

TEST(cpu_feed_forward, Contracts) {
  auto X = host_tensor<bf16>::zeros({4, 8});
  auto W = host_tensor<bf16>::zeros({8, 6});
  auto H = host_tensor<bf16>::zeros({4, 6});
  EXPECT_THROW(compute::gated_ffn(X, W, W, H), compute::ValidationError);   // host tensors
  const Layout x({4, 8}), w({8, 6}), w2({7, 6}), h({4, 5});
  auto* p = reinterpret_cast<bf16*>(0x1000);
  const TensorView<bf16> Xv(p, x), Wv(p, w), W2(p, w2), Hv(p, h);
  EXPECT_THROW(compute::gated_ffn(Xv, Wv, W2, Hv), compute::ValidationError);
  EXPECT_THROW(compute::gated_ffn(Xv, Wv, Wv, Hv), compute::ValidationError);
  EXPECT_THROW(compute::quantize_block(X, 64), compute::ValidationError);
  EXPECT_THROW(compute::BlockScaled(4, 4, 0), compute::ValidationError);
}

int main(int argc, char** argv) { return mini_main(argc, argv); }
