// The operators that follow a training step's two kinds of Allreduce, through the C++ front end: a layer split over
// two logical ranks goes through the norm and its backward pass, the weight's gradients of the two ranks are
// averaged by an Allreduce, their norm is taken and they are clipped.  Against the formulas in double.
#include <cmath>

#include "parity_harness.hpp"

int main() {
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1) { std::printf("no GPU\n"); return 2; }
  HIPCHK(hipSetDevice(0));
  hipStream_t stream;
  HIPCHK(hipStreamCreate(&stream));
  {
    const int P = 2;
    const size_t rows = 33, cols = 1027, n = rows * cols;
    const float eps = 1e-5f, max_norm = 0.25f;
    Al::amd::World world(P, stream);
    std::vector<std::vector<float>> part, dy;
    std::vector<std::unique_ptr<DevBuf<float>>> dpart, ddy, dweight;
    for (int r = 0; r < P; ++r) {
      part.push_back(gen<float>(n, ALO_DIST_UNIFORM_PM1, 10 + r));
      dy.push_back(gen<float>(n, ALO_DIST_UNIFORM_PM1, 20 + r));
      dpart.emplace_back(new DevBuf<float>(n));
      ddy.emplace_back(new DevBuf<float>(n));
      dweight.emplace_back(new DevBuf<float>(cols));
      dpart.back()->up(part.back());
      ddy.back()->up(dy.back());
    }
    const std::vector<float> res = gen<float>(n, ALO_DIST_UNIFORM_PM1, 30), w = gen<float>(cols, ALO_DIST_UNIFORM_09_11, 31);
    DevBuf<float> dres(n), dw(cols), out(n), sum(n), rstd(rows), dx(n), scales(rows), norm(1);
    DevBuf<uint8_t> q(n), space(Al::amd::rms_norm_grad_workspace(rows, cols)), norm_space(Al::amd::TensorList::workspace_bytes);
    dres.up(res);
    dw.up(w);
    const float *ins[P] = {dpart[0]->p, dpart[1]->p};
    Al::amd::Communicator &comm = world.comm(0);
    Al::amd::rms_norm(out.p, cols, sum.p, (const float *)dres.p, cols, ins, P, cols, (const float *)dw.p, rstd.p, rows, cols, eps, comm);
    Al::amd::rms_norm_e4m3(q.p, cols, scales.p, 0, (float *)nullptr, (const float *)dres.p, cols, ins, P, cols, (const float *)dw.p,
                           nullptr, rows, cols, eps, comm);
    for (int r = 0; r < P; ++r) {
      const float *one[1] = {ddy[r]->p};
      Al::amd::rms_norm_grad(dx.p, cols, one, 1, cols, (const float *)sum.p, cols, (const float *)nullptr, 0, rstd.p,
                             (const float *)dw.p, dweight[r]->p, rows, cols, space.p, world.comm(r));
    }
    for (int r = 0; r < P; ++r) Al::Allreduce<Backend>(dweight[r]->p, cols, Op::avg, world.comm(r));
    Al::amd::TensorList grads;
    grads.add(dweight[0]->p, cols);
    grads.make();
    grads.clip_global_norm(norm.p, max_norm, 1e-6f, norm_space.p, comm);
    HIPCHK(hipStreamSynchronize(stream));

    // the same in double; fp32 sums of a thousand terms of order one are off by far less than 1e-4 of the result
    const auto got_out = out.down(), got_sum = sum.down(), got_dx = dx.down(), got_dw = dweight[0]->down(), got_scales = scales.down();
    const auto got_q = q.down();
    std::vector<double> want_dw(cols, 0.0);
    for (size_t i = 0; i < rows; ++i) {
      double ss = 0, amax = 0;
      std::vector<double> s(cols), g(cols);
      for (size_t j = 0; j < cols; ++j) {
        s[j] = (double)part[0][i * cols + j] + part[1][i * cols + j] + res[i * cols + j];
        ss += s[j] * s[j];
      }
      const double r = 1 / std::sqrt(ss / cols + eps);
      double dot = 0;
      for (size_t j = 0; j < cols; ++j) {
        const double y = s[j] * r * w[j];
        amax = std::max(amax, std::fabs(y));
        EXPECT(std::fabs(got_out[i * cols + j] - y) < 1e-5, "out %zu %zu", i, j);
        EXPECT(std::fabs(got_sum[i * cols + j] - s[j]) < 1e-6, "sum %zu %zu", i, j);
        for (int k = 0; k < P; ++k) want_dw[j] += (double)dy[k][i * cols + j] * s[j] * r / P;
        g[j] = (double)dy[P - 1][i * cols + j] * w[j];
        dot += g[j] * s[j] * r;
      }
      EXPECT(std::fabs(got_scales[i] * 448 - amax) < 1e-5 * amax, "scale of row %zu", i);
      bool top = false;
      for (size_t j = 0; j < cols; ++j) {
        EXPECT(std::fabs(got_dx[i * cols + j] - r * (g[j] - s[j] * r * dot / cols)) < 1e-4, "dx %zu %zu", i, j);
        top = top || (got_q[i * cols + j] & 0x7f) == 0x7e;  // 448
      }
      EXPECT(top, "row %zu has no element of the largest value", i);
    }
    double total = 0;
    for (double d : want_dw) total += d * d;
    total = std::sqrt(total);
    EXPECT(std::fabs(norm.down()[0] / total - 1) < 1e-5, "norm %g, expected %g", norm.down()[0], total);
    EXPECT(total > max_norm, "the step is clipped");
    for (size_t j = 0; j < cols; ++j)
      EXPECT(std::fabs(got_dw[j] - want_dw[j] * max_norm / (total + 1e-6)) < 1e-4 * max_norm, "clipped gradient %zu", j);

    // errors arrive as exceptions
    bool threw = false;
    try {
      Al::amd::rms_norm(out.p, cols - 1, sum.p, (const float *)dres.p, cols, ins, P, cols, (const float *)dw.p, rstd.p, rows, cols, eps,
                        comm);
    } catch (const Al::al_exception &) { threw = true; }
    EXPECT(threw, "rows that overlap must throw");
    threw = false;
    try {
      Al::amd::TensorList twice;
      twice.add(out.p, 64);
      twice.add(out.p + 63, 64);
      twice.make();
    } catch (const Al::al_exception &) { threw = true; }
    EXPECT(threw, "a buffer that is in a list twice must throw");
    threw = false;
    try {
      Al::amd::TensorList unmade;
      unmade.global_norm(norm.p, norm_space.p, comm);
    } catch (const Al::al_exception &) { threw = true; }
    EXPECT(threw, "a list that was not made must throw");
  }
  HIPCHK(hipStreamDestroy(stream));
  std::printf("%d checks, %d failures\n%s\n", g_checks.load(), g_fail.load(), g_fail.load() ? "FAILED" : "PASSED");
  return g_fail.load() ? 1 : 0;
}
