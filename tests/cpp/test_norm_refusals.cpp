// Tables of the ranks' buffers that the C++ front end's norms refuse, with an exception and nothing read from them.
#include <cmath>

#include "parity_harness.hpp"

int main() {
  int ndev = 0;
  if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1) { std::printf("no GPU\n"); return 2; }
  HIPCHK(hipSetDevice(0));
  hipStream_t stream;
  HIPCHK(hipStreamCreate(&stream));
  {
    const size_t rows = 4, cols = 64, n = rows * cols;
    Al::amd::World world(1, stream);
    Al::amd::Communicator &comm = world.comm(0);
    DevBuf<float> in(n), out(n), rstd(rows), scales(rows);
    DevBuf<uint8_t> q(n);
    in.up(std::vector<float>(n, 1.0f));
    rstd.up(std::vector<float>(rows, 1.0f));
    const float *const one[1] = {in.p}, *const none[1] = {nullptr}, *const *const no_table = nullptr;
    const float *const w = nullptr;
    auto refused = [&](const float *const *table, int ranks, size_t r) {
      int threw = 0;
      try {
        Al::amd::rms_norm(out.p, cols, (float *)nullptr, (const float *)nullptr, 0, table, ranks, cols, w, (float *)nullptr, r, cols, 1e-6f, comm);
      } catch (const Al::al_exception &) { ++threw; }
      try {
        Al::amd::rms_norm_e4m3(q.p, cols, scales.p, 0, (float *)nullptr, (const float *)nullptr, 0, table, ranks, cols, w, (float *)nullptr, r, cols,
                               1e-6f, comm);
      } catch (const Al::al_exception &) { ++threw; }
      try {
        Al::amd::rms_norm_grad(out.p, cols, table, ranks, cols, (const float *)in.p, cols, (const float *)nullptr, 0, (const float *)rstd.p, w,
                               (float *)nullptr, r, cols, nullptr, comm);
      } catch (const Al::al_exception &) { ++threw; }
      return threw;
    };
    EXPECT(refused(no_table, 1, rows) == 3, "no table");
    EXPECT(refused(no_table, 1 << 30, rows) == 3, "no table of many");
    EXPECT(refused(one, 1 << 30, rows) == 3, "a table shorter than the number of ranks by far");
    EXPECT(refused(one, ALAMD_MAX_RANKS + 1, rows) == 3, "too many ranks");
    EXPECT(refused(one, 0, rows) == 3, "no ranks");
    EXPECT(refused(one, -1, rows) == 3, "fewer than no ranks");
    EXPECT(refused(none, 1, rows) == 3, "a null buffer");
    EXPECT(refused(no_table, 1, 0) == 0, "nothing to do");
    EXPECT(refused(one, 1, rows) == 0, "one rank");
    HIPCHK(hipStreamSynchronize(stream));
    EXPECT(std::fabs(out.down()[n - 1]) < 1e-5, "gradient of a row of equal elements");
  }
  HIPCHK(hipStreamDestroy(stream));
  std::printf("%d checks, %d failures\n%s\n", g_checks.load(), g_fail.load(), g_fail.load() ? "FAILED" : "PASSED");
  return g_fail.load() ? 1 : 0;
}
