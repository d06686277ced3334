// The gated scan and its gradient where the copies of one tile never come: the wait for them runs out, the kernel ends, its results are NaNs from there on, the
// status says so, and the same call on the same workspace is right once the copies are made.  Compiled with -DTB200_TEST_HOOKS and a
// limit of 65536 polls; all copies that are made stay in bounds.
#include "../../thrust_b200/csrc/abi_gated.cu"

#include <cmath>
#include <cstdio>
#include <vector>

void tb200_abi::call_begins(const void*) {}

static int failures = 0;
#define CHECK(cond) do { if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, #cond); ++failures; } } while (0)

int main() {
  const size_t n = 3000, dim = 128;
  std::vector<float> h(n * dim);
  for (size_t i = 0; i < h.size(); ++i) h[i] = (float)(i * 2654435761u % 1000) / 1000.f - 0.5f;
  float *x, *gate, *out, *last, *dx, *dgate, *dh0;
  void* ws;
  const size_t bytes = n * dim * 4;
  for (float** p : {&x, &gate, &out, &dx, &dgate}) CHECK(cudaMalloc(p, bytes) == cudaSuccess);
  for (float** p : {&last, &dh0}) CHECK(cudaMalloc(p, 2 * dim * 4) == cudaSuccess);
  CHECK(cudaMemcpy(x, h.data(), bytes, cudaMemcpyHostToDevice) == cudaSuccess);
  CHECK(cudaMemcpy(gate, h.data(), bytes, cudaMemcpyHostToDevice) == cudaSuccess);
  for (size_t batch : {(size_t)1, (size_t)2}) {      // clusters of CTAs
    size_t need = 0;
    CHECK(tb200_gated_scan(nullptr, dim, nullptr, dim, nullptr, nullptr, 0, batch, n, dim, TB200_F32, nullptr, nullptr, nullptr, &need, nullptr) == 0);
    CHECK(cudaMalloc(&ws, need) == cudaSuccess);
    auto status = [&] { tb200::ws_header head; CHECK(cudaDeviceSynchronize() == cudaSuccess); CHECK(cudaMemcpy(&head, ws, sizeof(head), cudaMemcpyDeviceToHost) == cudaSuccess); return head.error; };
    auto back = [&](const float* p) { std::vector<float> v(n * dim); CHECK(cudaMemcpy(v.data(), p, bytes, cudaMemcpyDeviceToHost) == cudaSuccess); return v; };
    auto forward = [&] { return tb200_gated_scan(x, dim, gate, dim, nullptr, nullptr, 0, batch, n, dim, TB200_F32, out, last, ws, &need, nullptr); };
    auto backward = [&] {
      return tb200_gated_scan_grad(x, dim, x, dim, gate, dim, out, dim, nullptr, nullptr, nullptr, 0, batch, n, dim, TB200_F32, dx, dgate, dh0, ws, &need, nullptr);
    };
    auto withhold = [&](unsigned on) { CHECK(cudaMemcpyToSymbol(withhold_copies, &on, 4) == cudaSuccess); };
    withhold(0);
    CHECK(forward() == 0);
    CHECK(status() == 0);
    const std::vector<float> good = back(out);
    double state = 0;
    for (size_t r = 0; r < n / batch; ++r) { const double keep = 1 / (1 + std::exp(-(double)h[r * dim])); state = keep * state + (1 - keep) * h[r * dim]; CHECK(std::fabs(good[r * dim] - state) < 1e-5); }
    CHECK(backward() == 0);
    CHECK(status() == 0);
    const std::vector<float> good_dx = back(dx);
    withhold(1);
    CHECK(forward() == 0);
    CHECK(status() == tb200::ERR_LOOKBACK_TIMEOUT);
    std::vector<float> bad = back(out);
    size_t nans = 0;
    for (size_t i = 0; i < bad.size(); ++i) { nans += std::isnan(bad[i]); CHECK(std::isnan(bad[i]) || bad[i] == good[i]); }
    CHECK(nans > 0 && std::isnan(bad[(n - 1) * dim]) && bad[0] == good[0]);
    CHECK(backward() == 0);
    CHECK(status() == tb200::ERR_LOOKBACK_TIMEOUT);
    bad = back(dx);
    CHECK(std::isnan(bad[0]));
    withhold(0);
    CHECK(forward() == 0);
    CHECK(status() == 0);
    CHECK(back(out) == good);
    CHECK(backward() == 0);
    CHECK(status() == 0);
    CHECK(back(dx) == good_dx);
    CHECK(cudaFree(ws) == cudaSuccess);
  }
  if (!failures) std::printf("ok\n");
  return failures != 0;
}
