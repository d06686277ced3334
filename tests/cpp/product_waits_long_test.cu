// As product_waits_test.cu, for contractions that are cut into groups (f16: of 4096), between which the writers add one half of tensor memory to the other: the copies of one
// tile never come, from its first stage or from the second group on, in the forward product of rows of 8192 and in the gradient of an expert's matrix over 5000 rows.  Compiled with -DTB200_TEST_HOOKS and a limit of 65536 polls;
// all copies that are made stay in bounds.
#include "../../thrust_b200/csrc/abi_product.cu"

#include <cmath>
#include <cstdio>
#include <vector>

void tb200_abi::call_begins(const void*) {}

static int failures = 0;
#define CHECK(cond) do { if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, #cond); ++failures; } } while (0)

static float value(unsigned short bits) { __half h; memcpy(&h, &bits, 2); return __half2float(h); }

int main() {
  const size_t n = 6000, experts = 3, in = 8192, out = 1280;
  const int offsets[4] = {0, 5000, 5000, 5990};
  std::vector<unsigned short> hx(n * in), hw(experts * in * out);
  for (size_t i = 0; i < hx.size(); ++i) hx[i] = (unsigned short)(0x3800 + (i * 2654435761u >> 20) % 1024 + ((i * 40503u >> 3) & 1 ? 0x8000 : 0));
  for (size_t i = 0; i < hw.size(); ++i) hw[i] = (unsigned short)(0x1000 + (i * 2246822519u >> 20) % 1024 + ((i * 69069u >> 4) & 1 ? 0x8000 : 0));
  void *x, *w, *o, *y, *dx, *dw, *ws;
  CHECK(cudaMalloc(&x, n * in * 2) == cudaSuccess && cudaMalloc(&w, experts * in * out * 2) == cudaSuccess && cudaMalloc(&o, sizeof(offsets)) == cudaSuccess);
  CHECK(cudaMalloc(&y, n * out * 2) == cudaSuccess && cudaMalloc(&dx, n * in * 2) == cudaSuccess && cudaMalloc(&dw, experts * in * out * 2) == cudaSuccess);
  CHECK(cudaMemcpy(x, hx.data(), hx.size() * 2, cudaMemcpyHostToDevice) == cudaSuccess && cudaMemcpy(w, hw.data(), hw.size() * 2, cudaMemcpyHostToDevice) == cudaSuccess);
  CHECK(cudaMemcpy(o, offsets, sizeof(offsets), cudaMemcpyHostToDevice) == cudaSuccess);
  size_t need = 0;
  auto forward = [&](void* room) {
    return tb200_expert_product(x, in, o, TB200_I32, w, in * out, out, 0, nullptr, nullptr, 0, TB200_ACT_NONE, n, experts, in, out, TB200_F16, y, nullptr, room, &need, nullptr);
  };
  auto backward = [&](void* room) {
    return tb200_expert_product_grad(y, out, x, in, o, TB200_I32, w, in * out, out, 0, n, experts, in, out, TB200_F16, TB200_F16, 0, dx, dw, nullptr, room, &need, nullptr);
  };
  CHECK(forward(nullptr) == 0);
  const size_t first = need;
  CHECK(backward(nullptr) == 0);
  need = need > first ? need : first;
  CHECK(cudaMalloc(&ws, need) == cudaSuccess);
  auto status = [&] { tb200::ws_header head; CHECK(cudaDeviceSynchronize() == cudaSuccess); CHECK(cudaMemcpy(&head, ws, sizeof(head), cudaMemcpyDeviceToHost) == cudaSuccess); return head.error; };
  auto withhold = [&](unsigned on) { CHECK(cudaMemcpyToSymbol(withhold_boxes, &on, 4) == cudaSuccess); };
  auto rows = [&](const void* p, size_t items) {
    std::vector<unsigned short> h(items);
    CHECK(cudaMemcpy(h.data(), p, items * 2, cudaMemcpyDeviceToHost) == cudaSuccess);
    std::vector<float> v(items);
    for (size_t i = 0; i < items; ++i) v[i] = value(h[i]);
    return v;
  };
  auto matrix = [&] { return rows(dw, experts * in * out); };
  withhold(0);
  CHECK(forward(ws) == 0);
  CHECK(status() == 0);
  const std::vector<float> good = rows(y, n * out);
  for (size_t r : {(size_t)0, (size_t)1499, (size_t)5000, (size_t)5989})
    for (size_t c : {(size_t)0, (size_t)700, out - 1}) {
      size_t e = 0;
      while (r >= (size_t)offsets[e + 1]) ++e;
      double sum = 0, size = 0;
      for (size_t i = 0; i < in; ++i) { const double t = (double)value(hx[r * in + i]) * value(hw[(e * in + i) * out + c]); sum += t; size += std::fabs(t); }
      CHECK(std::fabs(good[r * out + c] - sum) < std::fabs(sum) / 1024 + size * 1e-4);
    }
  CHECK(good[5995 * out] == 0);
  CHECK(backward(ws) == 0);
  CHECK(status() == 0);
  const std::vector<float> good_dx = rows(dx, n * in), good_dw = matrix();
  for (unsigned from : {1u, 35u}) {
    withhold(from);
    CHECK(forward(ws) == 0);
    CHECK(status() == tb200::ERR_LOOKBACK_TIMEOUT);
    std::vector<float> bad = rows(y, n * out);
    size_t nans = 0;
    for (size_t i = 0; i < bad.size(); ++i) { nans += std::isnan(bad[i]); CHECK(std::isnan(bad[i]) || bad[i] == good[i]); }
    CHECK(nans > 0 && nans < bad.size() / 4);
    withhold(0);
    CHECK(forward(ws) == 0);
    CHECK(status() == 0);
    withhold(from);
    CHECK(backward(ws) == 0);
    CHECK(status() == tb200::ERR_LOOKBACK_TIMEOUT);
    bad = matrix();
    nans = 0;
    for (size_t i = 0; i < bad.size(); ++i) { nans += std::isnan(bad[i]); CHECK(std::isnan(bad[i]) || bad[i] == good_dw[i]); }
    CHECK(nans > 0 && nans < bad.size() / 4);
    withhold(0);
    CHECK(backward(ws) == 0);
    CHECK(status() == 0);
    CHECK(rows(dx, n * in) == good_dx && matrix() == good_dw && rows(y, n * out) == good);
  }
  if (!failures) std::printf("ok\n");
  return failures != 0;
}
