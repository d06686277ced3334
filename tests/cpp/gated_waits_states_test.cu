// The states and their gradients (d_last, d_dh0) of the gated scan where the copies of one tile, or the pairs of one CTA, never come: a sequence that was not
// walked to its end has no finite state behind it.  Compiled with -DTB200_TEST_HOOKS and a limit of 65536 polls; all copies that are made stay in bounds.
#include "../../thrust_b200/csrc/abi_gated.cu"

#include <cmath>
#include <cstdio>
#include <vector>

void tb200_abi::call_begins(const void*) {}

static int failures = 0;
#define CHECK(cond) do { if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, #cond); ++failures; } } while (0)

int main() {
  const size_t most = 3000, dim = 128;
  std::vector<float> h(most * dim);
  for (size_t i = 0; i < h.size(); ++i) h[i] = (float)(i * 2654435761u % 1000) / 1000.f - 0.5f;
  float *x, *out, *last, *dx, *dgate, *dh0;
  long long* offsets;
  void* ws;
  const size_t bytes = most * dim * 4;
  for (float** p : {&x, &out, &dx, &dgate}) CHECK(cudaMalloc(p, bytes) == cudaSuccess);
  for (float** p : {&last, &dh0}) CHECK(cudaMalloc(p, 2 * dim * 4) == cudaSuccess);
  CHECK(cudaMalloc(&offsets, 3 * 8) == cudaSuccess);
  CHECK(cudaMemcpy(x, h.data(), bytes, cudaMemcpyHostToDevice) == cudaSuccess);
  // one sequence, two of equal lengths, and two packed ones of which one lies in the first window of any cluster; of 1100 rows window 1 is the scan's last one where
  // 16 CTAs walk together, of 600 rows its gradient's
  struct shape { size_t n, batch; bool packed; long long offsets[3]; };
  for (const shape& s : {shape{3000, 1, false, {}}, shape{3000, 2, false, {}}, shape{3000, 1, true, {0, 3000}}, shape{3000, 2, true, {0, 20, 3000}}, shape{3000, 2, true, {0, 2980, 3000}},
                         shape{1100, 1, false, {}}, shape{1100, 1, true, {0, 1100}}, shape{600, 1, false, {}}, shape{600, 1, true, {0, 600}}}) {
    const size_t n = s.n, batch = s.batch;
    CHECK(cudaMemcpy(offsets, s.offsets, 24, cudaMemcpyHostToDevice) == cudaSuccess);
    const void* const cut = s.packed ? offsets : nullptr;
    size_t need = 0;
    CHECK(tb200_gated_scan(nullptr, dim, nullptr, dim, nullptr, cut, TB200_I64, batch, n, dim, TB200_F32, nullptr, nullptr, nullptr, &need, nullptr) == 0);
    CHECK(cudaMalloc(&ws, need) == cudaSuccess);
    auto status = [&] { tb200::ws_header head; CHECK(cudaDeviceSynchronize() == cudaSuccess); CHECK(cudaMemcpy(&head, ws, sizeof(head), cudaMemcpyDeviceToHost) == cudaSuccess); return head.error; };
    auto back = [&](const float* p) { std::vector<float> v(batch * dim); CHECK(cudaMemcpy(v.data(), p, v.size() * 4, cudaMemcpyDeviceToHost) == cudaSuccess); return v; };
    auto forward = [&] { return tb200_gated_scan(x, dim, x, dim, nullptr, cut, TB200_I64, batch, n, dim, TB200_F32, out, last, ws, &need, nullptr); };
    auto backward = [&] {
      return tb200_gated_scan_grad(x, dim, x, dim, x, dim, out, dim, nullptr, nullptr, cut, TB200_I64, batch, n, dim, TB200_F32, dx, dgate, dh0, ws, &need, nullptr);
    };
    auto withhold = [&](unsigned copies, unsigned pairs) {
      CHECK(cudaMemcpyToSymbol(withhold_copies, &copies, 4) == cudaSuccess && cudaMemcpyToSymbol(withhold_pairs, &pairs, 4) == cudaSuccess);
    };
    withhold(0, 0);
    CHECK(forward() == 0 && status() == 0);
    const std::vector<float> good = back(last);
    CHECK(backward() == 0 && status() == 0);
    const std::vector<float> good_dh0 = back(dh0);
    for (int what = 0; what < 2; ++what) {      // the copies, the pairs
      withhold(what == 0, what == 1);
      // a state is NaN or what it should be; of the sequence that reaches over most of the rows it is NaN.  (600 rows are one window of the scan's.)
      const size_t longest = s.packed && batch == 2 && s.offsets[1] == 20 ? 1 : 0;
      auto lost = [&](const std::vector<float>& got, const std::vector<float>& want) {
        size_t wrong = 0;
        for (size_t i = 0; i < got.size(); ++i) wrong += !(std::isnan(got[i]) || (s.packed && got[i] == want[i] && i / dim != longest));
        return wrong == 0;
      };
      if (n > 600) {
        CHECK(forward() == 0 && status() == tb200::ERR_LOOKBACK_TIMEOUT);
        CHECK(lost(back(last), good));
      }
      CHECK(backward() == 0 && status() == tb200::ERR_LOOKBACK_TIMEOUT);
      CHECK(lost(back(dh0), good_dh0));
      withhold(0, 0);
      CHECK(forward() == 0 && status() == 0 && back(last) == good);
      CHECK(backward() == 0 && status() == 0 && back(dh0) == good_dh0);
    }
    CHECK(cudaFree(ws) == cudaSuccess);
  }
  if (!failures) std::printf("ok\n");
  return failures != 0;
}
