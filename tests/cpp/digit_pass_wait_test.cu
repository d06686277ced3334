// The general sort where tile 0 of the digit passes never publishes its counts: the wait for them runs out, status 1 is left, no pass writes outside the
// arrays, and what they hold are items of the input, whatever lay in the alternate buffers; the next call on the same workspace sorts.  Compiled with
// -DTB200_TEST_HOOKS and a limit of 65536 polls.
// Every array has as much room again on both sides as it is long, so that what should not be written can be looked at.
#include <cstdint>
#include <cstdio>
#include <algorithm>
#include <numeric>
#include <vector>

#include "thrust_b200/radix_sort.cuh"

static int failures = 0;
#define CHECK(cond) do { if (!(cond)) { std::printf("FAILED line %d: %s\n", __LINE__, #cond); ++failures; } } while (0)

template <class T> struct roomy {
  size_t n;
  T* all;
  explicit roomy(size_t count) : n(count) { CHECK(cudaMalloc(&all, 3 * n * sizeof(T)) == cudaSuccess); CHECK(cudaMemset(all, 0xff, 3 * n * sizeof(T)) == cudaSuccess); }
  ~roomy() { cudaFree(all); }
  T* at() const { return all + n; }
  std::vector<T> back() const { std::vector<T> v(3 * n); CHECK(cudaMemcpy(v.data(), all, 3 * n * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess); return v; }
  bool kept() const {
    const std::vector<T> v = back();
    for (size_t i = 0; i < n; ++i) if (v[i] != (T)~(T)0 || v[2 * n + i] != (T)~(T)0) return false;
    return true;
  }
};

template <class UK, class UV, bool HAS_V> static void sorts(size_t n) {
  std::vector<UK> h(n);
  for (size_t i = 0; i < n; ++i) h[i] = (UK)((i + 1) * 0x9e3779b97f4a7c15ull >> 17);
  std::vector<UV> v(n);
  std::iota(v.begin(), v.end(), (UV)0);
  roomy<UK> ka(n), kb(n);
  roomy<UV> va(n), vb(n);
  void* ws;
  const size_t bytes = tb200::radix_workspace_bytes<sizeof(UK), HAS_V ? sizeof(UV) : 0>(n);
  CHECK(cudaMalloc(&ws, bytes) == cudaSuccess);
  tb200::key_coding coding;
  coding.kind = tb200::KEY_UNSIGNED;
  coding.descending = 0;
  for (unsigned withheld : {1u, 0u}) {
    tb200::test_hook_flags() = withheld;
    CHECK(cudaMemcpy(ka.at(), h.data(), n * sizeof(UK), cudaMemcpyHostToDevice) == cudaSuccess && cudaMemcpy(va.at(), v.data(), n * sizeof(UV), cudaMemcpyHostToDevice) == cudaSuccess);
    CHECK((tb200::radix_sort_async<UK, UV, HAS_V>(ka.at(), kb.at(), va.at(), vb.at(), n, coding, 0, 8 * (int)sizeof(UK), ws, 0)) == cudaSuccess);
    unsigned status = 77;
    CHECK(cudaDeviceSynchronize() == cudaSuccess && cudaMemcpy(&status, ws, 4, cudaMemcpyDeviceToHost) == cudaSuccess);
    CHECK(status == (withheld ? tb200::ERR_LOOKBACK_TIMEOUT : tb200::ERR_NONE));
    CHECK(ka.kept() && kb.kept() && va.kept() && vb.kept());
    if (withheld) {      // some items twice, others not at all, but none that is no item: what a caller looks up by them is there
      const std::vector<UK> k = ka.back();
      const std::vector<UV> o = va.back();
      size_t odd = 0;
      for (size_t i = 0; i < n; ++i) odd += HAS_V ? o[n + i] >= n || k[n + i] != h[o[n + i]] : k[n + i] == (UK)~(UK)0;
      CHECK(odd == 0);
    }
  }
  std::vector<UV> order = v;
  std::stable_sort(order.begin(), order.end(), [&](UV a, UV b) { return h[a] < h[b]; });
  const std::vector<UK> k = ka.back();
  const std::vector<UV> o = va.back();
  bool same = true;
  for (size_t i = 0; i < n; ++i) same = same && k[n + i] == h[order[i]] && (!HAS_V || o[n + i] == order[i]);
  CHECK(same);
  CHECK(cudaFree(ws) == cudaSuccess);
}

int main() {
  sorts<uint32_t, uint32_t, true>(600011);      // past what the sorts of one launch take
  sorts<uint64_t, uint32_t, true>(600011);
  sorts<uint16_t, uint32_t, true>(600011);
  sorts<uint32_t, uint32_t, false>(600011);
  if (!failures) std::printf("all checks passed\n");
  return failures != 0;
}
