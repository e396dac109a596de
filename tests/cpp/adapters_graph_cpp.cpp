// A C++ host program that captures a step with adapters once, for any batch within the context's bounds
// (include/fqa_step.hpp: Pack, PlanAdapters with bounded = true, AddAdapters on a bf16 and on an fp32
// projection), and replays it for batches of other requests, lengths and adapters.  Inputs are small whole
// numbers, so that every sum is exact and each output is the integer result rounded once.  Prints "ok" or
// what differs.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "../../include/fqa_step.hpp"

static uint16_t Bf16(float f) {
  uint32_t b;
  std::memcpy(&b, &f, 4);
  return (uint16_t)((b + 0x7fff + ((b >> 16) & 1)) >> 16);
}
static int I(uint16_t h) {
  const uint32_t b = (uint32_t)h << 16;
  float f;
  std::memcpy(&f, &b, 4);
  return (int)f;
}
template <class T>
static void Copy(const fqa::DeviceBuffer<T>& d, const std::vector<T>& v, hipStream_t s) {
  fqa::HipCheck(hipMemcpyAsync(d.D(), v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice, s), "copy");
}

int main() try {
  const int K = 256, N = 384, F = 192, R = 32, n_adapters = 3, max_rows = 400, slots = 8;
  std::mt19937 rng(9);
  const auto random = [&](size_t n, int most) {
    std::vector<uint16_t> v(n);
    for (auto& x : v) x = Bf16((float)((int)(rng() % (2 * most + 1)) - most));
    return v;
  };
  fqa::StepContext ctx(max_rows, slots, 512, 1024);
  const std::vector<uint16_t> a = random((size_t)n_adapters * 2 * R * K, 1), b = random((size_t)n_adapters * N * R, 2);
  const std::vector<uint16_t> fa = random((size_t)n_adapters * R * K, 1), fb = random((size_t)n_adapters * F * R, 2);
  const std::vector<float> scale = {1.f, -1.f, 2.f};
  const std::vector<int32_t> rank = {32, 5, 16};
  fqa::DeviceBuffer<uint16_t> da(a.size()), db(b.size()), dfa(fa.size()), dfb(fb.size());
  fqa::DeviceBuffer<uint16_t> dx((size_t)max_rows * K), dy((size_t)max_rows * N);
  fqa::DeviceBuffer<float> dz((size_t)max_rows * F), ds(scale.size());
  fqa::DeviceBuffer<int32_t> dr(rank.size()), di(slots);
  hipStream_t stream;
  fqa::HipCheck(hipStreamCreate(&stream), "stream");
  Copy(da, a, stream);
  Copy(db, b, stream);
  Copy(dfa, fa, stream);
  Copy(dfb, fb, stream);
  Copy(ds, scale, stream);
  Copy(dr, rank, stream);
  const fqa_lora w{da.D(), db.D(), ds.D(), dr.D(), n_adapters, R, K, 2, {256, N, 0, 0}};
  const fqa_lora wf{dfa.D(), dfb.D(), ds.D(), dr.D(), n_adapters, R, K, 1, {F, 0, 0, 0}};
  const int64_t bytes = std::max(ctx.AdapterWorkspaceBytes(w), ctx.AdapterWorkspaceBytes(wf));
  fqa::DeviceBuffer<unsigned char> ws((size_t)bytes);
  const auto step = [&](bool bounded) {
    ctx.PlanAdapters(di.D(), n_adapters, stream, bounded);
    ctx.AddAdapters(w, dx.D(), K, dy.D(), N, false, ws.D(), bytes, stream);
    ctx.AddAdapters(wf, dx.D(), K, dz.D(), F, true, ws.D(), bytes, stream);
  };
  hipGraph_t graph = nullptr;
  hipGraphExec_t exec = nullptr;
  fqa::HipCheck(hipStreamSynchronize(stream), "sync");
  fqa::HipCheck(hipStreamBeginCapture(stream, hipStreamCaptureModeThreadLocal), "begin capture");
  ctx.Pack(stream);
  step(true);
  fqa::HipCheck(hipStreamEndCapture(stream, &graph), "end capture");
  fqa::HipCheck(hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0), "instantiate");

  const std::vector<std::vector<int>> batches = {
      {1}, {1, 140, 1, 1, 20, 1}, {1, 1, 1, 1, 1, 1, 1, 1}, {400}, {}, {130, 128, 127, 1, 1}, {2, 1, 3}};
  int all = 0;
  for (int turn = 0; turn < 2 * (int)batches.size(); ++turn) {
    const std::vector<int>& lens = batches[turn % batches.size()];
    const bool replay = turn % 3 != 2;  // eager steps between the replays
    fqa::BatchInput in;
    int page = 0, rows = 0;
    std::vector<int32_t> ids;
    for (const int n : lens) {
      in.computed.push_back((int)(rng() % 60));
      in.n_new.push_back(n);
      in.block_tables.emplace_back();
      for (int k = 0; k < (in.computed.back() + n + 15) / 16; ++k) in.block_tables.back().push_back(page++);
      ids.push_back((int)(rng() % (n_adapters + 2)) - 1);  // -1 and n_adapters: none
      rows += n;
    }
    const auto x = random((size_t)max_rows * K, 2), y = random((size_t)max_rows * N, 100);
    std::vector<float> z((size_t)max_rows * F);
    for (auto& v : z) v = (float)((int)(rng() % 2001) - 1000);
    if (!ids.empty()) Copy(di, ids, stream);
    Copy(dx, x, stream);
    Copy(dy, y, stream);
    Copy(dz, z, stream);
    if (replay) {
      ctx.UploadBatch(in, stream);
      fqa::HipCheck(hipGraphLaunch(exec, stream), "launch");
    } else {
      ctx.PrepareInputs(in, stream);
      step(false);
    }
    std::vector<uint16_t> gy(y.size());
    std::vector<float> gz(z.size());
    fqa::HipCheck(hipMemcpyAsync(gy.data(), dy.D(), gy.size() * 2, hipMemcpyDeviceToHost, stream), "copy");
    fqa::HipCheck(hipMemcpyAsync(gz.data(), dz.D(), gz.size() * 4, hipMemcpyDeviceToHost, stream), "copy");
    fqa::HipCheck(hipStreamSynchronize(stream), "sync");
    std::vector<int> of(max_rows, -1);  // rows past the batch have none
    for (size_t r = 0, row = 0; r < lens.size(); ++r)
      for (int k = 0; k < lens[r]; ++k) of[row++] = ids[r] >= 0 && ids[r] < n_adapters ? ids[r] : -1;
    for (int row = 0; row < max_rows; ++row) {
      const int g = of[row];
      std::vector<int> h(3 * R, 0);  // the bf16 projection's two slices, the fp32 one's
      if (g >= 0)
        for (int j = 0; j < 3 * R; ++j)
          if (j % R < rank[g])
            for (int k = 0; k < K; ++k)
              h[j] += I(x[(size_t)row * K + k]) *
                      I(j < 2 * R ? a[((size_t)g * 2 * R + j) * K + k] : fa[((size_t)g * R + j - 2 * R) * K + k]);
      for (int n = 0; n < N + F; ++n) {
        int sum = 0;
        if (g >= 0)
          for (int j = 0; j < rank[g]; ++j)
            sum += n < N ? h[(n < 256 ? 0 : R) + j] * I(b[((size_t)g * N + n) * R + j])
                         : h[2 * R + j] * I(fb[((size_t)g * F + n - N) * R + j]);
        if (g >= 0) sum *= (int)scale[g];
        const size_t at = n < N ? (size_t)row * N + n : (size_t)row * F + n - N;
        const bool same = n < N ? gy[at] == (g < 0 ? y[at] : Bf16((float)(I(y[at]) + sum)))
                                : gz[at] == z[at] + (float)sum;
        if (!same) {
          std::printf("turn %d (%s), row %d of %d, column %d differs\n", turn, replay ? "replay" : "eager", row,
                      rows, n);
          return 1;
        }
      }
    }
    all += rows;
  }
  fqa::HipCheck(hipGraphExecDestroy(exec), "destroy");
  fqa::HipCheck(hipGraphDestroy(graph), "destroy");
  std::printf("ok: %d rows\n", all);
  return 0;
} catch (const std::exception& e) {
  std::printf("%s\n", e.what());
  return 1;
}
