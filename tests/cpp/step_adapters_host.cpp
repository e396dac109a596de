// step_adapters_host.cpp — include/fqa_step.hpp's adapter calls under AddressSanitizer +
// UndefinedBehaviorSanitizer (tests/test_step_adapters.py), with the device stubbed out: "device" buffers
// are host memory, the pack is the CPU oracle's, and a stub fqa_lora_plan writes all that the call's
// bounds let the kernel write, so that a bound past a buffer's end is reported.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "../../include/fqa_step.hpp"
#include "../../oracle/fqa_oracle.h"

hipError_t hipMalloc(void** p, size_t n) {
  *p = std::malloc(n ? n : 1);
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void* p) {
  std::free(p);
  return hipSuccess;
}
hipError_t hipMemcpyAsync(void* dst, const void* src, size_t n, hipMemcpyKind, hipStream_t) {
  std::memcpy(dst, src, n);
  return hipSuccess;
}
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) {
  *e = nullptr;
  return hipSuccess;
}
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "stub"; }

static std::vector<int32_t> g_plan;  // the last plan: reqs bound, rows bound, items, rows of the pack
extern "C" {
int32_t fqa_dec_default_waves(int32_t) { return 1024; }
int32_t fqa_dec_wave_bound(int32_t, int32_t waves) { return waves > 0 ? waves : 0; }
int32_t fqa_pre_item_bound(int32_t n_reqs, int32_t max_rows, int32_t tile) {
  return max_rows / tile + n_reqs;
}
int64_t fqa_decode_workspace_bytes(const fqa_dims*, int32_t) { return 64; }
int64_t fqa_decode_prefix_workspace_bytes(const fqa_dims*, int32_t, int32_t) { return 64; }
int fqa_rope_tables(int32_t, int32_t, float, float*, float*) { return FQA_OK; }
int fqa_pack(const fqa_batch* b, const fqa_pack_cfg* c, const fqa_pack_out* o, void*) {
  fqo_pack(b->n_reqs_dev ? *b->n_reqs_dev : b->n_reqs, b->computed, b->n_new, b->bt_off, b->bt_pages,
           c->max_rows, c->max_blocks, c->pool_pages, c->dec_grid_waves, c->dec_min_pages, c->dec_wave_cap,
           c->pre_tile_q, c->pre_item_cap, c->dec_share, c->dec_prefix_pages, c->dec_pre_cap,
           o->cu_seqlens, o->qlen, o->positions, o->row_req, o->slot_mapping, o->block_tables,
           o->decode_rids, o->prefill_rids, o->dec_seqs, o->dec_waves, o->pre_items,
           o->dec_prefix, o->dec_pre_items, o->meta);
  return FQA_OK;
}
int32_t fqa_lora_item_bound(int32_t n_reqs, int32_t rows, int32_t n_adapters) {
  if (n_reqs < 0 || rows < 0 || n_adapters < 1) return FQA_EINVAL;
  return rows / FQA_LORA_TILE_ROWS + (n_reqs < n_adapters + 1 ? n_reqs : n_adapters + 1);
}
int fqa_lora_plan(const int32_t* adapter, int32_t n_ids, const int32_t*, const int32_t* cu,
                  const int32_t* meta, int32_t reqs, int32_t rows_bound, int32_t n_adapters,
                  int32_t* rows, int32_t* items, int32_t item_cap, int32_t* lora_meta, void*) {
  if (reqs < 0 || reqs > FQA_MAX_REQS || rows_bound < 0 ||
      item_cap < fqa_lora_item_bound(reqs, rows_bound, n_adapters))
    return FQA_EINVAL;
  const int n = meta[FQA_META_ROWS] < rows_bound ? meta[FQA_META_ROWS] : rows_bound;
  for (int r = 0; r < meta[FQA_META_REQS] && r < reqs && r < n_ids; ++r) {
    volatile int32_t id = adapter[r] + cu[r + 1];
    (void)id;
  }
  for (int i = 0; i < n; ++i) rows[i] = i;
  std::memset(items, 0, (size_t)item_cap * 16);
  std::memset(lora_meta, 0, FQA_LORA_META_LEN * 4);
  g_plan = {reqs, rows_bound, item_cap, n};
  return FQA_OK;
}
}

static fqa::BatchInput Batch(const std::vector<int>& lens) {
  fqa::BatchInput in;
  int page = 0;
  for (const int n : lens) {
    in.computed.push_back(3);
    in.n_new.push_back(n);
    in.block_tables.emplace_back();
    for (int k = 0; k < (3 + n + 15) / 16; ++k) in.block_tables.back().push_back(page++);
  }
  return in;
}

#define EXPECT(c)                                  \
  if (!(c)) {                                      \
    std::printf("line %d: %s\n", __LINE__, #c);    \
    return 1;                                      \
  }

int main() {
  const int max_rows = 40, slots = 6, n_adapters = 3;
  fqa::StepContext ctx(max_rows, slots, 100000, 10000, 0, 64);
  for (const bool bounded : {false, true}) {
    const std::vector<std::vector<int>> batches = {
        {1, 20, 1}, {40}, {1, 1, 1, 1, 1, 1}, {}, {30, 11}, {90000}, {1, 50000, 1}};
    for (const auto& lens : batches) {
      int rows = 0;
      for (const int n : lens) rows += n;
      const fqa::BatchInput in = Batch(lens);
      const std::vector<int32_t> ids(lens.size(), 1);  // one for every request, no more
      if (bounded) {
        ctx.UploadBatch(in, nullptr);
        ctx.Pack(nullptr);
      } else {
        ctx.PrepareInputs(in, nullptr);
      }
      ctx.PlanAdapters(ids.data(), n_adapters, nullptr, bounded);
      // more rows than the context holds: the pack says so and has none
      EXPECT(g_plan[1] <= max_rows && g_plan[3] == (rows <= max_rows ? rows : 0));
      EXPECT(g_plan[0] == (bounded ? slots : (int)lens.size()));
    }
  }
  std::printf("ok\n");
  return 0;
}
