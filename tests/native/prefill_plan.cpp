// The launch shapes of prompts, checked on the CPU (built against libqm38.so and run by
// tests/test_prefill_plan.py): what the prefill kernels take for granted of a plan, with
// the splits and after they were taken back, and the plans that the launcher refuses.
#include <stdio.h>

#include "../../qwen38-metal_amd/csrc/kv_internal.h"

static int g_failures = 0;

static void expect(bool ok, const char* what, const qm::AttnArgs& a) {
  if (ok) return;
  fprintf(stderr, "FAIL %s: %u rows at %u, %u/%u heads of %u: waves %u, splits %u, split_tiles %u\n", what, a.rows,
          a.start, a.heads, a.kv_heads, a.head_dim, a.wg_waves, a.splits, a.split_tiles);
  ++g_failures;
}

int main() {
  const uint32_t heads[][3] = {{64, 8, 128}, {24, 4, 256}, {32, 8, 64}, {20, 5, 80}, {16, 1, 128}, {6, 2, 37},
                               {3, 1, 256},  {2, 1, 64},   {1, 1, 1},   {9, 1, 200}};
  const uint32_t rows[] = {1, 2, 65, 130, 333, 512, 513, 700, 1000, 1101, 1500, 2048, 2101, 8192};
  const uint32_t starts[] = {0, 13, 1000, 4096, 20001, 131071};
  unsigned by_blocks = 0, plans = 0;
  for (const int cus : {64, 256, 304})
    for (const auto& h : heads)
      for (const uint32_t M : rows)
        for (const uint32_t start : starts)
          for (const bool q4 : {false, true})
            for (const uint16_t* gate : {(const uint16_t*)nullptr, (const uint16_t*)0x1000}) {
              qm_runtime rt;
              rt.cu_count = cus;
              qm::AttnArgs a{};
              a.gate = gate;
              a.heads = h[0];
              a.kv_heads = h[1];
              a.head_dim = h[2];
              a.head_dim_pad = qm::attn_padded_dim(h[2]);
              a.n_seqs = 1;
              a.prefill = 1;
              a.rows = M;
              a.start = start;
              a.seqs[0].len = start + M;
              qm::plan_prefill(&rt, q4, &a);
              ++plans;
              expect(a.wg_waves == 4 || a.wg_waves == 8, "waves", a);
              expect(a.splits >= 1, "no workgroup", a);
              if (a.split_tiles) {
                ++by_blocks;
                expect(q4, "blocks of their own over 8 bits", a);
                expect(a.splits > 1 && a.splits <= (uint32_t)qm::kMaxBlockSplits, "splits by blocks", a);
                // The longest block's tiles are all taken.
                const uint32_t gh = a.heads / a.kv_heads, block = 32 * a.wg_waves, cols = M * gh;
                const uint32_t tiles =
                    qm::prefill_tiles((cols + block - 1) / block - 1, block, cols, gh, start, start + M);
                expect((uint64_t)a.splits * a.split_tiles >= tiles, "tiles without a workgroup", a);
              }
              // A plan that needs partials is not launched without them (decided before
              // anything is launched).
              if (q4 && (a.splits > 1 || a.split_tiles))
                expect(qm::launch_q4kv_prefill(a, nullptr) == hipErrorInvalidValue, "launch without partials", a);
              qm::unsplit_prefill(&a);
              expect(a.splits == 1 && a.split_tiles == 0, "splits taken back", a);
              qm::AttnArgs one = a;
              one.split_tiles = 4;
              if (q4)
                expect(qm::launch_q4kv_prefill(one, nullptr) == hipErrorInvalidValue, "blocks of one split, no partials",
                       one);
            }
  if (by_blocks == 0) {
    fprintf(stderr, "FAIL no plan by blocks\n");
    ++g_failures;
  }
  printf("%u plans, %u by blocks, %d failures\n", plans, by_blocks, g_failures);
  return g_failures != 0;
}
