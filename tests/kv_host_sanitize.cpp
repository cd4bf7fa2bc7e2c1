// Exercises the host-only half of the paged 8-bit cache's launchers (torch_mlu_amd/csrc/fa_kv_host.h) over a grid of ordinary,
// extreme and malformed parameter blocks, under sanitizers, and checks what a plan has to hold: every row, key and slice inside
// the grid, and a workspace that covers every partial result.  Prints how many blocks it pushed through and how many had a plan.
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <initializer_list>

#include "fa_kv_host.h"

using namespace fa::kvhost;

static void must(bool ok, const char* what) {
  if (!ok) {
    fprintf(stderr, "does not hold: %s\n", what);
    abort();
  }
}

int main() {
  long blocks = 0, plans = 0;
  const int32_t kMax = 0x7fffffff;
  for (int32_t batch : {-1, 0, 1, 3, 64, 8192, kMax})
    for (int32_t hk : {0, 1, 2, 8, 1 << 20})
      for (int32_t group : {1, 7, 16, 128})
        for (int32_t sq : {-1, 0, 1, 5, 500, 1 << 29, kMax})
          for (int32_t d : {16, 64, 128, 256, 100})
            for (int32_t pages : {0, 1, 129, 1 << 20, kMax})
              for (int32_t page : {32, 64, 1 << 20, 48, kMax})
                for (int32_t packed : {0, 1})
                  for (int32_t splits : {0, 1, 7, 64, 65}) {
                    fa_kv_attn_params p;
                    memset(&p, 0, sizeof(p));
                    p.q = p.key_pages = p.value_pages = (const void*)0x1000;
                    p.out = (void*)0x1000;
                    p.lse = (float*)0x1000;
                    p.key_scales = p.value_scales = (const float*)0x1000;
                    p.block_table = p.seqused_k = (const int32_t*)0x1000;
                    if (packed) p.cu_seqlens_q = (const int32_t*)0x1000;
                    p.batch = batch; p.heads_k = hk;
                    p.heads_q = (int64_t)hk * group > kMax ? kMax : hk * group;
                    p.seqlen_q = sq; p.total_q = packed ? (sq > 1000 ? sq : 1000) : 0;
                    p.head_dim = d; p.num_pages = 100; p.table_pages = pages; p.block_table_stride = pages;
                    p.page_size = page; p.scale_block = 32; p.dtype = FA_DTYPE_BF16; p.num_splits = splits; p.scale = 0.1f;
                    ++blocks;
                    if (attn_validate(&p) != FA_OK) continue;
                    ++plans;
                    const AttnPlan r = attn_plan(&p);
                    const int64_t rows = (int64_t)p.seqlen_q * group, keys = (int64_t)pages * page;
                    must(r.splits >= 1 && r.splits <= FA_MAX_SPLITS, "1 to 64 slices");
                    must(r.splits == 1 || r.splits <= (keys + 31) / 32, "no more slices than blocks");
                    must(r.tiles == 8 || rows <= 16 * r.tiles, "the streaming kernel's rows");
                    must(r.tiles == 8 || p.heads_k % (1 << r.hw_log2) == 0, "whole groups of heads");
                    must(r.tiles == 8 || (1 << r.hw_log2) <= stream_waves(d <= 128 ? 128 : 256), "a wavefront a head");
                    if (r.tiles == 8 && !packed) must((int64_t)r.row_blocks * 128 >= rows, "a place for every block of rows");
                    must(attn_workspace_bytes(&p, r) == (r.splits == 1 ? 0 : (size_t)attn_rows(&p) * p.heads_q * r.splits * (d * 4 + 8)), "the workspace");
                    const int64_t wgs = attn_wgs(&p, r), threads = r.tiles == 8 ? 256 : 512;
                    must(wgs >= -1 && (wgs < 0 || wgs * threads <= 0xffffffffLL), "a launch's threads in 32 bits");
                  }
  // packed: sequence b's blocks begin at place c * group / 128 + b (c: rows before it) and end before the next one's
  for (int64_t group : {1, 3, 4, 7, 16, 128})
    for (int seed = 0; seed < 200; ++seed) {
      int64_t c = 0, end = 0;
      unsigned x = 12345u + seed;
      const int n = 1 + seed % 9;
      for (int b = 0; b < n; ++b) {
        x = x * 1664525u + 1013904223u;
        const int64_t len = (x >> 16) % (seed % 3 ? 300 : 40);
        const int64_t begin = c * group / 128 + b;
        must(begin >= end, "places of two sequences apart");
        end = begin + (len * group + 127) / 128;
        c += len;
      }
      must(end <= c * group / 128 + n, "places inside the grid");
    }
  for (int32_t batch : {-1, 0, 1, 8192, 8193, kMax})
    for (int32_t pages : {-1, 0, 1, 1 << 15, kMax})
      for (int32_t page : {0, 1, 64, 1 << 16, kMax})
        for (int32_t tokens : {-1, 0, 7, kMax}) {
          fa_kv_plan_params p;
          memset(&p, 0, sizeof(p));
          p.cached = (const int32_t*)0x1000; p.new_tokens = (const int32_t*)0x2000; p.block_table = (int32_t*)0x3000;
          p.free_count = (const int32_t*)0x4000; p.cu_seqlens = (int32_t*)0x5000; p.seqused = (int32_t*)0x6000;
          p.positions = (int32_t*)0x7000; p.slots = (int64_t*)0x8000; p.admitted = (uint8_t*)0x9000; p.free_left = (int32_t*)0xa000;
          p.batch = batch; p.table_pages = pages; p.block_table_stride = pages; p.page_size = page; p.max_tokens = tokens;
          ++blocks;
          plans += plan_validate(&p) == FA_OK;
        }
  printf("%ld blocks, %ld plans\n", blocks, plans);
  return 0;
}
