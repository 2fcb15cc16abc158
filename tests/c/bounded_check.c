/* The structures and argument errors of the entry points for bounded caches (attention with
   first rows in sight, its gradients, row weights, evictions) as a C caller sees them: sizes
   and last members' offsets, one a line, then the errors' codes. No device memory is touched. */
#include <stddef.h>
#include <stdio.h>
#include <string.h>

#include "sas.h"

#define SHOW(T, last) printf(#T " %zu %zu\n", sizeof(T), offsetof(T, last))

int main(void) {
  SHOW(SasFwdFirstArgs, ori_first);
  SHOW(SasBwdFirstArgs, ori_first);
  SHOW(SasRowWeightsArgs, cmp_rows);
  SHOW(SasCacheEvictArgs, keep_recent);
  SasFwdFirstArgs f;
  SasBwdFirstArgs b;
  SasRowWeightsArgs w;
  SasCacheEvictArgs e;
  int32_t dtype = 0;
  size_t ws = 1;
  memset(&f, 0, sizeof(f));
  memset(&b, 0, sizeof(b));
  memset(&w, 0, sizeof(w));
  memset(&e, 0, sizeof(e));
  printf("null %d %d %d %d %d\n", sas_fwd_first_v1(NULL, NULL), sas_bwd_first_v1(NULL, NULL),
         sas_bwd_first_plan(NULL, &dtype, &ws), sas_row_weights_v1(NULL, NULL), sas_cache_evict_v1(NULL, NULL));
  f.ori_first = b.ori_first = w.ori_first = -1;
  printf("errors %d %d %d %d\n", sas_fwd_first_v1(&f, NULL), sas_bwd_first_v1(&b, NULL), sas_row_weights_v1(&w, NULL),
         sas_cache_evict_v1(&e, NULL));
  printf("message %d\n", sas_last_error()[0] != 0);
  /* no sequences: nothing to do */
  e.row_bytes = 16;
  e.bt_stride = e.block_size = e.num_blocks = e.budget = 1;
  printf("empty %d\n", sas_cache_evict_v1(&e, NULL));
  return 0;
}
