/* The structures and argument errors of the norm, append and tree entry points as a C
   caller sees them: sizes and last members' offsets, one a line, then the errors'
   codes. No device memory is touched. */
#include <stddef.h>
#include <stdio.h>
#include <string.h>

#include "sas.h"

#define SHOW(T, last) printf(#T " %zu %zu\n", sizeof(T), offsetof(T, last))

int main(void) {
  SHOW(SasNormRopeArgs, reserved);
  SHOW(SasNormRopeBwdArgs, dkv_out_stride_t);
  SHOW(SasCacheAppendArgs, reserved);
  SHOW(SasFwdTreeArgs, tree_words);
  SasNormRopeArgs r;
  SasNormRopeBwdArgs b;
  SasCacheAppendArgs a;
  SasFwdTreeArgs t;
  size_t ws = 1;
  memset(&r, 0, sizeof(r));
  memset(&b, 0, sizeof(b));
  memset(&a, 0, sizeof(a));
  memset(&t, 0, sizeof(t));
  printf("errors %d %d %d %d %d\n", sas_norm_rope_v1(&r, NULL), sas_norm_rope_bwd_plan(&b, &ws), sas_norm_rope_bwd_v1(&b, NULL),
         sas_cache_append_v1(&a, NULL), sas_fwd_tree_v1(&t, NULL));
  printf("message %d\n", sas_last_error()[0] != 0);
  /* no rows: nothing to do */
  r.D = 512;
  r.weight_dtype = SAS_DT_FP32;
  b.fwd = r;
  const int forward = sas_norm_rope_v1(&r, NULL), plan = sas_norm_rope_bwd_plan(&b, &ws);
  printf("empty %d %d %zu\n", forward, plan, ws);
  return 0;
}
