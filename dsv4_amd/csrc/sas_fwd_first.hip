// The forward with first rows that stay visible, MI355X (gfx950): sas_fwd.hip's kernels
// with a slot resolution that puts the cache's first rows in front of the window's, and
// their entry points. A build of its own, so that the other calls' kernels stay as they
// are (sas_fwd_tree.hip holds what a run-time choice costs them).
//
// A token at position s attends rows j <= s of the raw cache with j >= s - win_left or
// j < ori_first: a first row that the window holds is resolved there, once.
// 8192 tokens, 64 heads of 512 channels, 4 + 128 rows: 279 us (two workgroups a CU; 429 with
// one), query and output alone 208 at the rate of a large copy. Top-k lists over fp8 rows:
// 442 us, 656 with one.
#define SAS_FWD_FIRST 1
#include "sas_fwd.hip"
