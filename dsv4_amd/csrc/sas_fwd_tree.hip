// The forward over trees of drafted tokens, MI355X (gfx950): sas_fwd.hip's kernels
// with a slot resolution that reads each token's mask of attended nodes, and their
// entry point. A build of its own, so that the chains' kernels stay as they are: with
// the mask as a run-time choice in one build, an fp8 decode of 8 sequences took
// 18.3 us for 18.0 and fp8 prefill chunks 574 for 570.
//
// A node's window is its path: the committed rows before the drafts, then its
// ancestors in query order, the last win_left + 1 of them. The row of window slot j is
// found from the mask's bits alone (counts and a select by halves, some 50 VALU
// operations beside two round trips of loads), so a tree costs a token what a chain does.
#define SAS_FWD_TREE 1
#include "sas_fwd.hip"
