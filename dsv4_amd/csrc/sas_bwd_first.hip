// The backward of the forward with first rows (sas_fwd_first.hip), MI355X (gfx950):
// sas_bwd.hip's per-token kernels and planner over that forward's keys. A first row is a
// key of every token behind its window, so prefills sum its gradient key-major
// (sas_bwd_pre_first.hip); calls outside that path add per token and row.
#define SAS_BWD_FIRST 1
#include "sas_bwd.hip"
