// The prefill path of the backward with first rows, MI355X (gfx950): sas_bwd_pre.hip's
// kernels, the key-major pass with tiles for the first rows, whose tokens are all those
// whose window starts behind them.
#define SAS_BWD_FIRST 1
#include "sas_bwd_pre.hip"
