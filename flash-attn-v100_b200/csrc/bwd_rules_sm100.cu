// The instances of the backward kernels for calls with rules (RULES = 1, 2 in bwd_sm100.cu) as a translation unit of their
// own, so that the sets of instances compile side by side.  B4 N4096 H32 D128 causal bf16: 1754-1860 us, without rules 1635-1670; with
// eight documents a row 720.
#define FA_RULES_INSTANCES 1
#include "bwd_sm100.cu"
