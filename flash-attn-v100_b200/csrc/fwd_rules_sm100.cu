// The instances of the forward kernel for calls with rules (RULES = 1, 2 in fwd_sm100.cu) as a translation unit of their
// own, so that the sets of instances compile side by side.  What the rules cost, B2 N4096 H32 causal bf16, us: D 64 227 without, ranges
// 233, distances 274, a cap 366, both 414; D 128 275, 290, 365, 405, 480: the softmax warps' instructions.
#define FA_RULES_INSTANCES 1
#include "fwd_sm100.cu"
