// The instances of the backward kernels for calls with rules (RULES = 1, 2 in bwd_sm100.cu) as a translation unit of their
// own, so that the sets of instances compile side by side.
#define FA_RULES_INSTANCES 1
#include "bwd_sm100.cu"
