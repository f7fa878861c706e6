// The instances of the forward kernel for calls with rules (RULES = 1, 2 in fwd_sm100.cu) as a translation unit of their
// own, so that the sets of instances compile side by side.
#define FA_RULES_INSTANCES 1
#include "fwd_sm100.cu"
