// policy_bf16.hip -- policy_kernels.h for one element type
#include "policy_kernels.h"

hipError_t az_policy_launch_bf16(const PolicyDev& a, bool grad, int& groups, hipStream_t stream) { return launch_o<2>(a, grad, groups, stream); }
