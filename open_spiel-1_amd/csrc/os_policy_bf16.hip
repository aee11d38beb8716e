// Policy kernels on bf16 logits (os_policy.h).
#include "os_policy_launch.h"

template struct osp::Kernels<__bf16>;
