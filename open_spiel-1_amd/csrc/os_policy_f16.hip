// Policy kernels on f16 logits (os_policy.h).
#include "os_policy_launch.h"

template struct osp::Kernels<_Float16>;
