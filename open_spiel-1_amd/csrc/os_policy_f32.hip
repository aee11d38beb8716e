// Policy kernels on f32 logits (os_policy.h).
#include "os_policy_launch.h"

template struct osp::Kernels<float>;
