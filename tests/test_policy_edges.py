"""The policy operators (os_amd/policy.py, csrc/os_policy.hip) at their edges."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import policy_ref as ref
from test_policy import TYPES, close, cuda, make, make_target

gpu = pytest.mark.gpu


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
  """A tangent would be lost (results without one read as constant): refused
  before anything else, whether or not the primal requires a gradient and in
  whatever gradient mode."""
  from os_amd import policy
  x = torch.zeros(4, 7, requires_grad=grad)
  t = torch.ones(4, 7)
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(x, torch.ones(4, 7))
    for mode in (torch.enable_grad, torch.no_grad):
      with mode():
        for call in (lambda: policy.logprobs(dual), lambda: policy.logprobs(dual[:, :5], top=2),
                     lambda: policy.distill(dual, t),
                     lambda: policy.distill(x, forward_ad.make_dual(t, t))):
          with pytest.raises(ValueError, match="forward-mode"):
            call()
    with pytest.raises(ValueError, match="GPU"):  # no tangent: the next check
      policy.logprobs(x)
  with pytest.raises(ValueError, match="forward-mode"):
    torch.func.jvp(lambda z: policy.logprobs(z).entropy, (torch.zeros(4, 7),), (t,))


@gpu
def test_gpu_forward_mode_is_refused(require_gpu):
  from os_amd import policy
  x = torch.randn(4, 7, device="cuda")
  t = torch.ones(4, 7, device="cuda")
  with forward_ad.dual_level():
    dual = forward_ad.make_dual(x, t)
    for call in (lambda: policy.logprobs(dual), lambda: policy.distill(dual, t),
                 lambda: policy.distill(x, forward_ad.make_dual(t, t))):
      with pytest.raises(ValueError, match="forward-mode"):
        call()
    policy.logprobs(x)
    policy.distill(x, t)
  with pytest.raises(ValueError, match="forward-mode"):
    torch.func.jvp(lambda z: policy.distill(z, t)[0], (x,), (t,))
