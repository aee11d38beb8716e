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


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("v", [65, 82, 130, 362, 500, 768, 1025, 1400, 2047, 2049, 4099, 20011, 33001,
                               70001, 150001, 300007])
def test_gpu_forced_moves_of_long_rows(require_gpu, v, dtype):
  """A row's only allowed action has log probability 0, entropy 0, gradient 0,
  whichever kernel takes it, whether a mask or logits of -inf exclude the rest;
  few rows and many go through different ones."""
  from os_amd import policy
  n = 33 if v < 33000 else 3
  logits, _, _ = make(n, v, dtype, False, seed=21, spread=1.0)
  logits[1:] *= 9
  moves = (torch.arange(n) * 7919 + v - 1) % v
  legal = torch.zeros(n, v, dtype=torch.uint8)
  legal[torch.arange(n), moves] = 1
  alone = logits.masked_fill(legal == 0, -math.inf)
  ids, one = moves[:, None].cuda(), torch.full((n, 1), 3.0, device="cuda")
  for x, lg in ((logits, legal.cuda()), (alone, None)):
    for t in (1.0, 0.7):
      leaf = x.cuda().requires_grad_()
      r = policy.logprobs(leaf, moves.cuda(), lg, top=1, temperature=t)
      loss, _ = policy.distill(leaf, one, ids, lg, temperature=t)
      for what, got in (("logprob", r.logprob), ("entropy", r.entropy), ("top", r.top_logprob),
                        ("loss", loss)):
        assert bool((got == 0).all()), (what, t, got[got != 0][:4])
      grad, = torch.autograd.grad((r.logprob * 0.3 + r.entropy - 2 * loss).sum(), leaf)
      assert bool((grad == 0).all())
      both, loss = torch.empty_like(leaf), torch.empty(n, device="cuda")
      policy.distill_into(leaf.detach(), one, loss, None, ids, lg, temperature=t, grad=both)
      assert bool((loss == 0).all()) and bool((both == 0).all())


@gpu
@pytest.mark.parametrize("v", [64, 65, 362, 700, 1500, 2049, 5000, 150001])
def test_gpu_log_probabilities_are_not_positive(require_gpu, v):
  """Rows whose likeliest action is far ahead: its probability is 1 within a few
  steps, its log probability never above 0."""
  from os_amd import policy
  n = 400 if v < 100000 else 40
  g = torch.Generator(device="cuda").manual_seed(v)
  x = torch.randn(n, v, generator=g, device="cuda") + torch.randn(n, 1, generator=g, device="cuda") * 5
  best = torch.randint(0, v, (n,), generator=g, device="cuda")
  x[torch.arange(n, device="cuda"), best] += 30.0
  for t in (1.0, 0.7):
    r = policy.logprobs(x, best, top=2, temperature=t)
    assert bool((r.logprob <= 0).all()) and bool((r.top_logprob <= 0).all())
    loss, _ = policy.distill(x, torch.ones(n, 1, device="cuda"), best[:, None], temperature=t)
    assert bool((loss >= 0).all())


def _merged(ids, q, v):
  """The target distribution over the actions (64 bits): repeats added up."""
  full = torch.zeros(len(q), v, dtype=torch.float64)
  return full.scatter_add_(1, ids.clamp(min=0).long(), torch.where(ids >= 0, q, torch.zeros_like(q)))


@gpu
@pytest.mark.parametrize("repeats", [False, True])
@pytest.mark.parametrize("v", [40, 700, 3000, 150001])
def test_gpu_target_entropy_is_that_of_the_entries(require_gpu, v, repeats):
  """target_entropy = -sum_j q_j log q_j over the listed entries.  With distinct
  actions loss - target_entropy is the divergence of the target distribution from
  the policy; an action listed m times with mass Q in all leaves it short of that
  by sum Q log m or less, which the entries' entropy has too much."""
  from os_amd import policy
  n, k = 6, 12
  logits, _, _ = make(n, v, "f32", False, seed=31)
  g = torch.Generator().manual_seed(v)
  ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
  if repeats:
    ids = ids[:, torch.arange(k) // 3]
  w = torch.rand(n, k, generator=g) + 0.1
  loss, h = policy.distill(logits.cuda(), w.cuda(), ids.cuda())
  want, tol = ref.distill(logits, w, ids)
  close(loss, want["loss"], tol["loss"], "loss")
  close(h, want["entropy"], tol["entropy"], "entropy")
  q = w.double() / w.double().sum(1, keepdim=True)
  full = _merged(ids, q, v)
  merged = -torch.special.xlogy(full, full).sum(1)
  _, logp = ref.softmax(logits.double())
  divergence = torch.special.xlogy(full, full).sum(1) - (full * logp).sum(1)
  assert bool((divergence > 0).all())
  got = (loss - h).cpu().double()
  # (the subtraction's own rounding: half a step of the result)
  bound = tol["loss"] + tol["entropy"] + got.abs() * ref.U
  if repeats:
    assert bool((h.cpu().double() > merged + bound).all()) and bool((got < divergence - bound).all())
    assert bool((got > divergence - math.log(3) - bound).all())
  else:
    assert bool(((got - divergence).abs() <= bound).all())


def test_the_divergence_is_stated_for_distinct_actions():
  """(two equal logits, the first action listed four times: loss log 2, entropy of
  the entries log 4)"""
  import os
  import re
  from os_amd import policy
  root = os.path.join(os.path.dirname(__file__), "..")
  texts = [policy.distill.__doc__, open(os.path.join(root, "include", "os_mcts.h")).read(),
           open(os.path.join(root, "INTEGRATION.md")).read()]
  for text in texts:
    text = re.sub(r"[\s*]+", " ", text)
    at = text.index("Kullback-Leibler")
    assert "distinct" in text[max(0, at - 200):at + 200]
