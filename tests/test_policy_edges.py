"""The policy operators (os_amd/policy.py, csrc/os_policy.hip) at their edges."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import policy_ref as ref
from test_policy import TYPES, check_distill, check_logprobs, close, cuda, make, make_target

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


def test_abi_refuses_overlapping_buffers():
  """A result that shares memory with an operand or another result, before any
  launch: each pair of a call's buffers in turn, disjoint columns of one buffer's
  rows let by (those calls fail later, at the launch: there is no GPU here)."""
  import ctypes
  from os_amd import _lib
  L = _lib.lib
  n, v, k, top = 4, 40000, 3, 2
  base = 1 << 20

  def at(i):
    return base * (1 + 2 * i)
  size = {"logits": n * v * 4, "legal": n * v, "actions": n * 8, "logprob": n * 4, "entropy": n * 4,
          "stats": n * 8, "top_action": n * top * 8, "top_logprob": n * top * 4, "g_logprob": n * 4,
          "g_entropy": n * 4, "g_top": n * top * 4, "grad": n * v * 4, "ids": n * k * 8,
          "target": n * k * 4, "weight": n * 4, "loss": n * 4, "target_entropy": n * 4}
  assert max(size.values()) <= base

  def call(name, p):
    rows = ctypes.byref(_lib.AzRows(logits=p["logits"], legal=p["legal"], num_rows=n, ld=v,
                                    legal_ld=v, num_actions=v, dtype=0, temperature=1.0))
    tg = None
    if "ids" in p:
      tg = ctypes.byref(_lib.AzTarget(actions=p["ids"], target=p["target"], actions_ld=k,
                                      target_ld=k, k=k, type=3, wide=1))
    if name == "logprobs":
      work = L.os_az_rows_workspace(rows, top)
      return L.os_az_logprobs_async(rows, p["actions"], 1, p["logprob"], p["entropy"], p["stats"], top,
                                    p["top_action"], p["top_logprob"], at(40), work, None)
    if name == "logprobs_grad":
      return L.os_az_logprobs_grad_async(rows, p["actions"], 1, p["entropy"], p["stats"], top,
                                         p["top_action"], p["g_logprob"], 1, p["g_entropy"], 1,
                                         p["g_top"], p["grad"], v, None)
    if name == "distill":
      work = L.os_az_rows_workspace(rows, 0)
      return L.os_az_distill_async(rows, tg, p["weight"], p["loss"], p["target_entropy"], p["stats"],
                                   p["grad"], v, at(40), work, None)
    return L.os_az_distill_grad_async(rows, tg, p["weight"], 1, p["stats"], p["grad"], v, None)
  calls = {
      "logprobs": (["logits", "legal", "actions"],
                   ["logprob", "entropy", "stats", "top_action", "top_logprob"]),
      "logprobs_grad": (["logits", "legal", "actions", "entropy", "stats", "top_action", "g_logprob",
                         "g_entropy", "g_top"], ["grad"]),
      "distill": (["logits", "legal", "ids", "target", "weight"],
                  ["loss", "target_entropy", "stats", "grad"]),
      "distill_grad": (["logits", "legal", "ids", "target", "weight", "stats"], ["grad"]),
  }
  for name, (ins, outs) in calls.items():
    names = ins + outs
    for o in outs:
      for other in names:
        if other == o:
          continue
        for shift in (0, size[other] - 8, 8 - size[o]):
          p = {x: at(i) for i, x in enumerate(names)}
          p[o] = p[other] + shift
          assert call(name, p) == _lib.OS_ERR_INVALID, (name, o, other, shift)
          assert b"overlap" in L.os_last_error(), (name, o, other, shift, L.os_last_error())


@gpu
def test_gpu_overlapping_results_are_refused(require_gpu):
  """From Python: ValueError; neighbours and disjoint columns are no overlap."""
  from os_amd import policy
  n, a = 6, 9
  f = dict(device="cuda")
  x, t = torch.zeros(n, a, **f), torch.rand(n, a, **f)
  legal = torch.ones(n, a, dtype=torch.uint8, **f)
  out, h = torch.zeros(n, **f), torch.zeros(n, **f)
  act = torch.zeros(n, dtype=torch.int64, **f)
  w = torch.ones(n, **f)
  buf = torch.zeros(3 * n * a, **f)
  ta = torch.zeros(n, 3, dtype=torch.int64, **f)
  for call in (lambda: policy.distill_into(x, t, out, None, None, grad=t),
               lambda: policy.distill_into(x, t, out, out),
               lambda: policy.distill_into(x, t, w, None, weight=w, grad=torch.empty_like(x)),
               lambda: policy.distill_into(x, t, t.view(-1)[:n]),
               lambda: policy.logprobs_into(x, x.view(-1)[:n]),
               lambda: policy.logprobs_into(x, out, out, act),
               lambda: policy.logprobs_into(x, out, act.view(torch.float32)[:n], act),
               lambda: policy.logprobs_into(x, out, top_action=ta,
                                            top_logprob=ta.view(-1).view(torch.float32)[:18].view(n, 3)),
               lambda: policy.logprobs_into(x, buf[:n], stats=buf[2:2 * n + 2].view(n, 2))):
    with pytest.raises(ValueError):
      call()
  # one buffer's neighbouring parts
  policy.logprobs_into(x, buf[:n], buf[n:2 * n], act, stats=buf[2 * n:4 * n].view(n, 2))
  both = torch.zeros(n, 3 * a, **f)
  both[:, a:2 * a] = t
  policy.distill_into(both[:, :a], both[:, a:2 * a], out, h, grad=both[:, 2 * a:])
  want, tol = ref.distill(x.cpu(), t.cpu())
  close(out, want["loss"], tol["loss"], "loss")
  close(both[:, 2 * a:], want["grad"], tol["grad"] + ref.rounding(torch.float32, want["grad"]), "grad")
  rows = torch.zeros(2 * n, a, **f)
  policy.distill_into(rows[::2], t, out, h, grad=rows[1::2])
  close(rows[1::2], want["grad"], tol["grad"] + ref.rounding(torch.float32, want["grad"]), "grad")
  assert bool((rows[::2] == 0).all())


@gpu
def test_gpu_written_tensors_change_their_version(require_gpu):
  """Autograd finds out that a tensor which an older graph has saved was written
  by logprobs_into or distill_into since."""
  from os_amd import policy
  n, a = 6, 9
  f = dict(device="cuda")
  x, t, w = torch.randn(n, a, **f), torch.rand(n, a, **f), torch.ones(n, **f)
  act = torch.zeros(n, dtype=torch.int64, **f)

  def new():
    return dict(entropy=torch.ones(n, **f), logprob=torch.ones(n, **f), stats=torch.ones(n, 2, **f),
                top_action=torch.zeros(n, 2, dtype=torch.int64, **f), top_logprob=torch.ones(n, 2, **f)), \
        dict(loss=torch.ones(n, **f), target_entropy=torch.ones(n, **f), grad=torch.ones(n, a, **f),
             stats=torch.ones(n, 2, **f))
  lp, ds = new()
  calls = ((lp, lambda o: policy.logprobs_into(x, actions=act, **o)),
           (ds, lambda o: policy.distill_into(x, t, weight=w, **o)))
  for out, call in calls:
    for key, tensor in out.items():
      scale = torch.ones_like(tensor, dtype=torch.float32).requires_grad_()
      before = tensor._version
      graph = (scale * tensor).sum()
      call(out)
      assert tensor._version > before, key
      if tensor.is_floating_point():
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
          graph.backward()
  # operands are not written
  assert x._version == t._version == w._version == act._version == 0
  # tensors made in inference mode have no version, and are written all the same
  with torch.inference_mode():
    lp, ds = new()
  policy.logprobs_into(x, actions=act, **lp)
  policy.distill_into(x, t, weight=w, **ds)
  want, tol = ref.distill(x.cpu(), t.cpu())
  close(ds["loss"], want["loss"], tol["loss"], "loss")


def test_abi_refuses_misaligned_buffers():
  """Each operand and result lies at a multiple of its element's size (values that
  are read for a whole row at once come through the scalar unit, which drops an
  address's low bits), or the call is refused before any launch."""
  import ctypes
  from os_amd import _lib
  L = _lib.lib
  n, v, k, top = 4, 9, 3, 2
  size = dict(actions=8, logprob=4, entropy=4, stats=4, top_action=8, top_logprob=4, g_logprob=4,
              g_entropy=4, g_top=4, ids=8, target=4, weight=4, loss=4, target_entropy=4)

  def call(name, p, wide, type_):
    rows = ctypes.byref(_lib.AzRows(logits=p["logits"], num_rows=n, ld=v, num_actions=v, dtype=0,
                                    temperature=1.0))
    tg = ctypes.byref(_lib.AzTarget(actions=p["ids"], target=p["target"], actions_ld=k, target_ld=k,
                                    k=k, type=type_, wide=wide))
    if name == "logprobs":
      return L.os_az_logprobs_async(rows, p["actions"], wide, p["logprob"], p["entropy"], p["stats"],
                                    top, p["top_action"], p["top_logprob"], None, 0, None)
    if name == "logprobs_grad":
      return L.os_az_logprobs_grad_async(rows, p["actions"], wide, p["entropy"], p["stats"], top,
                                         p["top_action"], p["g_logprob"], 1, p["g_entropy"], 1,
                                         p["g_top"], p["grad"], v, None)
    if name == "distill":
      return L.os_az_distill_async(rows, tg, p["weight"], p["loss"], p["target_entropy"], p["stats"],
                                   p["grad"], v, None, 0, None)
    return L.os_az_distill_grad_async(rows, tg, p["weight"], 1, p["stats"], p["grad"], v, None)
  used = dict(logprobs="actions logprob entropy stats top_action top_logprob",
              logprobs_grad="actions entropy stats top_action g_logprob g_entropy g_top",
              distill="ids target weight loss target_entropy stats",
              distill_grad="ids target weight stats")
  names = ["logits", "grad"] + sorted(size)
  for name, keys in used.items():
    for key in keys.split():
      for wide in (0, 1):
        for type_ in (_lib.AZ_LOGITS_F32, _lib.AZ_LOGITS_BF16, _lib.AZ_LOGITS_F16, _lib.AZ_WEIGHTS_F32,
                      _lib.AZ_WEIGHTS_I32):
          step = size[key]
          if key in ("actions", "ids") and not wide:
            step = 4
          if key == "target" and type_ in (_lib.AZ_LOGITS_BF16, _lib.AZ_LOGITS_F16):
            step = 2
          p = {x: 4096 * (1 + i) for i, x in enumerate(names)}
          p[key] += step // 2
          assert call(name, p, wide, type_) == _lib.OS_ERR_INVALID, (name, key, wide, type_)
          assert b"aligned" in L.os_last_error(), (name, key, wide, type_, L.os_last_error())


@gpu
@pytest.mark.parametrize("v", [2, 9, 82, 700, 3000, 40000, 150001])
def test_gpu_logits_at_both_ends_of_the_type(require_gpu, v):
  """x - m beyond the type's range at a temperature that brings it back in: the log
  probability is finite."""
  from os_amd import policy
  n, t = 3, 4.0
  big = torch.finfo(torch.float32).max
  logits = torch.zeros(n, v)
  logits[:, 0] = torch.tensor([big, 0.9 * big, 0.6 * big])
  logits[:, v - 1] = torch.tensor([-big, -0.9 * big, -0.7 * big])
  actions = torch.full((n,), v - 1)
  check_logprobs(logits, None, actions, 2, t)
  want, _ = ref.logprobs(logits, actions, None, 0, t)
  assert bool(torch.isfinite(want["logprob"]).all())
  ids = torch.tensor([[0, v - 1]] * n)
  w = torch.tensor([[1.0, 1.0]] * n)
  check_distill(logits, None, w, ids, "weights", t)


# ---- every size of kernel ----

# Rows of up to 64 actions share a wave, of up to 2048 have one that holds 0.5,
# 1, 1.5, 2, 3, 4, 6 or 8 KiB, longer ones have a workgroup: both sides of each
# border, in actions of 4 bytes (and of 2: up to 2048 actions, 4 KiB), and sizes
# whose last chunk is nearly empty or nearly full.
BORDERS = sorted({512 * b // size + d for b in (1, 2, 3, 4, 6, 8, 12, 16) for size in (2, 4)
                  for d in (-1, 0, 1) if 512 * b // size + d <= 2049} | {63, 64, 65, 67, 2050})


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("v", BORDERS)
def test_gpu_every_operation_at_the_kernels_borders(require_gpu, v, dtype, masked):
  from os_amd import policy
  n = 7
  logits, legal, actions = make(n, v, dtype, masked, 1 if v % 2 else 0, seed=v)
  # the last action is the likeliest, the given one, or excluded
  logits[1, v - 1] = 20.0
  actions[2] = v - 1
  logits[4, v - 1] = -math.inf
  if masked:
    legal[1, v - 1] = legal[2, v - 1] = 1
    legal[5, v - 1] = 0
  check_logprobs(logits, legal, actions, 0, 0.7)
  check_logprobs(logits, legal, actions, 9)
  g = torch.Generator().manual_seed(v)
  gl, gh, gt = torch.randn(n, generator=g), torch.randn(n, generator=g), torch.randn(n, 9, generator=g)
  for top in (0, 9):
    leaf = cuda(logits).requires_grad_()
    r = policy.logprobs(leaf, actions.cuda(), cuda(legal), top=top, temperature=1.3)
    outs, ups = [r.logprob, r.entropy], [gl.cuda(), gh.cuda()]
    if top:
      outs.append(r.top_logprob)
      ups.append(gt.cuda())
    grad, = torch.autograd.grad(outs, leaf, ups)
    want, tol = ref.logprobs_grad(logits, actions, legal, 1.3, gl, gh,
                                  r.top_action.cpu() if top else None, gt if top else None)
    close(grad, want, tol + ref.rounding(grad.dtype, want), "grad")
  weight = torch.randn(n, generator=g)
  k = min(v, 70)
  target, ids = make_target(n, v, k, legal, "weights", "i32")
  ids[1, 0] = torch.where(ids[1, 0] < 0, -1, v - 1)
  ids[1, 1:] = torch.where(ids[1, 1:] == v - 1, -1, ids[1, 1:])
  check_distill(logits, legal, target, ids, "weights", 1.0, weight, wide=False)
  ids[3, -1] = ids[3, 0]
  check_distill(logits, legal, target.float(), ids, "weights", 0.8, weight)
  if v <= 1024:
    target, _ = make_target(n, v, v, legal, "logits", dtype, dense=True)
    if masked:
      target = target.masked_fill(legal == 0, -math.inf)
    target[4, v - 1] = -math.inf
    check_distill(logits, legal, target, None, "logits", 1.5, weight)


# ---- float32 arithmetic, held to what it can do ----

def _roundings(v):
  """Roundings that a sum over a row of v float32 actions meets, at most.  Up to 64
  actions: four a lane, four steps over 16 lanes.  Up to 2048: the lane's elements
  one after the other (as many as the kernel holds), six steps, three more for the
  quotient by the maximum's own exponential.  Longer rows: four in a chunk, then up
  to 8 chunks (where rows are few; a product, a sum and two for the factor each), then
  lanes, waves and parts (6, 4 and 6 steps), four roundings for each of the three
  changes of the reference."""
  if v <= 64:
    return 8
  if v <= 2048:
    return 2 * min(u for u in (1, 2, 3, 4, 6, 8, 12, 16) if u * 128 >= v) + 6 + 3
  return 4 + 8 * 4 + 6 + 4 + 6 + 12 + 3


def _row_sizes(x):
  """p, log p, the distances to the maximum (nats) and their mean under p."""
  p, logp = ref.softmax(x)
  d = torch.where(p > 0, x.amax(1, keepdim=True) - x, torch.zeros_like(x))
  return p, logp, d, (p * d).sum(1)


@gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("v", [7, 64, 82, 362, 768, 1025, 2047, 4099, 20011, 32769, 70001, 131072])
def test_gpu_float32_precision(require_gpu, v, masked):
  """An exponential is off by an ulp (two half steps U) and by its argument's two
  roundings, 2 U a nat of distance d from the maximum (3 U where chunks were
  rescaled).  With R roundings in the sum, s is off by U (R + 2 + 3 E d), E under p;
  the logarithm of s by that, and 2 U of itself.  p = e / s in the gradient has
  U (R + 2 + 3 E d + 2 + 3 d + 3 log s + 6): the exponentials of d and of log s, and
  three products.  The entropy is log s + E d: an exponential's error e acts as
  p |log p + H| e on it, the two sums' R as U R (1 + 2 E d), the terms' products and
  the quotient as 4 U E d.  (Statistics of 11 bits, half a step of 2^-12, would be off
  by ten times these bounds and more.)"""
  from os_amd import policy
  n, t = 5, 0.8
  logits, legal, actions = make(n, v, "f32", masked, 0, seed=77)
  actions = torch.arange(n) * 31 % v
  if masked:
    legal[torch.arange(n), actions] = 1
  x = ref.masked(logits, legal, t)
  p, logp, d, mean = _row_sizes(x)
  logs = -(logp + d).amax(1)  # log p of the maximum, but for its sign
  logs = torch.where(torch.isfinite(logs), logs, torch.zeros_like(logs)).abs()
  R = _roundings(v)
  s_err = R + 2 + 3 * mean + 2 * logs
  assert float((s_err + 8 + 3 * logs).max()) * ref.U < 2.0 ** -12 / 10
  leaf = logits.cuda().requires_grad_()
  r = policy.logprobs(leaf, actions.cuda(), None if legal is None else legal.cuda(), temperature=t)
  entropy = -ref.plogp(p, logp).sum(1)
  own = torch.where(p > 0, p * (logp + entropy[:, None]).abs() * (2 + 3 * d), torch.zeros_like(p))
  h_err = R * (1 + 2 * mean) + own.sum(1) + 4 * mean + 2 * logs + entropy.abs() + 4
  close(r.entropy, entropy, ref.U * h_err, "entropy")
  at = actions[:, None]
  lp = logp.gather(1, at)[:, 0]
  close(r.logprob, lp, ref.U * (s_err + 4 * d.gather(1, at)[:, 0] + lp.abs() + 2), "logprob")
  # a log probability's gradient, p's relative error apart from the given action's 1
  one = torch.ones(n)
  grad, = torch.autograd.grad(r.logprob, leaf, one.cuda(), retain_graph=True)
  hot = torch.zeros(n, v, dtype=torch.float64).scatter_(1, at, 1.0)
  rel = (s_err + 8)[:, None] + 3 * d + 3 * logs[:, None]
  want = torch.where(x > -math.inf, hot - p, torch.zeros_like(p)) / t
  tol = torch.where(x > -math.inf, ref.U * (p * rel + 3 * hot) + ref.LEAST, torch.zeros_like(p)) / t
  close(grad, want, tol + ref.rounding(torch.float32, want), "logprob gradient")
  # cross entropy on that action: the same with the other sign
  both, loss = torch.empty_like(leaf), torch.empty(n, device="cuda")
  policy.distill_into(leaf.detach(), one[:, None].cuda(), loss, None, at.cuda(),
                      None if legal is None else legal.cuda(), temperature=t, grad=both)
  close(both, -want, tol + ref.rounding(torch.float32, want), "loss gradient")
  close(loss, -lp, ref.U * (s_err + 4 * d.gather(1, at)[:, 0] + 3 * lp.abs() + 2), "loss")
  # the entropy's gradient: -p (log p + H), the parts' errors on top of p's
  grad, = torch.autograd.grad(r.entropy, leaf, one.cuda())
  h = entropy[:, None]
  want = torch.where(p > 0, -p * (logp + h), torch.zeros_like(p)) / t
  size = torch.where(p > 0, p * (logp.abs() + h + d + logs[:, None] + 1), torch.zeros_like(p))
  tol = torch.where(x > -math.inf, ref.U * (size * (rel + 4) + p * h_err[:, None]) + ref.LEAST * (105 + h),
                    torch.zeros_like(p)) / t
  close(grad, want, tol + ref.rounding(torch.float32, want), "entropy gradient")
