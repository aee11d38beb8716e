"""Policy operators (os_amd/policy.py, csrc/os_policy.hip) against their formulas
in 64 bits (policy_ref.py), within bounds counted from the kernels' roundings."""
import ctypes
import math

import numpy as np
import pytest
import torch

import policy_ref as ref
from os_amd import _lib
from os_amd import engine as E

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# one wave, one block and several blocks a row; a size below, at and above
# powers of two and vector widths
SIZES = [(1, 1), (5, 2), (300, 7), (33, 64), (17, 65), (70, 82), (40, 121), (9, 362), (3, 768),
         (130, 1025), (2, 2047), (6, 4099), (3, 20011), (2, 70001)]


def close(got, want, tol, what):
  # (what is past float32's range is its infinity)
  got, want, tol = got.detach().cpu().double(), want.float().double(), tol.double()
  assert got.shape == want.shape, what
  same = (got == want) | (torch.isnan(got) & torch.isnan(want))
  ok = same | ((got - want).abs() <= tol)
  if not bool(ok.all()):
    i = tuple(int(k) for k in torch.nonzero(~ok)[0])
    raise AssertionError("%s: %d of %d off, first at %s: %r, expected %r +- %r"
                         % (what, int((~ok).sum()), ok.numel(), i, float(got[i]), float(want[i]),
                            float(tol[i])))


def make(n, v, dtype="f32", masked=True, pad=0, seed=0, spread=2.5):
  """(logits on the CPU as a view of wider rows, legal uint8 or None, actions)."""
  g = torch.Generator().manual_seed(seed * 7919 + n * 131 + v)
  x = torch.randn(n, v + pad, generator=g) * spread + torch.randn(n, 1, generator=g) * 3
  logits = x.to(TYPES[dtype])[:, :v]
  legal = None
  if masked:
    legal = (torch.rand(n, v, generator=g) < 0.6).to(torch.uint8)
    legal[torch.arange(n), torch.randint(0, v, (n,), generator=g)] = 1
    if n > 2:
      legal[n // 2] = 0
  actions = torch.randint(0, v, (n,), generator=g)
  if n > 1:
    actions[0] = -1
  return logits, legal, actions


def cuda(x):
  """On the GPU with the same strides (a wider buffer's view)."""
  if x is None or x.is_contiguous():
    return None if x is None else x.cuda()
  base = torch.zeros(x.shape[0], x.stride(0), dtype=x.dtype)
  base[:, :x.shape[1]] = x
  return base.cuda()[:, :x.shape[1]]


def check_logprobs(logits, legal, actions, top, temperature=1.0, wide=True):
  from os_amd import policy
  want, tol = ref.logprobs(logits, actions, legal, top, temperature)
  a = actions if wide else actions.to(torch.int32)
  got = policy.logprobs(cuda(logits), a.cuda(), cuda(legal), top=top, temperature=temperature)
  close(got.entropy, want["entropy"], tol["entropy"], "entropy")
  close(got.logprob, want["logprob"], tol["logprob"], "logprob")
  if top:
    assert torch.equal(got.top_action.cpu(), want["top_action"])
    close(got.top_logprob, want["top_logprob"], tol["top_logprob"], "top_logprob")


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("n,v", SIZES)
def test_gpu_logprobs(require_gpu, n, v, masked, dtype):
  for pad, top, t in ((0, 5, 1.0), (1, 20, 0.7), (3, 0, 2.0)):
    logits, legal, actions = make(n, v, dtype, masked, pad, seed=pad)
    check_logprobs(logits, legal, actions, top, t, wide=pad != 1)


@gpu
@pytest.mark.parametrize("top", [1, 2, 31, 64])
@pytest.mark.parametrize("v", [3, 64, 150, 3000, 40000])
def test_gpu_top_ties(require_gpu, v, top):
  """Equal logits by the lower action: constant rows, rows of few values, rows
  whose largest values crowd into one place, sorted rows, signed zeros."""
  g = torch.Generator().manual_seed(v * 100 + top)
  rows = [torch.zeros(v), torch.full((v,), -3.0), torch.arange(v).float(), -torch.arange(v).float(),
          torch.randint(0, 3, (v,), generator=g).float(), torch.randn(v, generator=g)]
  z = torch.zeros(v)
  z[::2] = -0.0
  rows.append(z)
  c = torch.randn(v, generator=g) - 50
  c[v // 3:v // 3 + 2000] += 60.0           # one contiguous stretch
  rows.append(c)
  s = torch.randn(v, generator=g) - 50
  s[(torch.arange(v) // 8) % 64 == 5] = 4.0  # one lane's elements, all equal
  rows.append(s)
  s2 = torch.randn(v, generator=g)
  s2[(torch.arange(v) // 4) % 64 == 9] += 50.0
  rows.append(s2)
  logits = torch.stack(rows)
  for dtype in ("f32", "bf16"):
    x = logits.to(TYPES[dtype])
    check_logprobs(x, None, torch.zeros(len(rows), dtype=torch.int64), top)


def _special_rows(v, dtype):
  """Rows with infinities, NaN in allowed and excluded places, the type's
  lowest value as a mask, empty rows; finite rows between them."""
  t = TYPES[dtype]
  low = torch.finfo(t).min
  x = torch.randn(16, v, generator=torch.Generator().manual_seed(v))
  legal = torch.ones(16, v, dtype=torch.uint8)
  x[1] = -math.inf
  legal[2] = 0
  x[2, 0] = math.nan
  x[3, : v // 2] = -math.inf
  legal[4, : v // 2] = 0
  x[4, : v // 2] = math.nan
  legal[5, 0] = 0
  x[5, 0] = math.inf
  x[6] = low
  x[7, : v - 1] = low
  x[8, v - 1] = math.nan
  x[9, 0] = math.inf
  x[10] = math.nan
  x[11, :] = torch.finfo(t).max
  x[11, 0] = 0.0
  x[12] = x[12] + 30000.0
  legal[13] = 0
  legal[13, v - 1] = 1
  x[14] = 0.0
  x[14, v // 2] = 120.0
  x = torch.where(x > torch.finfo(t).max, x, x.clamp(min=-math.inf))
  return x.to(t), legal


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("v", [2, 9, 82, 513, 5000, 33333])
def test_gpu_special_rows(require_gpu, v, dtype):
  from os_amd import policy
  logits, legal = _special_rows(v, dtype)
  actions = torch.full((16,), v - 1, dtype=torch.int64)
  actions[4] = 0
  actions[0], actions[7], actions[15] = v, -5, v + 100
  check_logprobs(logits, legal, actions, 4)
  # gradients: no NaN leaves its row
  gl = torch.randn(16, generator=torch.Generator().manual_seed(1))
  gh = torch.randn(16, generator=torch.Generator().manual_seed(2))
  want, tol = ref.logprobs_grad(logits, actions, legal, 1.0, gl, gh)
  leaf = logits.cuda().requires_grad_()
  r = policy.logprobs(leaf, actions.cuda(), legal.cuda())
  grad, = torch.autograd.grad([r.logprob, r.entropy], leaf, [gl.cuda(), gh.cuda()])
  close(grad, want, tol + ref.rounding(grad.dtype, want), "grad")
  ids = torch.zeros(16, 2, dtype=torch.int64)
  ids[:, 1] = v - 1
  counts = torch.tensor([[1, 3]] * 16, dtype=torch.int32)
  want, tol = ref.distill(logits, counts, ids, legal)
  leaf = logits.cuda().requires_grad_()
  loss, h = policy.distill(leaf, counts.cuda(), ids.cuda(), legal.cuda())
  close(loss, want["loss"], tol["loss"], "loss")
  close(h, want["entropy"], tol["entropy"], "target entropy")
  grad, = torch.autograd.grad(loss, leaf, torch.ones(16, device="cuda"))
  close(grad, want["grad"], tol["grad"] + ref.rounding(grad.dtype, want["grad"]), "grad")


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v", [(1, 1), (5, 2), (70, 7), (33, 82), (9, 362), (130, 1025), (6, 4099),
                                 (3, 20011), (2, 70001)])
def test_gpu_logprobs_gradient(require_gpu, n, v, dtype):
  """Against the formula: log probabilities, entropies, top log probabilities
  (the given action among them or not), shared and per-row upstreams."""
  from os_amd import policy
  for masked, pad, top, t in ((True, 1, 0, 1.0), (False, 0, 6, 0.7)):
    logits, legal, actions = make(n, v, dtype, masked, pad, seed=3)
    g = torch.Generator().manual_seed(n + v)
    gl, gh = torch.randn(n, generator=g), torch.randn(n, generator=g)
    gt = torch.randn(n, top, generator=g) if top else None
    leaf = cuda(logits).requires_grad_()
    r = policy.logprobs(leaf, actions.cuda(), cuda(legal), top=top, temperature=t)
    outs, ups = [r.logprob, r.entropy], [gl.cuda(), gh.cuda()]
    ta = None
    if top:
      outs.append(r.top_logprob)
      ups.append(gt.cuda())
      ta = r.top_action.cpu()
    grad, = torch.autograd.grad(outs, leaf, ups, retain_graph=True)
    want, tol = ref.logprobs_grad(logits, actions, legal, t, gl, gh, ta, gt)
    assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
    close(grad, want, tol + ref.rounding(grad.dtype, want), "grad")
    # expanded upstreams (a sum's, a mean's), one output alone
    one = torch.ones(n)
    grad, = torch.autograd.grad(r.entropy.mean(), leaf, retain_graph=True)
    want, tol = ref.logprobs_grad(logits, legal=legal, temperature=t, g_entropy=one / n)
    close(grad, want, tol + ref.rounding(grad.dtype, want), "entropy grad")
    grad, = torch.autograd.grad(r.logprob.sum(), leaf)
    want, tol = ref.logprobs_grad(logits, actions, legal, t, one)
    close(grad, want, tol + ref.rounding(grad.dtype, want), "logprob grad")


def make_target(n, v, k, legal, kind, dtype="f32", seed=0, dense=False):
  g = torch.Generator().manual_seed(seed * 31 + n + v + k)
  score = torch.rand(n, v, generator=g)
  if legal is not None:
    score = score.masked_fill(legal == 0, -1.0)
  best, ids = score.topk(k, 1)
  ids = ids.masked_fill(best < 0, -1)
  if kind == "weights":
    t = torch.exp(torch.randn(n, k, generator=g) * 1.5).mul(4).floor()
    if dense and legal is not None:
      t = t * legal
    t = t.to(torch.int32) if dtype == "i32" else t
  else:
    t = (torch.randn(n, k, generator=g) * 3 + 2).to(TYPES[dtype])
  return t, None if dense else ids


def check_distill(logits, legal, target, ids, kind, temperature=1.0, weight=None, wide=True):
  """distill_into (loss alone; loss and gradient) and the autograd form."""
  from os_amd import policy
  n, v = logits.shape
  want, tol = ref.distill(logits, target, ids, legal, kind, temperature, weight)
  x, lg = cuda(logits), cuda(legal)
  tg = cuda(target)
  i = None if ids is None else cuda(ids if wide else ids.to(torch.int32))
  w = None if weight is None else weight.cuda()

  def held(loss, h, what):
    close(loss, want["loss"], tol["loss"], what + " loss")
    close(h, want["entropy"], tol["entropy"], what + " entropy")
  loss = torch.full((n,), -7.0, device="cuda")
  h = torch.full((n,), -7.0, device="cuda")
  policy.distill_into(x, tg, loss, h, i, lg, kind, temperature)
  held(loss, h, "loss alone")
  wide_grad = torch.full((n, v + 2), -7.0, dtype=x.dtype, device="cuda")
  grad = wide_grad[:, :v]
  policy.distill_into(x, tg, loss.fill_(-7), h.fill_(-7), i, lg, kind, temperature, w, grad)
  held(loss, h, "fused")
  gt = tol["grad"] + ref.rounding(x.dtype, want["grad"])
  close(grad, want["grad"], gt, "fused grad")
  assert bool((wide_grad[:, v:] == -7).all())
  leaf = x.detach().requires_grad_()
  loss, h = policy.distill(leaf, tg, i, lg, kind, temperature)
  held(loss, h, "autograd")
  total = loss.sum() if w is None else (loss * w).sum()
  if bool(torch.isfinite(want["loss"]).all()):
    grad, = torch.autograd.grad(total, leaf)
    close(grad, want["grad"], gt, "autograd grad")


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (5, 2, 2), (300, 7, 7), (33, 64, 5), (17, 65, 33),
                                   (70, 82, 82), (9, 362, 362), (3, 768, 200), (130, 1025, 64),
                                   (5, 2047, 1024), (6, 4099, 64), (3, 20011, 1000), (2, 70001, 64)])
def test_gpu_distill(require_gpu, n, v, k, dtype):
  g = torch.Generator().manual_seed(n)
  weight = torch.randn(n, generator=g)
  logits, legal, _ = make(n, v, dtype, True, 1, seed=5)
  target, ids = make_target(n, v, k, legal, "weights", "i32")
  check_distill(logits, legal, target, ids, "weights", 1.0, weight, wide=False)
  logits, legal, _ = make(n, v, dtype, False, 0, seed=6)
  target, ids = make_target(n, v, k, None, "logits", dtype)
  check_distill(logits, None, target, ids, "logits", 2.0, None)
  target, ids = make_target(n, v, k, None, "weights", "f32", seed=1)
  check_distill(logits, None, target, ids, "weights", 0.5, weight)


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v", [(1, 1), (300, 7), (70, 82), (33, 121), (9, 362), (3, 768),
                                 (3, 1024)])
def test_gpu_distill_dense(require_gpu, n, v, dtype):
  logits, legal, _ = make(n, v, dtype, True, 1, seed=8)
  target, _ = make_target(n, v, v, legal, "weights", "i32", dense=True)
  check_distill(logits, legal, target, None, "weights")
  target, _ = make_target(n, v, v, None, "logits", dtype, dense=True)
  check_distill(logits, None, target, None, "logits", 1.5)


@gpu
@pytest.mark.parametrize("v", [5, 82, 700, 5000, 40001])
def test_gpu_distill_odd_targets(require_gpu, v):
  """Rows without a target, actions listed several times, padding between the
  entries, mass on excluded actions, actions past the end, weights that are 0,
  negative, tiny and huge, -inf and NaN teacher logits."""
  n, k = 12, 6
  logits, _, _ = make(n, v, "f32", False, 0, seed=4)
  legal = torch.ones(n, v, dtype=torch.uint8)
  legal[7, 3] = 0
  ids = torch.tensor([[0, 1, 2, 3, 4, -1]] * n)
  w = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 100.0]] * n)
  ids[0] = -1                                  # no target
  w[1] = 0.0                                   # no mass
  ids[2] = torch.tensor([1, 1, 1, 1, 4, 1])    # one action five times
  ids[3] = torch.tensor([-1, 3, -7, 3, -1, 0])  # padding between
  w[4] = torch.tensor([-3.0, 0.0, 2.0, -1.0, 2.0, 5.0])
  w[5] = torch.tensor([1e38, 3e38, 2e38, 3e38, 0.0, 1.0])
  w[6] = torch.tensor([1e-38, 3e-38, 0.0, 2e-38, 0.0, 1.0])
  # row 7: mass on an excluded action
  ids[8, 2] = v                                # past the end
  ids[9] = torch.tensor([v - 1, v - 1, 0, 0, v - 1, 0])
  w[10, 0] = math.nan
  check_distill(logits, legal, w, ids, "weights")
  check_distill(logits, legal, w[:, :0], ids[:, :0], "weights")
  z = torch.randn(n, k, generator=torch.Generator().manual_seed(3))
  z[1] = -math.inf
  z[4, 2] = -math.inf
  z[5] = torch.tensor([1e30, 0.0, -1e30, 2.0, 3e30, 4.0])
  z[6] = 5000.0
  z[10, 1] = math.nan
  z[11] = torch.finfo(torch.float32).min
  check_distill(logits, legal, z, ids, "logits", 2.0)


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("n,v", [(1, 2), (40, 7), (40, 82), (9, 362), (5, 1500), (1100, 5000),
                                 (2, 150001)])
def test_gpu_all_mass_in_one_place(require_gpu, n, v, dtype):
  """A target with one entry, or one that is not 0, has q = 1 there: its entropy
  is exactly 0."""
  from os_amd import policy
  logits, _, _ = make(n, v, dtype, False, seed=11)
  x = logits.cuda()
  g = torch.Generator().manual_seed(n + v)
  ids = torch.randint(0, v, (n, 1), generator=g).cuda()
  one = (torch.rand(n, 1, generator=g) * 400 + 1e-3).cuda()
  many = torch.zeros(n, 5, device="cuda")
  many[:, 2:3] = one
  for kind, target, at in (("weights", one, ids), ("weights", one.ceil().int(), ids),
                           ("weights", many, ids.repeat(1, 5)), ("logits", one, ids),
                           ("logits", many.masked_fill(many == 0, -math.inf), ids.repeat(1, 5))):
    loss, h = torch.empty(n, device="cuda"), torch.full((n,), -7.0, device="cuda")
    policy.distill_into(x, target, loss, h, at, kind=kind)
    assert bool((h == 0).all()), kind
    grad = torch.empty_like(x)
    policy.distill_into(x, target, loss, h.fill_(-7), at, kind=kind, grad=grad)
    assert bool((h == 0).all()), kind


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("v", [1, 2, 9, 64])
def test_gpu_forced_moves(require_gpu, v, dtype):
  """A row's only allowed action has log probability 0, entropy 0, gradient 0."""
  from os_amd import policy
  n = 33
  logits, _, _ = make(n, v, dtype, False, seed=12)
  moves = torch.arange(n) % v
  legal = torch.zeros(n, v, dtype=torch.uint8)
  legal[torch.arange(n), moves] = 1
  leaf = logits.cuda().requires_grad_()
  r = policy.logprobs(leaf, moves.cuda(), legal.cuda(), top=1, temperature=0.7)
  loss, _ = policy.distill(leaf, torch.full((n, 1), 3.0, device="cuda"), moves[:, None].cuda(),
                           legal.cuda(), temperature=0.7)
  for x in (r.logprob, r.entropy, r.top_logprob, loss):
    assert bool((x == 0).all())
  grad, = torch.autograd.grad((r.logprob * 0.3 + r.entropy - 2 * loss).sum(), leaf)
  assert bool((grad == 0).all())


@gpu
def test_gpu_strides_and_broadcasts(require_gpu):
  """Row strides of 0 (one row for all), legal [A], legal rows inside wider
  ones, target columns of wider buffers, and memory that starts off any
  vector boundary."""
  from os_amd import policy
  n = 37
  for v in (7, 83, 1300, 9001):
    logits, legal, actions = make(1, v, "bf16", True)
    wide = logits.expand(n, v)
    acts = torch.arange(n) % v
    want, tol = ref.logprobs(wide, acts, legal.expand(n, v), 3)
    gl = torch.randn(n, generator=torch.Generator().manual_seed(v))
    leaf = logits.cuda().requires_grad_()
    for lg in (legal[0].cuda(), legal.cuda().expand(n, v)):
      r = policy.logprobs(leaf.expand(n, v), acts.cuda(), lg.bool(), top=3)
      close(r.logprob, want["logprob"], tol["logprob"], "logprob")
      assert torch.equal(r.top_action.cpu(), want["top_action"])
    # the shared row's gradient: the rows' gradients rounded to bf16, summed
    grad, = torch.autograd.grad(r.logprob, leaf, gl.cuda())
    g, gt = ref.logprobs_grad(wide, acts, legal.expand(n, v), 1.0, gl)
    bound = (gt + ref.rounding(torch.bfloat16, g)).sum(0) + n * g.abs().sum(0) * 2.0 ** -24
    close(grad[0], g.sum(0), bound + g.sum(0).abs() * 2.0 ** -8, "shared grad")
    for dtype in sorted(TYPES):
      for off in (1, 3):
        logits, legal, actions = make(n, v, dtype, True, 5, seed=off)
        base = torch.zeros(n * (v + 5) + off, dtype=TYPES[dtype], device="cuda")
        x = base[off:].view(n, v + 5)[:, :v]
        x.copy_(logits)
        lbase = torch.ones(n * (v + 2) + off, dtype=torch.uint8, device="cuda")
        lg = lbase[off:].view(n, v + 2)[:, :v]
        lg.copy_(legal)
        want, tol = ref.logprobs(logits, actions, legal, 5)
        r = policy.logprobs(x, actions.cuda(), lg, top=5)
        close(r.logprob, want["logprob"], tol["logprob"], "logprob")
        close(r.entropy, want["entropy"], tol["entropy"], "entropy")
        assert torch.equal(r.top_action.cpu(), want["top_action"])
        k = min(v, 6)
        target, ids = make_target(n, v, k, legal, "weights")
        tw = torch.zeros(n, k + 3, device="cuda")[:, 1:k + 1]
        tw.copy_(target)
        iw = torch.zeros(n, k + 2, dtype=torch.int32, device="cuda")[:, 1:k + 1]
        iw.copy_(ids)
        gbase = torch.full((n * (v + 3) + off,), -7.0, dtype=TYPES[dtype], device="cuda")
        grad = gbase[off:].view(n, v + 3)[:, :v]
        loss = torch.empty(n, device="cuda")
        policy.distill_into(x, tw, loss, None, iw, lg, grad=grad)
        want, tol = ref.distill(logits, target, ids, legal)
        close(loss, want["loss"], tol["loss"], "loss")
        close(grad, want["grad"], tol["grad"] + ref.rounding(grad.dtype, want["grad"]), "grad")
        assert bool((gbase[off:].view(n, v + 3)[:, v:] == -7).all()) and bool((gbase[:off] == -7).all())


@gpu
def test_gpu_offsets_past_32_bits(require_gpu):
  from os_amd import policy
  n, v, ld = 3, 4099, (1 << 31) + 5
  base = torch.empty((n - 1) * ld + v, dtype=torch.bfloat16, device="cuda")
  x = base.as_strided((n, v), (ld, 1))
  logits, _, actions = make(n, v, "bf16", False)
  x.copy_(logits)
  want, tol = ref.logprobs(logits, actions, None, 5)
  r = policy.logprobs(x, actions.cuda(), top=5)
  close(r.logprob, want["logprob"], tol["logprob"], "logprob")
  assert torch.equal(r.top_action.cpu(), want["top_action"])
  target, ids = make_target(n, v, 9, None, "logits")
  want, tol = ref.distill(logits, target, ids, None, "logits")
  gbase = torch.empty((n - 1) * ld + v, dtype=torch.bfloat16, device="cuda")
  grad = gbase.as_strided((n, v), (ld, 1))
  loss = torch.empty(n, device="cuda")
  policy.distill_into(x, target.cuda(), loss, None, ids.cuda(), kind="logits", grad=grad)
  close(grad, want["grad"], tol["grad"] + ref.rounding(grad.dtype, want["grad"]), "grad")


@gpu
@pytest.mark.parametrize("n,v", [(1 << 20, 2), (70000, 9), (40000, 300)])
def test_gpu_many_rows(require_gpu, n, v):
  """More rows than a launch holds blocks, against torch in 64 bits."""
  from os_amd import policy
  g = torch.Generator(device="cuda").manual_seed(n)
  x = torch.randn(n, v, generator=g, device="cuda")
  a = torch.randint(0, v, (n,), generator=g, device="cuda")
  r = policy.logprobs(x, a, top=2)
  lp = torch.log_softmax(x.double(), 1)
  bound = ref.U * (ref.adds(v) + 12 * 12 + 40)  # |log p| and |x - m| < 12 here
  assert float((r.logprob - lp.gather(1, a[:, None])[:, 0]).abs().max()) < bound
  assert torch.equal(r.top_action, torch.sort(x, dim=1, descending=True, stable=True)[1][:, :2])
  loss = torch.empty(n, device="cuda")
  grad = torch.empty_like(x)
  one = torch.ones(n, 1, device="cuda")
  policy.distill_into(x, one, loss, None, a[:, None], grad=grad)
  want = lp.exp()
  want.scatter_add_(1, a[:, None], -one.double())
  assert float((grad - want).abs().max()) < 3 * bound


def held_there(got, want, tol, what):
  """close() without leaving the GPU."""
  want, tol, got = want.float().double(), tol.double(), got.detach().double()
  ok = (got == want) | (torch.isnan(got) & torch.isnan(want)) | ((got - want).abs() <= tol)
  if not bool(ok.all()):
    i = tuple(int(k) for k in torch.nonzero(~ok)[0])
    raise AssertionError("%s: %d of %d off, first at %s: %r, expected %r +- %r"
                         % (what, int((~ok).sum()), ok.numel(), i, float(got[i]), float(want[i]),
                            float(tol[i])))


@gpu
@pytest.mark.parametrize("n,v,k,dtype,masked", [
    (1200, 1500, 70, "f32", False), (2600, 3001, 200, "bf16", True), (1100, 2047, 33, "f32", True),
    (1200, 2500, 1024, "f32", False), (1200, 2500, 600, "f32", True), (2600, 4099, 70, "f16", True),
    (2600, 4099, 70, "bf16", False), (1100, 9001, 70, "f32", False), (1100, 9001, 300, "bf16", True),
    (1030, 40000, 70, "bf16", False), (1030, 40001, 70, "f32", True), (1030, 70001, 9, "f32", False)])
def test_gpu_many_long_rows(require_gpu, n, v, k, dtype, masked):
  """Workgroups that go over several long rows, far ones, empty ones and ones
  with actions listed twice among them (the 64-bit formulas on the GPU)."""
  from os_amd import policy
  g = torch.Generator(device="cuda").manual_seed(n + v + k)
  f = dict(device="cuda", generator=g)
  x = torch.randn(n, v, **f) * 2.5
  x[7::97] += 30000.0
  if dtype == "f32":
    x[5::89] *= 2.0 ** 30
  x = x.to(TYPES[dtype])
  legal = None
  if masked:
    legal = (torch.rand(n, v, **f) < 0.6).to(torch.uint8)
    legal[::71] = 0
  actions = torch.randint(-1, v, (n,), **f)
  ids = torch.randint(0, v, (n, k), **f)
  ids[3::13, 1] = ids[3::13, 0]
  ids[::3, k // 2] = -1
  w = torch.rand(n, k, **f)
  if masked:
    w = w * legal.gather(1, ids.clamp(min=0))
  weight = torch.randn(n, **f)
  gl, gh, gt = torch.randn(n, **f), torch.randn(n, **f), torch.randn(n, 5, **f)
  leaf = x.clone().requires_grad_()
  r = policy.logprobs(leaf, actions, legal, top=5, temperature=0.9)
  grad, = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], leaf, [gl, gh, gt])
  loss, h, both = torch.empty(n, device="cuda"), torch.empty(n, device="cuda"), torch.empty_like(x)
  policy.distill_into(x, w, loss, h, ids, legal, "weights", 0.9, weight, both)
  alone, _ = policy.distill(leaf, w, ids, legal, temperature=0.9)
  again, = torch.autograd.grad((alone * weight).sum(), leaf)
  with torch.device("cuda"):
    want, tol = ref.logprobs(x, actions, legal, 5, 0.9)
    for key in ("logprob", "entropy", "top_logprob"):
      held_there(getattr(r, key), want[key], tol[key], key)
    assert torch.equal(r.top_action, want["top_action"])
    want, tol = ref.logprobs_grad(x, actions, legal, 0.9, gl, gh, r.top_action, gt)
    held_there(grad, want, tol + ref.rounding(x.dtype, want), "grad")
    want, tol = ref.distill(x, w, ids, legal, "weights", 0.9, weight)
    held_there(loss, want["loss"], tol["loss"], "loss")
    held_there(alone, want["loss"], tol["loss"], "loss alone")
    held_there(h, want["entropy"], tol["entropy"], "target entropy")
    for got in (both, again):
      held_there(got, want["grad"], tol["grad"] + ref.rounding(x.dtype, want["grad"]), "grad")


@gpu
@pytest.mark.parametrize("n,v,dtype", [(2300, 33001, "f32"), (2100, 70002, "bf16"),
                                       (2100, 70001, "f16"), (1500, 60000, "f32")])
def test_gpu_more_logits_than_the_cache(require_gpu, n, v, dtype):
  """Batches of more than 256 MiB equal their halves, bit for bit."""
  from os_amd import policy
  g = torch.Generator(device="cuda").manual_seed(v)
  f = dict(device="cuda", generator=g)
  x = torch.randn(n, v, **f).to(TYPES[dtype])
  actions = torch.randint(0, v, (n,), **f)
  ids = torch.randint(0, v, (n, 64), **f)
  w = torch.rand(n, 64, **f)
  gl = torch.randn(n, **f)

  def run(rows):
    leaf = x[rows].requires_grad_()
    r = policy.logprobs(leaf, actions[rows], top=7)
    grad, = torch.autograd.grad([r.logprob, r.entropy], leaf, [gl[rows], gl[rows]])
    m = len(leaf)
    loss, h, both = (torch.empty(m, device="cuda"), torch.empty(m, device="cuda"),
                     torch.empty(m, v, dtype=x.dtype, device="cuda"))
    policy.distill_into(x[rows], w[rows], loss, h, ids[rows], weight=gl[rows], grad=both)
    alone, _ = policy.distill(leaf, w[rows], ids[rows])
    again, = torch.autograd.grad(alone, leaf, gl[rows])
    return [r.logprob, r.entropy, r.top_action, r.top_logprob, grad, loss, h, both, alone, again]
  half = n // 2
  # (both above a thousand rows or both below: the same kernels)
  whole, parts = run(slice(0, n)), [run(slice(0, half)), run(slice(half, n))]
  if half >= 1024:
    for i, p in enumerate(whole):
      assert torch.equal(p, torch.cat([q[i] for q in parts])), i
  last = slice(n - 40, n)
  with torch.device("cuda"):
    want, tol = ref.logprobs(x[last], actions[last], None, 7)
    held_there(whole[0][last], want["logprob"], tol["logprob"], "logprob")
    assert torch.equal(whole[2][last], want["top_action"])
    want, tol = ref.logprobs_grad(x[last], actions[last], None, 1.0, gl[last], gl[last])
    held_there(whole[4][last], want, tol + ref.rounding(x.dtype, want), "grad")
    want, tol = ref.distill(x[last], w[last], ids[last], weight=gl[last])
    held_there(whole[5][last], want["loss"], tol["loss"], "loss")
    for i in (7, 9):
      held_there(whole[i][last], want["grad"], tol["grad"] + ref.rounding(x.dtype, want["grad"]),
                 "grad")


@gpu
@pytest.mark.parametrize("t", [1.0, 0.25, 3.0])
@pytest.mark.parametrize("v", [50, 900, 2500, 20011, 150001])
def test_gpu_common_offsets(require_gpu, v, t):
  """Rows far from zero on either side of where the scaled maximum has no
  fraction left (2^24), actions a few units below the maximum included."""
  edge = 2.0 ** 24 / math.log2(math.e) * t
  tops = [s * (edge + d) for s in (-1.0, 1.0) for d in (-1000.0, -150.0, -4.0, -1.0, 1.0, 40.0)]
  tops += [1e8, -1e8, 1e30, -1e30]
  g = torch.Generator().manual_seed(v)
  logits = torch.stack([torch.tensor(m) - torch.randint(1, 30, (v,), generator=g) for m in tops])
  logits[:, v // 3] = torch.tensor(tops)
  n = len(tops)
  actions = torch.randint(0, v, (n,), generator=g)
  check_logprobs(logits, None, actions, 3, t)
  target, ids = make_target(n, v, 6, None, "weights")
  check_distill(logits, None, target, ids, "weights", t)
  gl, gh = torch.randn(n, generator=g), torch.randn(n, generator=g)
  from os_amd import policy
  leaf = logits.cuda().requires_grad_()
  r = policy.logprobs(leaf, actions.cuda(), temperature=t)
  grad, = torch.autograd.grad([r.logprob, r.entropy], leaf, [gl.cuda(), gh.cuda()])
  want, tol = ref.logprobs_grad(logits, actions, None, t, gl, gh)
  close(grad, want, tol + ref.rounding(grad.dtype, want), "grad")


@gpu
@pytest.mark.parametrize("n,v,dtype,masked", [(2, 1 << 21, "f32", False), (1, (1 << 21) - 1, "f32", True),
                                              (3, (1 << 21) - 63, "bf16", True),
                                              (70, (1 << 20) + 1, "f16", False)])
def test_gpu_largest_rows(require_gpu, n, v, dtype, masked):
  logits, legal, actions = make(n, v, dtype, masked, seed=2)
  check_logprobs(logits, legal, actions, 64)
  target, ids = make_target(n, v, 64, legal, "weights")
  ids[:, -1] = torch.where(ids[:, 0] >= 0, v - 1, -1)
  if masked:
    legal[:, v - 1] = torch.where(ids[:, 0] >= 0, 1, 0).to(torch.uint8)
  check_distill(logits, legal, target, ids, "weights")

@gpu
@pytest.mark.parametrize("v,k", [(40, 1024), (700, 1024), (2047, 700), (20011, 1024)])
def test_gpu_distill_long_lists_with_repeats(require_gpu, v, k):
  n = 7
  logits, _, _ = make(n, v, "f32", False, seed=9)
  g = torch.Generator().manual_seed(v + k)
  ids = torch.randint(-1, max(2, v // 2), (n, k), generator=g)
  w = torch.rand(n, k, generator=g)
  check_distill(logits, None, w, ids, "weights", 1.0, torch.randn(n, generator=g))
  check_distill(logits, None, (w * 5).to(torch.float16), ids, "logits", 0.8, None, wide=False)


@gpu
def test_gpu_gradient_against_differences(require_gpu):
  """The kernels' own losses at x +- h: central differences with h = 2^-5 are
  off by h^2 / 6 times the third derivative (below 2 in size for the sum of
  these three terms) and by two losses' bounds over 2 h."""
  from os_amd import policy
  n, v, h = 3, 11, 2.0 ** -5
  logits, legal, _ = make(n, v, "f32", True, spread=1.0)
  legal[1, 2] = 1
  actions = torch.tensor([int(torch.nonzero(legal[r])[0]) if legal[r].any() else -1
                          for r in range(n)])
  target, ids = make_target(n, v, 4, legal, "weights")
  x0, lg, act = logits.cuda(), legal.cuda(), actions.cuda()

  def value(x):
    r = policy.logprobs(x, act, lg)
    loss, _ = policy.distill(x, target.cuda(), ids.cuda(), lg)
    return r.logprob.sum() + r.entropy.sum() + loss.sum()
  leaf = x0.clone().requires_grad_()
  grad, = torch.autograd.grad(value(leaf), leaf)
  terms = 3 * n * ref.U * 3 * ref.adds(v) * (1 + math.log2(v))
  bound = h * h / 3 + terms / h
  for r in range(n):
    for i in range(v):
      up, down = x0.clone(), x0.clone()
      up[r, i] += h
      down[r, i] -= h
      diff = (float(value(up).double()) - float(value(down).double())) / (2 * h)
      assert abs(float(grad[r, i]) - diff) < bound, (r, i)


def test_reference_gradient_against_differences():
  """policy_ref's own gradients, in 64 bits: central differences of its losses
  (h = 1e-4: h^2 / 6 times a third derivative below 8, and 1e-16 / h)."""
  n, v, h, t = 3, 9, 1e-4, 0.8
  logits, legal, actions = make(n, v, "f32", True)
  logits = logits.double()
  target, ids = make_target(n, v, 4, legal, "weights")
  top = ref.logprobs(logits, actions, legal, 2, t)[0]["top_action"]
  gl, gh = torch.randn(n).double(), torch.randn(n).double()
  gt = torch.randn(n, 2).double()
  legal_at = torch.where(legal[range(n), actions.clamp(min=0)] == 0, -1, actions)

  def value(x):
    o, _ = ref.logprobs(x, legal_at, legal, 0, t)
    lp = ref.softmax(ref.masked(x, legal, t))[1]
    tl = torch.where(top >= 0, lp.gather(1, top.clamp(min=0)), torch.zeros(n, 2).double())
    return ((o["logprob"] * gl).sum() + (o["entropy"] * gh).sum() + (tl * gt).sum(),
            ref.distill(x, target, ids, legal, temperature=t)[0]["loss"].sum())
  g1 = ref.logprobs_grad(logits, legal_at, legal, t, gl, gh, top, gt)[0]
  g2 = ref.distill(logits, target, ids, legal, temperature=t)[0]["grad"]
  for r in range(n):
    for i in range(v):
      up, down = logits.clone(), logits.clone()
      up[r, i] += h
      down[r, i] -= h
      a, b = value(up), value(down)
      assert abs(float((a[0] - b[0]) / (2 * h)) - float(g1[r, i])) < 1e-6
      assert abs(float((a[1] - b[1]) / (2 * h)) - float(g2[r, i])) < 1e-6


@gpu
@pytest.mark.parametrize("n,v,top", [(64, 7, 3), (33, 362, 5), (1, 40000, 20), (3, 131072, 8),
                                     (2, 200003, 4), (9, 5000, 20)])
def test_gpu_graph_replays_match_eager(require_gpu, n, v, top):
  """A captured training step (both operators and their gradients), replayed
  over new inputs with eager work between, equals the eager step bit for bit;
  two captured graphs do not disturb each other."""
  from os_amd import policy
  k = min(v, 7)

  def step(s):
    policy.logprobs_into(s["x"], s["h"], s["lp"], s["a"], None, s["ta"], s["tl"])
    policy.distill_into(s["x"], s["t"], s["loss"], s["th"], s["ids"], grad=s["grad"])

  def state(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = dict(device="cuda")
    return dict(x=torch.randn(n, v, generator=g, **f).bfloat16(),
                a=torch.randint(0, v, (n,), generator=g, **f), h=torch.empty(n, **f),
                lp=torch.empty(n, **f), ta=torch.empty(n, top, dtype=torch.int64, **f),
                tl=torch.empty(n, top, **f), t=torch.rand(n, k, generator=g, **f),
                ids=torch.randint(0, v, (n, k), generator=g, **f), loss=torch.empty(n, **f),
                th=torch.empty(n, **f), grad=torch.empty(n, v, dtype=torch.bfloat16, **f))
  graphs, states = [], []
  for seed in (1, 2):
    s = state(seed)
    step(s)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
      step(s)
    graphs.append(gr)
    states.append(s)
  for seed in (10, 11, 12, 13):
    for i, (gr, s) in enumerate(zip(graphs, states)):
      fresh = state(seed + 100 * i)
      for key in ("x", "a", "t", "ids"):
        s[key].copy_(fresh[key])
      for key in ("h", "lp", "tl", "loss", "th", "grad"):
        s[key].fill_(-7)
      s["ta"].fill_(-7)
      gr.replay()
      step(fresh)
      torch.cuda.synchronize()
      for key in s:
        assert torch.equal(s[key], fresh[key]), (key, seed, i)


@gpu
def test_gpu_autograd_step_captured(require_gpu):
  """The autograd forms inside a capture (torch.autograd.grad)."""
  from os_amd import policy
  n, v = 40, 82
  x = torch.randn(n, v, device="cuda")
  a = torch.randint(0, v, (n,), device="cuda")
  t = torch.rand(n, v, device="cuda")

  def step(leaf):
    r = policy.logprobs(leaf, a)
    loss, _ = policy.distill(leaf, t)
    return torch.autograd.grad(loss.mean() - r.logprob.mean() - 0.1 * r.entropy.mean(), leaf)[0]
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    step(x.clone().requires_grad_())
  torch.cuda.current_stream().wait_stream(side)
  torch.cuda.synchronize()
  leaf = x.clone().requires_grad_()
  gr = torch.cuda.CUDAGraph()
  with torch.cuda.graph(gr):
    out = step(leaf)
  for seed in range(4):
    with torch.no_grad():
      leaf.copy_(torch.randn(n, v, device="cuda"))
    gr.replay()
    want = step(leaf.detach().clone().requires_grad_())
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@gpu
def test_gpu_streams(require_gpu):
  """Calls on two streams at once equal the same calls one after the other."""
  from os_amd import policy
  xs = [torch.randn(n, 131072, device="cuda").to(torch.bfloat16) for n in (2, 3)]
  a = [torch.zeros(len(x), dtype=torch.int64, device="cuda") for x in xs]
  want = [policy.logprobs(x, i, top=20) for x, i in zip(xs, a)]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in xs]
  for _ in range(5):
    got = []
    for s, x, i in zip(streams, xs, a):
      with torch.cuda.stream(s):
        got.append(policy.logprobs(x, i, top=20))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
      for p, q in zip(g, w):
        assert torch.equal(p, q)


@gpu
def test_gpu_empty_batches(require_gpu):
  from os_amd import policy
  x = torch.zeros(0, 9, device="cuda", requires_grad=True)
  r = policy.logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
  assert r.logprob.shape == (0,) and r.top_action.shape == (0, 2)
  loss, _ = policy.distill(x, torch.zeros(0, 3, device="cuda"),
                           torch.zeros(0, 3, dtype=torch.int64, device="cuda"))
  grad, = torch.autograd.grad(loss.sum() + r.logprob.sum(), x)
  assert grad.shape == (0, 9)


@gpu
def test_gpu_repeats_are_bitwise_equal(require_gpu):
  """No result depends on the order waves run in (listed actions repeat)."""
  from os_amd import policy
  for v in (50, 700, 30000):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = torch.randn(200, v, generator=g, device="cuda")
    ids = torch.randint(0, min(v, 9), (200, 40), generator=g, device="cuda")
    t = torch.rand(200, 40, generator=g, device="cuda")
    first = None
    for _ in range(4):
      loss, h = torch.empty(200, device="cuda"), torch.empty(200, device="cuda")
      grad = torch.empty_like(x)
      policy.distill_into(x, t, loss, h, ids, grad=grad)
      if first is None:
        first = (loss, h, grad)
      for p, q in zip(first, (loss, h, grad)):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("game", ["connect_four", "go(board_size=5)"])
def test_gpu_search_then_train(require_gpu, game):
  """As they are used together: a PUCT search with the network's logits, its
  visit counts as the target, the loss and gradient, the log probability of
  the move played; then a step along the gradient lowers nothing but must run
  through the same calls again."""
  from os_amd import policy
  from os_amd.az import ExternalEvaluatorSearch, heads_into
  search = ExternalEvaluatorSearch(game)
  A, size = search.num_actions, int(np.prod(search.obs_shape))
  g = torch.Generator().manual_seed(3)
  w = (torch.randn(size, A + 1, generator=g) / size ** 0.5).cuda().requires_grad_()
  seen = {}

  class Net:
    def evaluate_into(self, obs, legal, kind, prior, value):
      with torch.no_grad():
        logits = obs.reshape(len(obs), -1) @ w
      seen.setdefault("obs", obs.clone())
      seen.setdefault("legal", legal.clone())
      heads_into(logits, legal, prior, value)
  acts, offs = E.make_roots(game, 48, seed_base=3, max_plies=4)
  out = search.run(acts, offs, np.arange(48, dtype=np.uint32), Net(), puct=True,
                   max_simulations=24, solve=False)
  ids, counts = policy.search_targets(out, "cuda")
  nchild = out["nchild"]
  for r in range(48):
    n = int(nchild[r])
    assert ids[r, :n].tolist() == list(out["child_action"][r, :n])
    assert counts[r, :n].tolist() == list(out["child_n"][r, :n])
    assert (ids[r, n:] == -1).all()
  move = torch.from_numpy(np.asarray(out["best_action"], np.int64)).cuda()
  logits = seen["obs"].reshape(48, -1) @ w
  pol = logits[:, :A]
  loss, h = policy.distill(pol, counts, ids, seen["legal"])
  r = policy.logprobs(pol, move, seen["legal"], top=3)
  total = loss.mean() - 0.5 * r.logprob.mean() - 0.1 * r.entropy.mean()
  grad, = torch.autograd.grad(total, w)
  x, lg = pol.detach().cpu(), seen["legal"].cpu()
  want, tol = ref.distill(x, counts.cpu(), ids.cpu(), lg,
                          weight=torch.full((48,), 1 / 48, dtype=torch.float64))
  close(loss, want["loss"], tol["loss"], "loss")
  one = torch.full((48,), 1.0 / 48)
  g2, t2 = ref.logprobs_grad(x, move.cpu(), lg, 1.0, -0.5 * one, -0.1 * one)
  o = seen["obs"].reshape(48, -1).cpu().double()
  full = o.t() @ (want["grad"] + g2)
  bound = o.t().abs() @ (tol["grad"] + t2 + 3 * ref.U * (want["grad"].abs() + g2.abs()))
  # the network's own product in float32: 48 terms
  bound = bound + 64 * ref.U * (o.t().abs() @ (want["grad"] + g2).abs())
  close(grad[:, :A], full, bound, "weights' gradient")
  with torch.no_grad():
    w -= 0.1 * grad
  loss, _ = policy.distill((seen["obs"].reshape(48, -1) @ w)[:, :A], counts, ids, seen["legal"])
  assert bool(torch.isfinite(loss).all())


@gpu
def test_gpu_documented_training_step(require_gpu):
  """INTEGRATION.md's block runs as written and reaches the model's weights."""
  import os
  import re
  doc = open(os.path.join(os.path.dirname(__file__), "..", "INTEGRATION.md")).read()
  block, = [b for b in re.findall(r"```python\n(.*?)```", doc, flags=re.S)
            if "policy.search_targets" in b]
  n, a = 20, 9
  nchild = np.array([r % 4 for r in range(n)], np.int32)
  model = torch.nn.Linear(5, a + 1).cuda()
  env = dict(model=model, num_actions=a, obs=torch.randn(n, 5, device="cuda"),
             legal=torch.ones(n, a, dtype=torch.uint8, device="cuda"),
             moves=torch.arange(n, device="cuda") % a - 1,
             out=dict(nchild=nchild, child_action=np.tile(np.arange(a, dtype=np.int32), (n, 1)),
                      child_n=np.ones((n, a), np.int32)))
  exec(block, env)
  want, tol = ref.distill(env["logits"].detach().cpu(), env["counts"].cpu(), env["ids"].cpu())
  close(env["loss"], want["loss"], tol["loss"], "loss")
  assert env["r"].top_action.shape == (n, 3)
  assert bool(torch.isfinite(model.weight.grad).all()) and bool((model.weight.grad[:a] != 0).any())
  assert bool((model.weight.grad[a] == 0).all())


@gpu
def test_gpu_selfplay_visits_as_target(require_gpu):
  """Engine.selfplay's dense int32 visits, padded moves among them."""
  from os_amd import policy
  eng = E.Engine("tic_tac_toe")
  acts, offs = E.roots_from_histories([[]] * 6)
  seeds = np.arange(12, dtype=np.uint32).reshape(6, 2)
  out = eng.selfplay(acts, offs, seeds, np.arange(6, dtype=np.uint32), record_visits=True,
                     max_simulations=30)
  visits = torch.from_numpy(np.ascontiguousarray(out["visits"]).astype(np.int32)).reshape(-1, 9)
  logits = torch.randn(len(visits), 9, generator=torch.Generator().manual_seed(0))
  want, tol = ref.distill(logits, visits)
  loss, h = policy.distill(logits.cuda(), visits.cuda())
  close(loss, want["loss"], tol["loss"], "loss")
  close(h, want["entropy"], tol["entropy"], "entropy")
  played = visits.sum(1) > 0
  assert bool(played.any()) and bool((loss.cpu()[~played] == 0).all())


# ---- refusals ----

def test_python_refuses_host_tensors():
  from os_amd import policy
  x = torch.zeros(4, 7)
  with pytest.raises(ValueError, match="GPU"):
    policy.logprobs(x)
  with pytest.raises(ValueError, match="GPU"):
    policy.distill(x, torch.zeros(4, 7))
  for bad in (torch.zeros(4, 7, dtype=torch.float64), torch.zeros(4, 7, dtype=torch.int32)):
    with pytest.raises(ValueError, match="float32"):
      policy.logprobs(bad)
  for bad in (torch.zeros(7), torch.zeros(2, 4, 7), torch.zeros(4, 0), torch.zeros(7, 4).t()):
    with pytest.raises(ValueError, match=r"\[N, A\]"):
      policy.logprobs(bad)
  for top in (-1, 65):
    with pytest.raises(ValueError, match="top"):
      policy.logprobs(x, top=top)


def _c_rows(**kw):
  f = dict(logits=4096, legal=None, num_rows=4, ld=7, legal_ld=7, num_actions=7, dtype=0,
           temperature=1.0, reserved=0)
  f.update(kw)
  return ctypes.byref(_lib.AzRows(**f))


def _c_target(**kw):
  f = dict(actions=4096, target=4096, actions_ld=3, target_ld=3, k=3, type=4, wide=0, reserved=0)
  f.update(kw)
  return ctypes.byref(_lib.AzTarget(**f))


BAD_ROWS = [dict(logits=None), dict(num_rows=-1), dict(ld=-1), dict(legal_ld=-1),
            dict(num_actions=0), dict(num_actions=2097153), dict(dtype=-1), dict(dtype=3),
            dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.inf),
            dict(temperature=math.nan), dict(temperature=1e-38), dict(reserved=1),
            dict(logits=4098), dict(logits=4097, dtype=1)]


@pytest.mark.parametrize("bad", BAD_ROWS, ids=str)
def test_abi_refuses_bad_rows(bad):
  """Every refusal comes before any launch (no GPU needed)."""
  L, r = _lib.lib, _c_rows(**bad)
  p = 4096
  if bad.get("logits", 1) is not None:
    assert L.os_az_rows_workspace(r, 0) < 0
  assert L.os_az_logprobs_async(r, p, 1, p, p, p, 0, None, None, None, 0, None) < 0
  assert L.os_az_logprobs_grad_async(r, p, 1, p, p, 0, None, p, 1, p, 1, None, p, 1 << 23, None) < 0
  assert L.os_az_distill_async(r, _c_target(), None, p, p, p, None, 0, None, 0, None) < 0
  assert L.os_az_distill_grad_async(r, _c_target(), p, 1, p, p, 1 << 23, None) < 0
  assert L.os_last_error()


def test_abi_refuses_bad_calls():
  L, r, p = _lib.lib, _c_rows(), 4096
  assert L.os_az_rows_workspace(None, 0) < 0
  for top in (-1, 65):
    assert L.os_az_rows_workspace(r, top) < 0
    assert L.os_az_logprobs_async(r, p, 1, p, p, p, top, p, p, None, 0, None) < 0
    assert L.os_az_logprobs_grad_async(r, p, 1, p, p, top, p, p, 1, p, 1, p, p, 7, None) < 0
  # missing buffers
  assert L.os_az_logprobs_async(r, p, 1, None, p, p, 0, None, None, None, 0, None) < 0
  assert L.os_az_logprobs_async(r, None, 1, p, p, p, 0, None, None, None, 0, None) < 0
  assert L.os_az_logprobs_async(r, p, 1, p, None, p, 0, None, None, None, 0, None) < 0
  assert L.os_az_logprobs_async(r, p, 1, p, p, p, 2, None, p, None, 0, None) < 0
  assert L.os_az_logprobs_async(r, p, 1, p, p, p, 2, p, None, None, 0, None) < 0
  g = L.os_az_logprobs_grad_async
  assert g(r, p, 1, p, None, 0, None, p, 1, p, 1, None, p, 7, None) < 0
  assert g(r, p, 1, p, p, 0, None, p, 1, p, 1, None, None, 7, None) < 0
  assert g(r, p, 1, None, p, 0, None, p, 1, p, 1, None, p, 7, None) < 0
  assert g(r, None, 1, p, p, 0, None, p, 1, p, 1, None, p, 7, None) < 0
  assert g(r, p, 1, p, p, 2, None, p, 1, p, 1, p, p, 7, None) < 0
  assert g(r, p, 1, p, p, 0, None, p, 1, p, 1, None, p, 6, None) < 0
  assert g(r, p, 1, p, p, 0, None, p, -1, p, 1, None, p, 7, None) < 0
  assert g(r, p, 1, p, p, 0, None, p, 1, p, 1, None, 4097, 7, None) < 0
  d = L.os_az_distill_async
  for bad in (dict(k=-1), dict(k=1025), dict(type=-1), dict(type=5), dict(actions_ld=-1),
              dict(target_ld=-1), dict(reserved=2), dict(target=None), dict(actions=None)):
    assert d(r, _c_target(**bad), None, p, p, p, None, 0, None, 0, None) < 0, bad
    assert L.os_az_distill_grad_async(r, _c_target(**bad), p, 1, p, p, 7, None) < 0, bad
  assert d(r, None, None, p, p, p, None, 0, None, 0, None) < 0
  assert d(r, _c_target(), None, None, p, p, None, 0, None, 0, None) < 0
  assert d(r, _c_target(), None, p, p, p, p, 6, None, 0, None) < 0
  assert L.os_az_distill_grad_async(r, _c_target(), p, 1, None, p, 7, None) < 0
  assert L.os_az_distill_grad_async(r, _c_target(), p, 1, p, None, 7, None) < 0
  assert L.os_az_distill_grad_async(r, _c_target(), p, -1, p, p, 7, None) < 0
  # no rows: nothing to do, nothing launched
  none = _c_rows(num_rows=0, logits=None)
  assert L.os_az_logprobs_async(none, None, 1, None, None, None, 0, None, None, None, 0, None) == 0
  assert d(none, _c_target(), None, None, None, None, None, 0, None, 0, None) == 0
  assert L.os_az_distill_grad_async(none, _c_target(), None, 0, None, None, 7, None) == 0
  assert g(none, None, 1, None, None, 0, None, None, 0, None, 0, None, None, 7, None) == 0


@gpu
def test_gpu_python_refusals(require_gpu):
  from os_amd import policy
  n, a = 6, 9
  f = dict(device="cuda")
  x = torch.zeros(n, a, **f)
  act = torch.zeros(n, dtype=torch.int64, **f)
  legal = torch.ones(n, a, dtype=torch.uint8, **f)
  out = torch.zeros(n, **f)
  t = torch.ones(n, 3, **f)
  ids = torch.zeros(n, 3, dtype=torch.int64, **f)
  policy.logprobs(x, act, legal, top=2)
  policy.distill(x, t, ids, legal)
  bad = [
      lambda: policy.logprobs(x, act.float()), lambda: policy.logprobs(x, act[:3]),
      lambda: policy.logprobs(x, act.cpu()), lambda: policy.logprobs(x, act, legal.cpu()),
      lambda: policy.logprobs(x, act, legal.float()), lambda: policy.logprobs(x, act, legal[:, :5]),
      lambda: policy.logprobs(x, act, legal[0, :5]),
      lambda: policy.logprobs(x, act, torch.ones(a, n, dtype=torch.uint8, **f).t()),
      lambda: policy.logprobs(x, temperature=0), lambda: policy.logprobs(x, temperature=math.nan),
      lambda: policy.logprobs_into(x, out, out.clone()),
      lambda: policy.logprobs_into(x, out, None, act),
      lambda: policy.logprobs_into(x, None),
      lambda: policy.logprobs_into(x, out.double()),
      lambda: policy.logprobs_into(x, out[:3]),
      lambda: policy.logprobs_into(x, torch.zeros(n, 2, **f)[:, 0]),
      lambda: policy.logprobs_into(x, out, top_action=ids),
      lambda: policy.logprobs_into(x, out, top_action=ids.int(), top_logprob=t),
      lambda: policy.logprobs_into(x, out, stats=t),
      lambda: policy.logprobs_into(x, out, top_action=torch.zeros(n, 65, dtype=torch.int64, **f),
                                   top_logprob=torch.zeros(n, 65, **f)),
      lambda: policy.distill(x, t), lambda: policy.distill(x, t, ids, kind="counts"),
      lambda: policy.distill(x, t, ids.float()), lambda: policy.distill(x, t, ids[:, :2]),
      lambda: policy.distill(x, t.double(), ids), lambda: policy.distill(x, t.int(), ids, kind="logits"),
      lambda: policy.distill(x, t.bfloat16(), ids), lambda: policy.distill(x, t[:3], ids[:3]),
      lambda: policy.distill(x, t.cpu(), ids), lambda: policy.distill(x, t, ids.cpu()),
      lambda: policy.distill(x, t.clone().requires_grad_(), ids),
      lambda: policy.distill(x, torch.ones(3, n, **f).t(), ids),
      lambda: policy.distill(x, torch.ones(n, 1025, **f), torch.zeros(n, 1025, dtype=torch.int32, **f)),
      lambda: policy.distill_into(x, t, None, None, ids),
      lambda: policy.distill_into(x, t, out, None, ids, weight=out),
      lambda: policy.distill_into(x, t, out, None, ids, grad=x),
      lambda: policy.distill_into(x, t, out, None, ids, grad=x.bfloat16()),
      lambda: policy.distill_into(x, t, out, None, ids, grad=torch.zeros(n, a + 1, **f)),
      lambda: policy.distill_into(x, t, out, None, ids, grad=torch.zeros(1, a, **f).expand(n, a)),
      lambda: policy.distill_into(x, t, out, None, ids, grad=torch.zeros(a, n, **f).t()),
  ]
  for i, call in enumerate(bad):
    with pytest.raises(ValueError):
      call()
      raise AssertionError("call %d was not refused" % i)
  # disjoint columns of one buffer are no overlap; shifted rows are
  both = torch.zeros(n, 2 * a, **f)
  policy.distill_into(both[:, :a], t, out, None, ids, grad=both[:, a:])
  flat = torch.zeros(n * a + 4, **f)
  with pytest.raises(ValueError, match="overlap"):
    policy.distill_into(flat[:n * a].view(n, a), t, out, None, ids, grad=flat[4:].view(n, a))
  # the second derivative is refused, not wrong
  leaf = x.clone().requires_grad_()
  g, = torch.autograd.grad(policy.distill(leaf, t, ids)[0].sum(), leaf, create_graph=True)
  with pytest.raises(RuntimeError):
    g.sum().backward()
