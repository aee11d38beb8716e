"""The policy operators (os_amd/policy.py) from their formulas, in 64 bits on
the CPU, with the rounding bounds their float32 kernels are held to."""
import math

import torch

U = 2.0 ** -24  # half a step of float32, relative
# The gradients' p = e f is a float32 exponential e of (x - m) / T <= 0 times
# f = 1 / sum e <= 1.  The exponential keeps no subnormal results: e < 2^-126 is
# 0, so p is off by up to 2^-126 beside its relative error.
LEAST = 2.0 ** -126


def adds(v):
  """Roundings a sum over v actions may meet in one chain: each lane adds at
  most 128 elements of a row part, lanes, waves and parts are joined in trees
  (counted generously: 64 more), every exponential is off by less than 4 half
  steps, and its argument's own error (3 half steps of d, averaging at most
  log2 v under p) adds 3 log2 v."""
  return 128 + 64 + 4 + 3 * math.log2(max(v, 2))


def masked(logits, legal, temperature):
  x = logits.double() / temperature
  if legal is not None:
    x = torch.where(legal.bool().expand_as(x), x, torch.full_like(x, -math.inf))
  return x


def softmax(x):
  """(p, log p), empty rows: p = 0.  (log p from x - m: m + log s would lose
  log s next to an m like the type's lowest value.)"""
  m = x.amax(1, keepdim=True)
  m = torch.where(m == -math.inf, torch.zeros_like(m), m)
  s = torch.exp(x - m).sum(1, keepdim=True)
  s = torch.where(s == 0, torch.ones_like(s), s)
  logp = (x - m) - torch.log(s)
  return torch.exp(logp), logp


def plogp(p, logp):
  return torch.where(p > 0, p * logp, torch.where(torch.isnan(p), p, torch.zeros_like(p)))


def logprobs(logits, actions=None, legal=None, top=0, temperature=1.0):
  """dict(logprob, entropy, top_action, top_logprob) and the bounds dict."""
  x = masked(logits, legal, temperature)
  n, v = x.shape
  p, logp = softmax(x)
  out, tol = {}, {}
  a_ = adds(v)
  out["entropy"] = -plogp(p, logp).sum(1)
  # H = ln 2 (l - t / s), |l| and |t / s| <= log2 v
  tol["entropy"] = torch.full((n,), 3 * a_ * U * (1 + math.log2(max(v, 2))), dtype=torch.float64)
  span = x - x.amax(1, keepdim=True)  # (x - m) / T

  def lp_tol(lp, d):
    return U * (a_ + 4 * lp.abs() + 6 * d.abs() + 2 * math.log2(max(v, 2)))
  if actions is not None:
    a = actions.long()
    ok = (a >= 0) & (a < v)
    i = torch.where(ok, a, torch.zeros_like(a))[:, None]
    g = logp.gather(1, i)[:, 0]
    g = torch.where(a < 0, torch.zeros_like(g), g)
    g = torch.where(a >= v, torch.full_like(g, math.nan), g)
    out["logprob"] = g
    tol["logprob"] = lp_tol(g, span.gather(1, i)[:, 0])
  if top:
    raw = logits.double()
    if legal is not None:
      raw = torch.where(legal.bool().expand_as(raw), raw, torch.full_like(raw, -math.inf))
    bad = torch.isnan(p).any(1, keepdim=True)
    val, ids = torch.sort(raw, dim=1, descending=True, stable=True)
    if v < top:
      val = torch.cat([val, torch.full((n, top - v), -math.inf, dtype=val.dtype)], 1)
      ids = torch.cat([ids, torch.zeros(n, top - v, dtype=ids.dtype)], 1)
    val, ids = val[:, :top], ids[:, :top]
    none = (val == -math.inf) | bad
    lp = logp.gather(1, ids)
    lp = torch.where(val == -math.inf, val, lp)
    out["top_logprob"] = torch.where(bad, torch.full_like(lp, math.nan), lp)
    out["top_action"] = torch.where(none, torch.full_like(ids, -1), ids)
    tol["top_logprob"] = lp_tol(lp, span.gather(1, ids))
  return out, tol


def logprobs_grad(logits, actions=None, legal=None, temperature=1.0, g_logprob=None,
                  g_entropy=None, top_action=None, g_top=None):
  """(gradient, its bound before the rounding to the logits' type)."""
  x = masked(logits, legal, temperature)
  n, v = x.shape
  p, logp = softmax(x)
  h = -plogp(p, logp).sum(1, keepdim=True)
  zero = torch.zeros(n, dtype=torch.float64)
  listed = torch.zeros_like(x)
  amount = torch.zeros_like(x)
  total, size = zero.clone(), zero.clone()
  ids, gs = [], []
  if g_logprob is not None:
    ids.append(actions.long()[:, None])
    gs.append(g_logprob.double()[:, None])
  if g_top is not None:
    ids.append(top_action.long())
    gs.append(g_top.double())
  if ids:
    ids, gs = torch.cat(ids, 1), torch.cat(gs, 1)
    bad = (ids >= v).any(1)
    gs = torch.where(ids >= 0, gs, torch.zeros_like(gs))
    i = ids.clamp(0, v - 1)
    gs_in = torch.where(ids < v, gs, torch.zeros_like(gs))
    listed.scatter_add_(1, i, gs_in)
    amount.scatter_add_(1, i, gs_in.abs())
    total, size = gs.sum(1), gs.abs().sum(1)
    total = torch.where(bad, torch.full_like(total, math.nan), total)
  gh = zero if g_entropy is None else g_entropy.double()
  grad = -p * total[:, None] - gh[:, None] * (plogp(p, logp) + p * h) + listed
  grad = torch.where(x > -math.inf, grad, torch.where(x == -math.inf, torch.zeros_like(grad), grad))
  lp = torch.where(p > 0, logp.abs(), torch.zeros_like(p))
  span = torch.where(p > 0, (x - x.amax(1, keepdim=True)).abs(), torch.zeros_like(x))
  part = p * (size[:, None] + gh.abs()[:, None] * (lp + h.abs() + 1))
  k = 0 if not torch.is_tensor(ids) else ids.shape[1]
  bound = U * ((3 * adds(v) * (1 + math.log2(max(v, 2))) + 12 * span + k) * part
               + (k + 4) * amount)
  # (p |log p| <= LEAST |log LEAST| < 104 LEAST where p <= LEAST)
  bound = bound + LEAST * (size + gh.abs() * (104 + 1 + h[:, 0].abs()))[:, None]
  return grad / temperature, bound / temperature


def target_mass(target, ids, kind, temperature):
  """(q [N, K], relative bound [N, K])."""
  there = torch.ones_like(target, dtype=torch.bool) if ids is None else ids >= 0
  t = target.double()
  if kind == "weights":
    w = torch.where(there & ~(t <= 0), t, torch.zeros_like(t))
    err = torch.full_like(w, 4.0)
  else:
    z = torch.where(there, t / temperature, torch.full_like(t, -math.inf))
    zm = z.amax(1, keepdim=True) if z.shape[1] else z.sum(1, keepdim=True)
    zm = torch.where(zm == -math.inf, torch.zeros_like(zm), zm)
    w = torch.exp(z - zm)
    err = 8 + 6 * torch.where(w > 0, (z - zm).abs(), torch.zeros_like(w))
  total = w.sum(1, keepdim=True)
  q = torch.where(total == 0, torch.zeros_like(w), w / total)
  # the sum's own error: K / 64 additions a lane, a tree, each term's own
  mean = (q * err).sum(1, keepdim=True)
  return q, U * (err + mean + target.shape[1] / 64 + 16)


def distill(logits, target, ids=None, legal=None, kind="weights", temperature=1.0, weight=None):
  """dict(loss, entropy, grad) and the bounds dict (grad's before rounding)."""
  x = masked(logits, legal, temperature)
  n, v = x.shape
  p, logp = softmax(x)
  q, q_err = target_mass(target, ids, kind, temperature)
  i = torch.arange(v).expand(n, v) if ids is None else ids.long()
  ok = (i >= 0) & (i < v)
  j = i.clamp(0, v - 1)
  at = logp.gather(1, j)
  nil = torch.zeros_like(q)
  terms = torch.where((q > 0) & ok, -q * at, nil)
  terms = torch.where(torch.isnan(q), q, terms)
  loss = terms.sum(1)
  bad = (i >= v).any(1)
  loss = torch.where(bad, torch.full_like(loss, math.nan), loss)
  hq = -plogp(q, torch.log(torch.where(q > 0, q, torch.ones_like(q)))).sum(1)
  span = (x - x.amax(1, keepdim=True)).gather(1, j).abs()
  fin = (q > 0) & ok & torch.isfinite(at)
  k = q.shape[1]
  each = torch.where(fin, q * (at.abs() * (q_err + U * (k / 64 + 16))
                               + U * (adds(v) + 6 * span + 4 * at.abs()
                                      + 2 * math.log2(max(v, 2)))), nil)
  lq = torch.where(q > 0, torch.log(torch.where(q > 0, q, torch.ones_like(q))).abs(), nil)
  out = dict(loss=loss, entropy=hq)
  tol = dict(loss=each.sum(1),
             entropy=(q * (lq + 1) * (q_err + U * (k / 64 + 24))).sum(1))
  w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
  sq = torch.zeros_like(x)
  sq_err = torch.zeros_like(x)
  qk = torch.where(ok, q, nil)
  sq.scatter_add_(1, j, qk)
  sq_err.scatter_add_(1, j, torch.where(ok, q * (q_err + U * (k + 4)), nil))
  mass = q.sum(1, keepdim=True)
  mass = torch.where(bad[:, None], torch.full_like(mass, math.nan), mass)
  grad = p * mass - sq
  grad = torch.where(x == -math.inf, torch.zeros_like(grad), grad)
  sp = torch.where(p > 0, (x - x.amax(1, keepdim=True)).abs(), torch.zeros_like(x))
  s = (w / temperature)[:, None]
  out["grad"] = grad * s
  tol["grad"] = (p * U * (3 * adds(v) + 12 * sp + 16) + sq_err + 4 * U * sq + LEAST) * s.abs()
  return out, tol


def rounding(t, ref):
  """The bound a value rounded once to type t adds: half a step, or half the
  least subnormal."""
  f = torch.finfo(t)
  return ref.abs() * (f.eps / 2) + f.smallest_normal * f.eps
