"""Policy operators on a network's logits, on the GPU (include/os_mcts.h,
"Policy operators"; csrc/os_policy.hip).

`os_amd.az.heads_into` turns a network's logits into the priors a search reads;
these are what a program that trains or reports a policy does with the same
logits.  `logits` is [N, A] (float32, bfloat16 or float16, unit column stride,
any row stride: the policy columns `out[:, :A]` of rows that end in the value's
logit fit as they are) and `legal` its optional mask (uint8 or bool, [N, A], or
[A] for all rows; 0 excludes an action, and so does a logit of -inf).

  logprobs       log probability of each row's given action (a played move, a
                 sampled token), the row's entropy and its `top` most likely
                 actions; differentiable
  distill        cross entropy against a target on listed actions: the visit
                 counts of searches (`search_targets`), self-play's dense
                 `visits`, or a teacher network's top logits; differentiable
  logprobs_into, distill_into
                 the same into given tensors, without autograd: nothing but
                 the kernels' own launches, so a training or serving step can
                 be captured into a HIP graph.  distill_into writes the loss
                 and the logits' gradient together, from one read of the
                 logits where a row fits the compute unit.

Rows are independent.  A row without any allowed action is empty: entropy 0,
gradient 0.  A NaN or +inf logit on an allowed action makes its own row's
results NaN.  Arithmetic is float32; gradients are rounded once to the logits'
type.  Calls run on the current stream of the logits' device.

Gradients of the first order only.  Capture a training step with the `_into`
calls, or with torch.autograd.grad: like any autograd operator, a `.backward()`
captured while an eager graph of the same leaves is alive is not supported by
torch.
"""
import ctypes
from typing import NamedTuple, Optional

import numpy as np
import torch

from . import _lib
from ._lib import check, lib

_DTYPES = {torch.float32: _lib.AZ_F32, torch.bfloat16: _lib.AZ_BF16, torch.float16: _lib.AZ_F16}
_TARGETS = {
    ("logits", torch.float32): _lib.AZ_LOGITS_F32,
    ("logits", torch.bfloat16): _lib.AZ_LOGITS_BF16,
    ("logits", torch.float16): _lib.AZ_LOGITS_F16,
    ("weights", torch.float32): _lib.AZ_WEIGHTS_F32,
    ("weights", torch.int32): _lib.AZ_WEIGHTS_I32,
}
_IDS = {torch.int32: 0, torch.int64: 1}


class LogProbs(NamedTuple):
  """Results of logprobs (float32; top_action int64)."""
  logprob: Optional[torch.Tensor]      # [N], None without actions
  entropy: torch.Tensor                # [N]
  top_action: Optional[torch.Tensor]   # [N, top], None when top = 0
  top_logprob: Optional[torch.Tensor]  # [N, top]


def _rows(logits, legal, temperature):
  """The checked os_az_rows of a call; its tensors must outlive it."""
  if logits.dtype not in _DTYPES:
    raise ValueError("logits must be float32, bfloat16 or float16")
  if logits.dim() != 2 or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
    raise ValueError("logits must be [N, A] with unit column stride")
  if not logits.is_cuda:
    raise ValueError("logits must be on a GPU")
  n, a = logits.shape
  if a > _lib.AZ_MAX_ACTIONS:
    raise ValueError("more than %d actions" % _lib.AZ_MAX_ACTIONS)
  t = float(temperature)
  if not 1e-30 <= t <= 1e30:
    raise ValueError("temperature must be in [1e-30, 1e30]")
  r = _lib.AzRows(logits=logits.data_ptr(), num_rows=n, ld=logits.stride(0), num_actions=a,
                  dtype=_DTYPES[logits.dtype], temperature=t)
  if legal is not None:
    if legal.dtype not in (torch.uint8, torch.bool):
      raise ValueError("legal must be uint8 or bool")
    if tuple(legal.shape) not in ((n, a), (a,)) or (a > 1 and legal.stride(-1) != 1):
      raise ValueError("legal must be [N, A] or [A] with unit column stride")
    if legal.device != logits.device:
      raise ValueError("legal must be on the logits' GPU")
    r.legal = legal.data_ptr()
    r.legal_ld = legal.stride(0) if legal.dim() == 2 else 0
  return r


def _like(what, x, logits, dtype, *shape):
  """Checks an optional result or per-row tensor: contiguous, of this shape."""
  if x is None:
    return None
  if x.dtype != dtype or tuple(x.shape) != shape or not x.is_contiguous():
    raise ValueError("%s must be contiguous %s %s" % (what, dtype, list(shape)))
  if x.device != logits.device:
    raise ValueError("%s must be on the logits' GPU" % what)
  return x.data_ptr()


def _actions(actions, logits):
  """(address, wide) of the given actions, one a row."""
  if actions is None:
    return None, 0
  if actions.dtype not in _IDS:
    raise ValueError("actions must be int32 or int64")
  return (_like("actions", actions, logits, actions.dtype, logits.shape[0]),
          _IDS[actions.dtype])


def _target(target, target_actions, logits, kind):
  """The checked os_az_target of a call."""
  n, a = logits.shape
  if kind not in ("logits", "weights"):
    raise ValueError("kind must be 'logits' or 'weights'")
  if (kind, target.dtype) not in _TARGETS:
    raise ValueError("target must be float32, bfloat16 or float16 logits, or float32 or int32 "
                     "weights")
  if target.requires_grad:
    raise ValueError("the target is not differentiated: detach() it")
  if target.dim() != 2 or target.shape[0] != n or (target.shape[1] > 1 and target.stride(1) != 1):
    raise ValueError("target must be [N, K] with unit column stride")
  k = target.shape[1]
  if k > _lib.AZ_MAX_TARGETS:
    raise ValueError("more than %d listed actions" % _lib.AZ_MAX_TARGETS)
  if target.device != logits.device:
    raise ValueError("target must be on the logits' GPU")
  t = _lib.AzTarget(target=target.data_ptr(), target_ld=target.stride(0), k=k,
                    type=_TARGETS[kind, target.dtype])
  if target_actions is None:
    if k != a:
      raise ValueError("a target without target_actions must be [N, A]")
    return t
  if target_actions.dtype not in _IDS:
    raise ValueError("target_actions must be int32 or int64")
  if tuple(target_actions.shape) != (n, k) or (k > 1 and target_actions.stride(1) != 1):
    raise ValueError("target_actions must be shaped as target, with unit column stride")
  if target_actions.device != logits.device:
    raise ValueError("target_actions must be on the logits' GPU")
  t.actions = target_actions.data_ptr()
  t.actions_ld = target_actions.stride(0)
  t.wide = _IDS[target_actions.dtype]
  return t


def _grad_buffer(grad, logits):
  n, a = logits.shape
  if grad.dtype != logits.dtype or tuple(grad.shape) != (n, a):
    raise ValueError("grad must have the logits' type and shape")
  if grad.device != logits.device:
    raise ValueError("grad must be on the logits' GPU")
  if (a > 1 and grad.stride(1) != 1) or (n > 1 and grad.stride(0) < a):
    raise ValueError("grad must have unit column stride and rows that do not overlap")
  if n > 0:
    size = grad.element_size()
    g0, x0 = grad.data_ptr(), logits.data_ptr()
    if (g0 < x0 + ((n - 1) * logits.stride(0) + a) * size
        and x0 < g0 + ((n - 1) * grad.stride(0) + a) * size
        and not _interleaved(grad, logits, a)):
      raise ValueError("grad overlaps the logits")
  return grad.data_ptr(), max(grad.stride(0), a)


def _interleaved(grad, logits, a):
  """Whether two tensors of one row stride are disjoint columns of it (the
  halves of one buffer)."""
  ld = logits.stride(0)
  if grad.stride(0) != ld:
    return False
  off = (grad.data_ptr() - logits.data_ptr()) // grad.element_size() % ld
  return off >= a and off + a <= ld


def _launch(fn, logits, *args):
  """Calls a C entry on the current stream of the logits' device."""
  dev = logits.device
  if dev.index != torch.cuda.current_device():
    with torch.cuda.device(dev):
      check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))
  else:
    check(fn(*args, torch.cuda.current_stream(dev).cuda_stream))


def _workspace(rows, top, logits):
  n = lib.os_az_rows_workspace(ctypes.byref(rows), top)
  if n < 0:
    check(int(n))
  if n == 0:
    return None, None, 0
  w = torch.empty(n, dtype=torch.uint8, device=logits.device)
  return w, w.data_ptr(), n


def logprobs_into(logits, entropy, logprob=None, actions=None, legal=None, top_action=None,
                  top_logprob=None, temperature=1.0, stats=None):
  """logprobs into given tensors: entropy and logprob float32 [N], top_action
  int64 and top_logprob float32 [N, top], stats float32 [N, 2] (what the
  gradient needs; optional).  logprob and actions go together, and so do the
  top pair."""
  rows = _rows(logits, legal, temperature)
  n = logits.shape[0]
  act, wide = _actions(actions, logits)
  if (logprob is None) != (actions is None):
    raise ValueError("logprob and actions go together")
  if (top_action is None) != (top_logprob is None):
    raise ValueError("top_action and top_logprob go together")
  if entropy is None:
    raise ValueError("entropy is needed")
  top = 0
  if top_action is not None:
    if top_action.dim() != 2 or top_action.shape[1] > _lib.AZ_MAX_TOP:
      raise ValueError("top_action must be [N, top], top <= %d" % _lib.AZ_MAX_TOP)
    top = top_action.shape[1]
  out = (_like("logprob", logprob, logits, torch.float32, n),
         _like("entropy", entropy, logits, torch.float32, n),
         _like("stats", stats, logits, torch.float32, n, 2), top,
         _like("top_action", top_action, logits, torch.int64, n, top),
         _like("top_logprob", top_logprob, logits, torch.float32, n, top))
  keep, work, size = _workspace(rows, top, logits)
  _launch(lib.os_az_logprobs_async, logits, ctypes.byref(rows), act, wide, *out, work, size)
  del keep


def distill_into(logits, target, loss, target_entropy=None, target_actions=None, legal=None,
                 kind="weights", temperature=1.0, weight=None, grad=None, stats=None):
  """distill into given tensors: loss and target_entropy float32 [N], stats
  float32 [N, 2] (what the gradient needs; optional).  With `grad` (the logits'
  type and shape, any row stride) also the logits' gradient of
  (weight * loss).sum(); weight float32 [N], None: 1."""
  rows = _rows(logits, legal, temperature)
  n = logits.shape[0]
  t = _target(target, target_actions, logits, kind)
  if loss is None:
    raise ValueError("loss is needed")
  if weight is not None and grad is None:
    raise ValueError("weight scales the gradient: it needs grad")
  g, ld = (None, 0) if grad is None else _grad_buffer(grad, logits)
  out = (_like("weight", weight, logits, torch.float32, n),
         _like("loss", loss, logits, torch.float32, n),
         _like("target_entropy", target_entropy, logits, torch.float32, n),
         _like("stats", stats, logits, torch.float32, n, 2))
  keep, work, size = _workspace(rows, 0, logits)
  _launch(lib.os_az_distill_async, logits, ctypes.byref(rows), ctypes.byref(t), *out, g, ld, work,
          size)
  del keep


def _per_row(g):
  """(address, element stride) of a float32 [N] upstream gradient: an expanded
  one (of a sum or a mean) is read as it is."""
  return (None, 0) if g is None else (g.data_ptr(), g.stride(0))


class _LogProbs(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, actions, legal, top, temperature):
    n = logits.shape[0]
    f32 = dict(dtype=torch.float32, device=logits.device)
    entropy = torch.empty(n, **f32)
    stats = torch.empty(n, 2, **f32)
    logprob = None if actions is None else torch.empty(n, **f32)
    top_action = top_logprob = None
    if top > 0:
      top_action = torch.empty(n, top, dtype=torch.int64, device=logits.device)
      top_logprob = torch.empty(n, top, **f32)
      ctx.mark_non_differentiable(top_action)
    logprobs_into(logits, entropy, logprob, actions, legal, top_action, top_logprob, temperature,
                  stats)
    ctx.save_for_backward(logits, actions, legal, entropy, stats, top_action)
    ctx.temperature = temperature
    ctx.set_materialize_grads(False)
    return logprob, entropy, top_action, top_logprob

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, g_logprob, g_entropy, _, g_top):
    if g_logprob is None and g_entropy is None and g_top is None:
      return (None,) * 5
    logits, actions, legal, entropy, stats, top_action = ctx.saved_tensors
    rows = _rows(logits, legal, ctx.temperature)
    act, wide = _actions(actions, logits)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    top = 0
    if g_top is not None:
      g_top = g_top.contiguous()
      top = g_top.shape[1]
    _launch(lib.os_az_logprobs_grad_async, logits, ctypes.byref(rows), act, wide,
            entropy.data_ptr(), stats.data_ptr(), top,
            None if top == 0 else top_action.data_ptr(), *_per_row(g_logprob),
            *_per_row(g_entropy), None if top == 0 else g_top.data_ptr(), grad.data_ptr(),
            logits.shape[1])
    return grad, None, None, None, None


class _Distill(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, target, target_actions, legal, kind, temperature):
    n = logits.shape[0]
    f32 = dict(dtype=torch.float32, device=logits.device)
    loss, entropy, stats = torch.empty(n, **f32), torch.empty(n, **f32), torch.empty(n, 2, **f32)
    distill_into(logits, target, loss, entropy, target_actions, legal, kind, temperature,
                 stats=stats)
    ctx.save_for_backward(logits, target, target_actions, legal, stats)
    ctx.kind, ctx.temperature = kind, temperature
    ctx.mark_non_differentiable(entropy)
    ctx.set_materialize_grads(False)
    return loss, entropy

  @staticmethod
  @torch.autograd.function.once_differentiable
  def backward(ctx, g_loss, _):
    if g_loss is None:
      return (None,) * 6
    logits, target, target_actions, legal, stats = ctx.saved_tensors
    rows = _rows(logits, legal, ctx.temperature)
    t = _target(target, target_actions, logits, ctx.kind)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _launch(lib.os_az_distill_grad_async, logits, ctypes.byref(rows), ctypes.byref(t),
            *_per_row(g_loss), stats.data_ptr(), grad.data_ptr(), logits.shape[1])
    return grad, None, None, None, None, None


def logprobs(logits, actions=None, legal=None, top=0, temperature=1.0):
  """LogProbs(logprob, entropy, top_action, top_logprob) of the policies
  softmax(logits / temperature) over the allowed actions.

  actions (int32 or int64 [N]): logprob[r] is the log probability of
  actions[r]; -inf for an action that is excluded, 0 for a negative one
  (padding, without a gradient), NaN for one >= A.  entropy is in nats.  The
  `top` (<= 64) most likely actions are in descending order, equal logits by
  the lower action; past the row's allowed actions top_action is -1 and
  top_logprob -inf.  Gradients flow from logprob, entropy and top_logprob to
  the logits; an excluded action's is 0."""
  top = int(top)
  if not 0 <= top <= _lib.AZ_MAX_TOP:
    raise ValueError("top must be in [0, %d]" % _lib.AZ_MAX_TOP)
  return LogProbs(*_LogProbs.apply(logits, actions, legal, top, float(temperature)))


def distill(logits, target, target_actions=None, legal=None, kind="weights", temperature=1.0):
  """(loss, target_entropy), float32 [N]: the cross entropy -sum_j q_j log p of
  the policies softmax(logits / temperature) over the allowed actions against
  the target distribution q, and q's entropy; loss - target_entropy is the
  Kullback-Leibler divergence from q.

  Entry j of row r is action target_actions[r, j] (int32 or int64 [N, K], K <=
  1024; negative: padding; listed twice counts twice) with target[r, j], which
  is a weight (kind="weights", float32 or int32: q = w / sum w, weights not
  above 0 count as 0) or a teacher's logit (kind="logits": q =
  softmax(target / temperature) over the row's entries).  Without
  target_actions the target is [N, A], entry j action j.

  The loss is 0 for a row without a target, +inf where an excluded action has
  mass, NaN where an action >= A is listed.  The gradient reaches the logits,
  not the target; an excluded action's is 0."""
  return _Distill.apply(logits, target, target_actions, legal, kind, float(temperature))


def search_targets(out, device):
  """(target_actions, counts), int32 [R, K] on `device`: the root children and
  visit counts of a batch of searches (`Engine.mcts_batch`,
  `ExternalEvaluatorSearch.run`) as distill's target, K the most children of
  any root, padded with action -1."""
  nchild = np.asarray(out["nchild"])
  k = max(1, int(nchild.max(initial=0)))
  there = np.arange(k)[None, :] < nchild[:, None]
  acts = np.where(there, out["child_action"][:, :k], -1).astype(np.int32)
  counts = np.where(there, out["child_n"][:, :k], 0).astype(np.int32)
  return torch.from_numpy(acts).to(device), torch.from_numpy(counts).to(device)
