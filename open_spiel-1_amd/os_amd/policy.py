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

Gradients of the first order and in reverse mode only: a forward-mode tangent
is refused, not dropped.  Capture a training step with the `_into`
calls, or with torch.autograd.grad: like any autograd operator, a `.backward()`
captured while an eager graph of the same leaves is alive is not supported by
torch.
"""
import struct
from typing import NamedTuple, Optional

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check, lib

_F32 = torch.float32
_DTYPES = {torch.float32: _lib.AZ_F32, torch.bfloat16: _lib.AZ_BF16, torch.float16: _lib.AZ_F16}
_TARGETS = {
    "logits": {torch.float32: _lib.AZ_LOGITS_F32, torch.bfloat16: _lib.AZ_LOGITS_BF16,
               torch.float16: _lib.AZ_LOGITS_F16},
    "weights": {torch.float32: _lib.AZ_WEIGHTS_F32, torch.int32: _lib.AZ_WEIGHTS_I32},
}
_IDS = {torch.int32: 0, torch.int64: 1}

# os_az_rows and os_az_target, packed as C lays them out: for the smallest
# batches a call costs what its checks cost, and a ctypes.Structure takes four
# times as long to fill.
_ROWS = struct.Struct("@PPqqqiifi")
_TARGET = struct.Struct("@PPqqiiii")
if _ROWS.size != _lib.AZ_ROWS_BYTES or _TARGET.size != _lib.AZ_TARGET_BYTES:
  raise ImportError("os_az_rows / os_az_target are not laid out as their bindings")

try:  # the current stream's handle, without a torch.cuda.Stream around it
  _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:
  def _raw_stream(device):
    return torch.cuda.current_stream(device).cuda_stream

# How autograd learns that a call wrote given tensors: a graph that saved one of
# them before refuses to run backward.
try:  # (the public one's check of its argument takes three times as long as the rest)
  _increment_version = torch._C._increment_version
except AttributeError:
  _increment_version = torch.autograd.graph.increment_version


class LogProbs(NamedTuple):
  """Results of logprobs (float32; top_action int64)."""
  logprob: Optional[torch.Tensor]      # [N], None without actions
  entropy: torch.Tensor                # [N]
  top_action: Optional[torch.Tensor]   # [N, top], None when top = 0
  top_logprob: Optional[torch.Tensor]  # [N, top]


def _rows(logits, legal, temperature):
  """(packed os_az_rows, N, A, device index) of a call, checked; its tensors
  must outlive it."""
  dtype = _DTYPES.get(logits.dtype)
  if dtype is None:
    raise ValueError("logits must be float32, bfloat16 or float16")
  shape = logits.shape
  if len(shape) != 2:
    raise ValueError("logits must be [N, A] with unit column stride")
  n, a = shape
  ld, step = logits.stride()
  if a < 1 or (step != 1 and a > 1):
    raise ValueError("logits must be [N, A] with unit column stride")
  if not logits.is_cuda:
    raise ValueError("logits must be on a GPU")
  dev = logits.get_device()
  if a > _lib.AZ_MAX_ACTIONS:
    raise ValueError("more than %d actions" % _lib.AZ_MAX_ACTIONS)
  if not 1e-30 <= temperature <= 1e30:
    raise ValueError("temperature must be in [1e-30, 1e30]")
  mask = legal_ld = 0
  if legal is not None:
    if legal.dtype is not torch.uint8 and legal.dtype is not torch.bool:
      raise ValueError("legal must be uint8 or bool")
    if legal.shape == shape:
      legal_ld, step = legal.stride()
    elif legal.shape == (a,):
      step, = legal.stride()
    else:
      raise ValueError("legal must be [N, A] or [A]")
    if step != 1 and a > 1:
      raise ValueError("legal must have unit column stride")
    if legal.get_device() != dev:
      raise ValueError("legal must be on the logits' GPU")
    mask = legal.data_ptr()
  return (_ROWS.pack(logits.data_ptr(), mask, n, ld, legal_ld, a, dtype, temperature, 0), n, a,
          dev)


def _like(what, x, dev, dtype, *shape):
  """The address of a result or per-row tensor: contiguous, of this shape."""
  if x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
    raise ValueError("%s must be contiguous %s %s" % (what, dtype, list(shape)))
  if x.get_device() != dev:
    raise ValueError("%s must be on the logits' GPU" % what)
  return x.data_ptr()


def _actions(actions, n, dev):
  """(address, wide) of the given actions, one a row."""
  if actions is None:
    return None, 0
  wide = _IDS.get(actions.dtype)
  if wide is None:
    raise ValueError("actions must be int32 or int64")
  return _like("actions", actions, dev, actions.dtype, n), wide


def _target(target, target_actions, n, a, dev, kind):
  """The packed os_az_target of a call, checked."""
  kinds = _TARGETS.get(kind)
  if kinds is None:
    raise ValueError("kind must be 'logits' or 'weights'")
  dtype = kinds.get(target.dtype)
  if dtype is None:
    raise ValueError("target must be float32, bfloat16 or float16 logits, or float32 or int32 "
                     "weights")
  if target.requires_grad:
    raise ValueError("the target is not differentiated: detach() it")
  shape = target.shape
  if len(shape) != 2 or shape[0] != n:
    raise ValueError("target must be [N, K] with unit column stride")
  k = shape[1]
  ld, step = target.stride()
  if step != 1 and k > 1:
    raise ValueError("target must be [N, K] with unit column stride")
  if k > _lib.AZ_MAX_TARGETS:
    raise ValueError("more than %d listed actions" % _lib.AZ_MAX_TARGETS)
  if target.get_device() != dev:
    raise ValueError("target must be on the logits' GPU")
  ids = ids_ld = wide = 0
  if target_actions is None:
    if k != a:
      raise ValueError("a target without target_actions must be [N, A]")
  else:
    wide = _IDS.get(target_actions.dtype)
    if wide is None:
      raise ValueError("target_actions must be int32 or int64")
    if target_actions.shape != shape:
      raise ValueError("target_actions must be shaped as target")
    ids_ld, step = target_actions.stride()
    if step != 1 and k > 1:
      raise ValueError("target_actions must have unit column stride")
    if target_actions.get_device() != dev:
      raise ValueError("target_actions must be on the logits' GPU")
    ids = target_actions.data_ptr()
  return _TARGET.pack(ids, target.data_ptr(), ids_ld, ld, k, dtype, wide, 0)


def _grad_buffer(grad, logits, n, a, dev):
  """(address, row stride) of the caller's gradient buffer, checked."""
  if grad.dtype is not logits.dtype or grad.shape != logits.shape:
    raise ValueError("grad must have the logits' type and shape")
  if grad.get_device() != dev:
    raise ValueError("grad must be on the logits' GPU")
  ld, step = grad.stride()
  if (step != 1 and a > 1) or (ld < a and n > 1):
    raise ValueError("grad must have unit column stride and rows that do not overlap")
  return grad.data_ptr(), max(ld, a)


def _launch(fn, dev, *args):
  """Calls a C entry on the device's current stream (it also refuses results that
  overlap each other or an operand)."""
  if dev == torch.cuda.current_device():
    rc = fn(*args, _raw_stream(dev))
  else:
    with torch.cuda.device(dev):
      rc = fn(*args, _raw_stream(dev))
  if rc == _lib.OS_ERR_INVALID:
    raise ValueError(lib.os_last_error().decode(errors="replace"))
  if rc:
    check(rc)


def _workspace(rows, a, top, dev):
  """(tensor to keep until the call, address, bytes): rows of few actions need
  none (os_az_rows_workspace)."""
  if a <= _lib.AZ_NO_WORKSPACE_ACTIONS:
    return None, None, 0
  n = lib.os_az_rows_workspace(rows, top)
  if n < 0:
    check(int(n))
  if n == 0:
    return None, None, 0
  w = torch.empty(n, dtype=torch.uint8, device=torch.device("cuda", dev))
  return w, w.data_ptr(), n


def logprobs_into(logits, entropy, logprob=None, actions=None, legal=None, top_action=None,
                  top_logprob=None, temperature=1.0, stats=None):
  """logprobs into given tensors: entropy and logprob float32 [N], top_action
  int64 and top_logprob float32 [N, top], stats float32 [N, 2] (what
  os_az_logprobs_grad_async reads; optional).  logprob and actions go together,
  and so do the top pair.  What is written may not overlap anything else of the
  call."""
  rows, n, a, dev = _rows(logits, legal, temperature)
  act, wide = _actions(actions, n, dev)
  if (logprob is None) != (actions is None):
    raise ValueError("logprob and actions go together")
  if (top_action is None) != (top_logprob is None):
    raise ValueError("top_action and top_logprob go together")
  if entropy is None:
    raise ValueError("entropy is needed")
  written, lp, st, top, ta, tl = [entropy], None, None, 0, None, None
  if logprob is not None:
    lp = _like("logprob", logprob, dev, _F32, n)
    written.append(logprob)
  if stats is not None:
    st = _like("stats", stats, dev, _F32, n, 2)
    written.append(stats)
  if top_action is not None:
    if top_action.dim() != 2 or top_action.shape[1] > _lib.AZ_MAX_TOP:
      raise ValueError("top_action must be [N, top], top <= %d" % _lib.AZ_MAX_TOP)
    top = top_action.shape[1]
    ta = _like("top_action", top_action, dev, torch.int64, n, top)
    tl = _like("top_logprob", top_logprob, dev, _F32, n, top)
    written += (top_action, top_logprob)
  h = _like("entropy", entropy, dev, _F32, n)
  keep, work, size = _workspace(rows, a, top, dev)
  _launch(lib.os_az_logprobs_async, dev, rows, act, wide, lp, h, st, top, ta, tl, work, size)
  _increment_version(written)
  del keep


def distill_into(logits, target, loss, target_entropy=None, target_actions=None, legal=None,
                 kind="weights", temperature=1.0, weight=None, grad=None, stats=None):
  """distill into given tensors: loss and target_entropy float32 [N], stats
  float32 [N, 2] (what os_az_distill_grad_async reads; optional).  With `grad`
  (the logits' type and shape, any row stride) also the logits' gradient of
  (weight * loss).sum(); weight float32 [N], None: 1.  What is written may not
  overlap anything else of the call."""
  rows, n, a, dev = _rows(logits, legal, temperature)
  t = _target(target, target_actions, n, a, dev, kind)
  if loss is None:
    raise ValueError("loss is needed")
  if weight is not None and grad is None:
    raise ValueError("weight scales the gradient: it needs grad")
  written, g, ld, h, st = [loss], None, 0, None, None
  if grad is not None:
    g, ld = _grad_buffer(grad, logits, n, a, dev)
    written.append(grad)
  w = None if weight is None else _like("weight", weight, dev, _F32, n)
  out = _like("loss", loss, dev, _F32, n)
  if target_entropy is not None:
    h = _like("target_entropy", target_entropy, dev, _F32, n)
    written.append(target_entropy)
  if stats is not None:
    st = _like("stats", stats, dev, _F32, n, 2)
    written.append(stats)
  keep, work, size = _workspace(rows, a, 0, dev)
  _launch(lib.os_az_distill_async, dev, rows, t, w, out, h, st, g, ld, work, size)
  _increment_version(written)
  del keep


def _per_row(g):
  """(address, element stride) of a float32 [N] upstream gradient: an expanded
  one (of a sum or a mean) is read as it is."""
  return (None, 0) if g is None else (g.data_ptr(), g.stride(0))


def _new_logprobs(logits, actions, legal, top, temperature, keep_stats):
  """logprobs' results in new tensors, and the stats their gradient needs."""
  rows, n, a, dev = _rows(logits, legal, temperature)
  act, wide = _actions(actions, n, dev)
  device = logits.device
  entropy = torch.empty(n, dtype=_F32, device=device)
  logprob = top_action = top_logprob = stats = lp = st = ta = tl = None
  if actions is not None:
    logprob = torch.empty(n, dtype=_F32, device=device)
    lp = logprob.data_ptr()
  if keep_stats:
    stats = torch.empty(n, 2, dtype=_F32, device=device)
    st = stats.data_ptr()
  if top > 0:
    top_action = torch.empty(n, top, dtype=torch.int64, device=device)
    top_logprob = torch.empty(n, top, dtype=_F32, device=device)
    ta, tl = top_action.data_ptr(), top_logprob.data_ptr()
  keep, work, size = _workspace(rows, a, top, dev)
  _launch(lib.os_az_logprobs_async, dev, rows, act, wide, lp, entropy.data_ptr(), st, top, ta, tl,
          work, size)
  del keep
  return logprob, entropy, top_action, top_logprob, stats


def _new_distill(logits, target, target_actions, legal, kind, temperature, keep_stats):
  rows, n, a, dev = _rows(logits, legal, temperature)
  t = _target(target, target_actions, n, a, dev, kind)
  device = logits.device
  loss = torch.empty(n, dtype=_F32, device=device)
  entropy = torch.empty(n, dtype=_F32, device=device)
  stats = st = None
  if keep_stats:
    stats = torch.empty(n, 2, dtype=_F32, device=device)
    st = stats.data_ptr()
  keep, work, size = _workspace(rows, a, 0, dev)
  _launch(lib.os_az_distill_async, dev, rows, t, None, loss.data_ptr(), entropy.data_ptr(), st,
          None, 0, work, size)
  del keep
  return loss, entropy, stats


def _once(backward):
  """torch.autograd.function.once_differentiable, but for the usual call (no
  graph of the gradient is asked for), which needs none of its bookkeeping."""
  checked = torch.autograd.function.once_differentiable(backward)

  def call(ctx, *grads):
    return (checked if torch.is_grad_enabled() else backward)(ctx, *grads)
  return call


class _LogProbs(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, actions, legal, top, temperature):
    logprob, entropy, top_action, top_logprob, stats = _new_logprobs(
        logits, actions, legal, top, temperature, True)
    if top_action is not None:
      ctx.mark_non_differentiable(top_action)
    ctx.save_for_backward(logits, actions, legal, entropy, stats, top_action)
    ctx.temperature = temperature
    ctx.set_materialize_grads(False)
    return logprob, entropy, top_action, top_logprob

  @staticmethod
  @_once
  def backward(ctx, g_logprob, g_entropy, _, g_top):
    if g_logprob is None and g_entropy is None and g_top is None:
      return (None,) * 5
    logits, actions, legal, entropy, stats, top_action = ctx.saved_tensors
    rows, n, a, dev = _rows(logits, legal, ctx.temperature)
    act, wide = _actions(actions, n, dev)
    grad = torch.empty(n, a, dtype=logits.dtype, device=logits.device)
    top, ta, gt = 0, None, None
    if g_top is not None:
      g_top = g_top.contiguous()
      top, ta, gt = g_top.shape[1], top_action.data_ptr(), g_top.data_ptr()
    _launch(lib.os_az_logprobs_grad_async, dev, rows, act, wide, entropy.data_ptr(),
            stats.data_ptr(), top, ta, *_per_row(g_logprob), *_per_row(g_entropy), gt,
            grad.data_ptr(), a)
    return grad, None, None, None, None


class _Distill(torch.autograd.Function):

  @staticmethod
  def forward(ctx, logits, target, target_actions, legal, kind, temperature):
    loss, entropy, stats = _new_distill(logits, target, target_actions, legal, kind, temperature,
                                        True)
    ctx.save_for_backward(logits, target, target_actions, legal, stats)
    ctx.kind, ctx.temperature = kind, temperature
    ctx.mark_non_differentiable(entropy)
    ctx.set_materialize_grads(False)
    return loss, entropy

  @staticmethod
  @_once
  def backward(ctx, g_loss, _):
    if g_loss is None:
      return (None,) * 6
    logits, target, target_actions, legal, stats = ctx.saved_tensors
    rows, n, a, dev = _rows(logits, legal, ctx.temperature)
    t = _target(target, target_actions, n, a, dev, ctx.kind)
    grad = torch.empty(n, a, dtype=logits.dtype, device=logits.device)
    _launch(lib.os_az_distill_grad_async, dev, rows, t, *_per_row(g_loss), stats.data_ptr(),
            grad.data_ptr(), a)
    return grad, None, None, None, None, None


def _no_tangent(x):
  # (in any gradient mode: torch.no_grad() leaves forward mode on)
  if forward_ad.unpack_dual(x).tangent is not None:
    raise ValueError("forward-mode derivatives are not supported")


def _differentiated(logits):
  _no_tangent(logits)
  return logits.requires_grad and torch.is_grad_enabled()


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
  if _differentiated(logits):
    return LogProbs(*_LogProbs.apply(logits, actions, legal, top, temperature))
  return LogProbs(*_new_logprobs(logits, actions, legal, top, temperature, False)[:4])


def distill(logits, target, target_actions=None, legal=None, kind="weights", temperature=1.0):
  """(loss, target_entropy), float32 [N]: the cross entropy -sum_j q_j log p of
  the policies softmax(logits / temperature) over the allowed actions against
  the target distribution q, and the entropy -sum_j q_j log q_j of q's entries as
  they are listed.  Where a row's actions are distinct, loss - target_entropy is
  the Kullback-Leibler divergence from q; an action listed more than once adds
  the entropy of its split, so merge repeats first for a divergence (the loss and
  its gradient are the same either way).

  Entry j of row r is action target_actions[r, j] (int32 or int64 [N, K], K <=
  1024; negative: padding; listed twice counts twice) with target[r, j], which
  is a weight (kind="weights", float32 or int32: q = w / sum w, weights not
  above 0 count as 0) or a teacher's logit (kind="logits": q =
  softmax(target / temperature) over the row's entries).  Without
  target_actions the target is [N, A], A <= 1024, entry j action j.

  The loss is 0 for a row without a target, +inf where an excluded action has
  mass, NaN where an action >= A is listed.  The gradient reaches the logits,
  not the target; an excluded action's is 0."""
  _no_tangent(target)
  if _differentiated(logits):
    return _Distill.apply(logits, target, target_actions, legal, kind, temperature)
  return _new_distill(logits, target, target_actions, legal, kind, temperature, False)[:2]


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
