"""What a learner computes between two trajectories, on the tensors
`BatchedCoupEnv` reads and writes (include/coup_mi355x.h, "learner-side
operators"; kernels: csrc/coup_policy.h).

    sample_actions        an action and its log probability per row of logits,
                          under the env's legal-action words: the actions
                          `BatchedCoupEnv.step` takes
    advantages            generalised advantages and value targets of a
                          [T, B] window in which the players take turns
    policy_loss           the clipped policy loss with a KL term (and its
                          gradient: policy_loss_and_grad)
    preference_loss       the paired log-ratio loss of preferred against
                          rejected sequences of decisions (and its gradient:
                          preference_loss_and_grad)

A row is one decision: A <= 31 logits in the last dimension, one legal-action
word, one action; the leading dimensions are any, the same for every argument
([B], [T, B], ...).  A row counts where its action is legal -- 0 <= action < A,
the word's bit `action` set, bit 31 (a chance node) clear.  Lanes that were
reset or skipped (action -1), finished games and chance nodes give zeros,
whatever the row holds besides; so do logits of actions outside the word.
Logits are float32, float16 or bfloat16; arithmetic is in 32 bits or more,
gradients have the logits' type.  Logits may be strided; the other arguments
are made contiguous.  Nothing but a loss is differentiable, and that in its
logits and in reverse mode: tensors that carry a forward-mode derivative are
refused.

Everything runs on the tensors' device, on torch's current stream of it,
without a synchronisation or a memory that outlives the call.  All calls may be
captured into a HIP graph except the losses with logits that require a
gradient, which raise there (and the backward pass of an eager loss must not
run inside a capture): capture the *_and_grad form and hand its gradient on
(`logits.backward(grad)`).
"""
import ctypes
import weakref
from typing import NamedTuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16}


class PolicyLoss(NamedTuple):
    """policy_loss's results.  loss: 0-d float32; stats: float32 [4], means
    over the decisions that count of the clipped surrogate, KL(pi || ref), the
    entropy and the share of clipped ratios; count: 0-d int64, the decisions
    that count; log_probs: float32, log pi(action) per row, 0 where it does
    not count."""
    loss: torch.Tensor
    stats: torch.Tensor
    count: torch.Tensor
    log_probs: torch.Tensor


class PolicyLossAndGrad(NamedTuple):
    """PolicyLoss and grad, d loss / d logits (contiguous, the logits' shape and type)."""
    loss: torch.Tensor
    stats: torch.Tensor
    count: torch.Tensor
    log_probs: torch.Tensor
    grad: torch.Tensor


class PreferenceLoss(NamedTuple):
    """preference_loss's results.  loss: 0-d float32; rewards: float32 [S],
    beta times each sequence's summed log ratio."""
    loss: torch.Tensor
    rewards: torch.Tensor


class PreferenceLossAndGrad(NamedTuple):
    """PreferenceLoss and grad, d loss / d logits (contiguous, the logits' shape and type)."""
    loss: torch.Tensor
    rewards: torch.Tensor
    grad: torch.Tensor


# ------------------------------------------------------------ arguments
_lib = None


def _enqueue(name, device, *args):
    """Call the library's `name` with the device current and torch's current
    stream of it as the last argument."""
    global _lib
    if _lib is None:
        _lib = _native.load()
    index, before = device.index, torch._C._cuda_getDevice()
    if before != index:
        torch.cuda.set_device(index)
    try:
        rc = getattr(_lib, name)(*args, torch._C._cuda_getCurrentRawStream(index))
    finally:
        if before != index:
            torch.cuda.set_device(before)
    if rc != _native.COUP_OK:
        _native.check(rc)


def _capturing(device):
    """Whether torch's current stream of `device` (which need not be the current one) is being captured."""
    if device.index == torch._C._cuda_getDevice():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _refuse_duals(*args):
    """Raise where an argument carries a forward-mode derivative (asked for inside a dual level alone)."""
    for t in args:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError("a tensor carries a forward-mode derivative, which these calls do not pass on: detach() it")


def _wrong(t, name, device, shape, dtypes):
    """What is wrong with an argument, as an exception."""
    if not isinstance(t, torch.Tensor):
        return ValueError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        return ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, not {str(t.dtype)[6:]}")
    if t.device != device:
        return ValueError(f"{name} is on {t.device}, not on {device}")
    if t.shape != shape:
        return ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    return ValueError(f"{name} is held constant: detach() it")


def _arg(t, name, device, shape, dtypes):
    """`t` checked and contiguous."""
    if (not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.device != device or t.shape != shape
            or (t.requires_grad and torch.is_grad_enabled())):
        raise _wrong(t, name, device, shape, dtypes)
    return t if t.is_contiguous() else t.contiguous()


def _table(t, name):
    """(the rows of a [..., A] tensor of logits, their stride in elements)"""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be a float32, float16 or bfloat16 tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a HIP device")
    A = t.shape[-1] if t.dim() else 0
    if not 1 <= A <= _native.MAX_POLICY_ACTIONS:
        raise ValueError(f"{name} must have 1..{_native.MAX_POLICY_ACTIONS} actions in the last dimension")
    if t.is_contiguous():
        return t, A
    rows = t.detach()
    if rows.dim() != 2:
        rows = rows.reshape(-1, A)
    if (A > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < A):
        rows = rows.contiguous()
    return rows, max(rows.stride(0), A)


_INT8, _INT32, _FLOAT32 = (torch.int8,), (torch.int32, torch.uint32), (torch.float32,)
_BOOL, _OFFSET, _BYTE = (torch.bool, torch.uint8), (torch.int32, torch.int64), (torch.uint8,)


def _decisions(logits, legal_mask, actions=None, ref_logits=None):
    """A coup_decisions of the arguments, and the tensors it points into."""
    rows, stride = _table(logits, "logits")
    lead, device = logits.shape[:-1], logits.device
    A = logits.shape[-1]
    mask = _arg(legal_mask, "legal_mask", device, lead, _INT32)
    ref = acts = None
    ref_stride = 0
    if actions is not None:
        acts = _arg(actions, "actions", device, lead, _INT8)
    if ref_logits is not None:
        if not isinstance(ref_logits, torch.Tensor) or ref_logits.dtype != logits.dtype or ref_logits.shape != logits.shape:
            raise ValueError("ref_logits must have the type and shape of logits")
        _arg_held(ref_logits, "ref_logits", device)
        ref, ref_stride = _table(ref_logits, "ref_logits")
    d = _native.Decisions(rows.data_ptr(), stride, None if ref is None else ref.data_ptr(), ref_stride,
                          None if acts is None else acts.data_ptr(), mask.data_ptr(), logits.numel() // A, A,
                          _DTYPES[logits.dtype])
    return d, (rows, mask, acts, ref)


def _arg_held(t, name, device):
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is held constant: detach() it")


# ------------------------------------------------------------ acting
def sample_actions(logits, legal_mask, uniform):
    """One action per row, drawn from softmax(logits) over the legal actions.

    logits [..., A]; legal_mask int32 [...], the env's legal-action words;
    uniform float32 [...], numbers in [0, 1) (torch.rand): the action is the
    first legal one, in ascending order, whose running probability exceeds
    its number, compared in 64 bits where 32 could turn it.  Returns
    (actions int8 [...], log_probs float32 [...]).  A row without a legal
    action gives -1 (which `BatchedCoupEnv.step` skips) and 0; one with a NaN
    or +inf logit at a legal action, or only -inf ones, gives -1 and NaN."""
    if forward_ad._current_level >= 0:
        _refuse_duals(logits, legal_mask, uniform)
    d, keep = _decisions(logits, legal_mask)
    device = logits.device
    u = _arg(uniform, "uniform", device, logits.shape[:-1], _FLOAT32)
    actions = torch.empty(u.shape, dtype=torch.int8, device=device)
    log_probs = torch.empty_like(u)
    _enqueue("coup_sample_actions", device, ctypes.byref(d), u.data_ptr(), actions.data_ptr(), log_probs.data_ptr())
    return actions, log_probs


# ------------------------------------------------------------ advantages
def advantages(rewards, step_type, players, values, bootstrap=None, gamma=1.0, lam=0.95):
    """Generalised advantages over a [T, B] window of a game in which the
    players take turns.

    rewards int8 [T, B, P], step_type uint8 [T, B]: a trajectory's, as
    `collect_trajectory` records them; players int8 [T, B]: the player that
    acts in step t (the current player before it); values [T, B] (float32,
    float16 or bfloat16): that player's value of the state it acts in;
    bootstrap [B, P], values' type: each player's value of the state behind
    the window, e.g. a critic's of the last step's obs [B, P, ...] (None: 0,
    which takes games that are still open there to be worth nothing).  Each
    player's decisions are one chain: its rewards up to its next decision, that
    one's value discounted by gamma, advantages decayed by gamma * lam; a LAST
    step ends every chain, a FIRST step cuts.
    Returns (advantages, targets = advantages + values), float32 [T, B], 0 at
    steps that are no decision (FIRST, SKIPPED, no acting player)."""
    if not isinstance(values, torch.Tensor) or values.dtype not in _DTYPES:
        raise ValueError("values must be a float32, float16 or bfloat16 tensor")
    device = values.device
    if device.type != "cuda":
        raise ValueError("values must be on a HIP device")
    if forward_ad._current_level >= 0:
        _refuse_duals(rewards, step_type, players, values, bootstrap)
    _arg_held(values, "values", device)
    if values.dim() != 2:
        raise ValueError("values must be [T, B]")
    T, B = values.shape
    if not isinstance(rewards, torch.Tensor) or rewards.dim() != 3 or not 2 <= rewards.shape[2] <= _native.MAX_PLAYERS:
        raise ValueError(f"rewards must be [T, B, P] with 2..{_native.MAX_PLAYERS} players")
    P = rewards.shape[2]
    gamma, lam = float(gamma), float(lam)
    if not (0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0):
        raise ValueError("gamma and lam must be in 0..1")
    r = _arg(rewards, "rewards", device, (T, B, P), _INT8)
    st = _arg(step_type, "step_type", device, (T, B), _BYTE)
    pl = _arg(players, "players", device, (T, B), _INT8)
    v = values.contiguous()
    boot = None if bootstrap is None else _arg(bootstrap, "bootstrap", device, (B, P), (values.dtype,))
    adv = torch.empty(T, B, dtype=torch.float32, device=device)
    target = torch.empty_like(adv)
    w = _native.Window(r.data_ptr(), st.data_ptr(), pl.data_ptr(), v.data_ptr(),
                       None if boot is None else boot.data_ptr(), T, B, P, _DTYPES[v.dtype])
    _enqueue("coup_advantages", device, ctypes.byref(w), gamma, lam, adv.data_ptr(), target.data_ptr())
    return adv, target


# ------------------------------------------------------------ losses
class _LossOf(torch.autograd.Function):
    """A loss whose call also wrote its gradient: backward hands that out,
    times the incoming derivative (one pass over it in place, or none where it
    is 1).  A second backward over a retained graph makes the call again, on
    the saved arguments and with the derivative as the gradient's factor; so
    does the first of float16 logits, whose range a gradient over many rows
    needs the factor (a loss scaler's) for before it is rounded."""

    @staticmethod
    def forward(ctx, logits, call, tensors, numbers):
        out, ctx.grad, again, read = call(logits.dtype != torch.float16, logits, *tensors, *numbers)
        ctx.save_for_backward(logits, *tensors)
        given = [(weakref.ref(t), t.data_ptr()) for t in (logits, *tensors) if t is not None]
        # a call to come for sure may take this one's addresses, where these are the arguments' own and still hold
        as_given = ctx.grad is None and {t.data_ptr() for t in read} <= {at for _, at in given}
        ctx.later = call, numbers, given, again if as_given else None
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, incoming, *_):
        if torch.cuda.is_current_stream_capturing():  # this thread's device is the incoming derivative's
            raise RuntimeError("the backward pass of this loss cannot be captured into a graph: capture its "
                               "_and_grad form and hand the gradient on")
        if forward_ad._current_level >= 0:
            _refuse_duals(incoming)
        grad, ctx.grad = ctx.grad, None
        if grad is not None:
            scale = incoming.contiguous()
            _enqueue("coup_scale_grad", grad.device, grad.data_ptr(), _DTYPES[grad.dtype], grad.numel(), scale.data_ptr())
            return grad, None, None, None
        call, numbers, given, again = ctx.later
        saved = ctx.saved_tensors  # torch checks their versions
        for t, (one, at) in zip([t for t in saved if t is not None], given):
            if t is not one():
                again = None  # a hook's equal one
            elif t.data_ptr() != at:
                raise RuntimeError("an argument of this loss was given other data since")
        grad = again(incoming) if again is not None else call(True, *saved, *numbers, grad_scale=incoming)[1]
        return grad, None, None, None


def _loss(call, logits, tensors, numbers):
    if forward_ad._current_level >= 0:
        _refuse_duals(logits, *tensors)
    if not (isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled()):
        return call(False, logits, *tensors, *numbers)[0]
    for t in tensors:  # unseen inside the function below
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError("every argument but logits is held constant: detach() those that require a gradient")
    if logits.is_cuda and _capturing(logits.device):
        raise RuntimeError("a loss whose logits require a gradient cannot be captured into a graph: capture its "
                           "_and_grad form and hand the gradient on")
    return _LossOf.apply(logits, call, tensors, numbers)


def _again(name, outputs, d, terms, nbytes, logits):
    """The call `name` once more, for its gradient times a factor.  Holds no
    tensor: those that d and terms point into are its caller's to keep."""
    shape, dtype, device = logits.shape, logits.dtype, logits.device

    def call(factor):
        grad = torch.empty(shape, dtype=dtype, device=device)
        loss = torch.empty((), dtype=torch.float32, device=device)
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        out = outputs(loss=loss.data_ptr(), grad=grad.data_ptr(), grad_scale=factor.data_ptr())
        _enqueue(name, device, ctypes.byref(d), ctypes.byref(terms), ctypes.byref(out), scratch.data_ptr(), nbytes)
        return grad
    return call


def _policy(want_grad, logits, actions, legal_mask, old_log_probs, advantages, ref_logits, active, clip_low, clip_high,
            kl_coef, entropy_coef, grad_scale=None):
    """((loss, stats, count, log_probs), gradient or None, the call for a
    gradient with a factor alone, the tensors that it reads)"""
    d, keep = _decisions(logits, legal_mask, actions, ref_logits)
    lead, device = logits.shape[:-1], logits.device
    old = _arg(old_log_probs, "old_log_probs", device, lead, _FLOAT32)
    adv = _arg(advantages, "advantages", device, lead, _FLOAT32)
    act = None if active is None else _arg(active, "active", device, lead, _BOOL)
    factor = None if grad_scale is None else _arg(grad_scale, "grad_scale", device, (), _FLOAT32)
    clip_low, clip_high, kl_coef, entropy_coef = float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef)
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError("clip_low must be in 0..1, clip_high finite and not negative")
    if not (-1e4 <= kl_coef <= 1e4 and -1e4 <= entropy_coef <= 1e4):
        raise ValueError("kl_coef and entropy_coef must be finite, within 1e4")
    terms = _native.PolicyTerms(old.data_ptr(), adv.data_ptr(), None if act is None else act.data_ptr(), clip_low,
                                clip_high, kl_coef, entropy_coef)
    loss = torch.empty((), dtype=torch.float32, device=device)
    stats = torch.empty(4, dtype=torch.float32, device=device)
    count = torch.empty((), dtype=torch.int64, device=device)
    log_probs = torch.empty_like(old)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=device) if want_grad else None
    nbytes = _native.load().coup_policy_workspace(d.rows)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    out = _native.PolicyOutputs(*[None if t is None else t.data_ptr() for t in (loss, stats, count, log_probs, grad, factor)])
    _enqueue("coup_policy_loss", device, ctypes.byref(d), ctypes.byref(terms), ctypes.byref(out), scratch.data_ptr(),
             nbytes)
    again = _again("coup_policy_loss", _native.PolicyOutputs, d, terms, nbytes, logits)
    return (loss, stats, count, log_probs), grad, again, [t for t in (*keep, old, adv, act) if t is not None]


def policy_loss(logits, actions, legal_mask, old_log_probs, advantages, ref_logits=None, active=None, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, entropy_coef=0.0) -> PolicyLoss:
    """The clipped policy loss with a KL term, differentiable in logits:

        mean of -min(rho adv, clip(rho, 1 - clip_low, 1 + clip_high) adv)
                + kl_coef KL(pi || pi_ref) - entropy_coef H(pi)

    over the decisions that count, rho = exp(log pi(action) - old_log_probs).

    logits [..., A]; actions int8 [...] and legal_mask int32 [...]: the action
    taken and the legal-action word it was taken under; old_log_probs,
    advantages float32 [...]; ref_logits [..., A]: the reference policy's, in
    the logits' type (None: the KL is 0, whatever kl_coef); active bool [...]:
    which rows to train on (e.g. one player's; None: all).  Everything but
    logits is held constant.
    The loss is 0, with zero gradients, where nothing counts.  A ratio exactly
    on a border is not clipped.  A legal action that the reference gives no
    probability (a logit of -inf) and the policy some (a logit within 745 of
    the row's largest) makes the KL infinite, and with a kl_coef its row's
    gradient NaN."""
    return PolicyLoss(*_loss(_policy, logits, (actions, legal_mask, old_log_probs, advantages, ref_logits, active),
                             (float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef))))


def policy_loss_and_grad(logits, actions, legal_mask, old_log_probs, advantages, ref_logits=None, active=None,
                         clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0,
                         grad_scale=None) -> PolicyLossAndGrad:
    """policy_loss and its gradient in the logits in one pass, outside
    autograd (hand the gradient on with logits.backward(grad)).  grad_scale
    (0-d float32): what the gradient is multiplied by before it is rounded to
    the logits' type (a loss scaler's factor)."""
    if forward_ad._current_level >= 0:
        _refuse_duals(logits, old_log_probs, advantages, ref_logits, grad_scale)
    out, grad, *_ = _policy(True, logits, actions, legal_mask, old_log_probs, advantages, ref_logits, active, clip_low,
                        clip_high, kl_coef, entropy_coef, grad_scale)
    return PolicyLossAndGrad(*out, grad)


def _preference(want_grad, logits, actions, legal_mask, offsets, ref_logits, beta, label_smoothing, grad_scale=None):
    """((loss, rewards), gradient or None, and as _policy)"""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("logits must be [rows, A]: the sequences' decisions one after another")
    d, keep = _decisions(logits, legal_mask, actions, ref_logits)
    device = logits.device
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() % 2 == 0:
        raise ValueError("offsets must be [2 * pairs + 1]")
    off = _arg(offsets, "offsets", device, offsets.shape, _OFFSET)
    factor = None if grad_scale is None else _arg(grad_scale, "grad_scale", device, (), _FLOAT32)
    pairs = off.numel() // 2
    beta, label_smoothing = float(beta), float(label_smoothing)
    if beta - beta != 0.0:
        raise ValueError("beta must be finite")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError("label_smoothing must be in 0..0.5")
    terms = _native.PreferenceTerms(off.data_ptr(), off.element_size(), pairs, beta, label_smoothing)
    loss = torch.empty((), dtype=torch.float32, device=device)
    rewards = torch.empty(2 * pairs, dtype=torch.float32, device=device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=device) if want_grad else None
    nbytes = _native.load().coup_preference_workspace(d.rows, pairs)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    out = _native.PreferenceOutputs(*[None if t is None else t.data_ptr() for t in (loss, rewards, grad, factor)])
    _enqueue("coup_preference_loss", device, ctypes.byref(d), ctypes.byref(terms), ctypes.byref(out),
             scratch.data_ptr(), nbytes)
    again = _again("coup_preference_loss", _native.PreferenceOutputs, d, terms, nbytes, logits)
    return (loss, rewards), grad, again, [t for t in (*keep, off) if t is not None]


def preference_loss(logits, actions, legal_mask, offsets, ref_logits=None, beta=0.1,
                    label_smoothing=0.0) -> PreferenceLoss:
    """The paired log-ratio loss of preferred against rejected sequences of
    decisions, differentiable in logits.

    logits [rows, A], actions int8 [rows], legal_mask int32 [rows]: the
    sequences' decisions one after another; offsets int32 or int64 [2 P + 1],
    ascending: sequence s is rows [offsets[s], offsets[s + 1]), and pair i
    prefers sequence 2 i to 2 i + 1 (e.g. a game's winner's decisions to its
    loser's).  A sequence's reward is beta times the sum over its decisions of
    log pi(action) - log pi_ref(action); with x the difference of a pair's
    rewards the loss is the mean over pairs of
        -(1 - label_smoothing) log sigmoid(x) - label_smoothing log sigmoid(-x).
    Sequences may be empty; rows outside every sequence get zero gradients.
    Offsets that do not ascend within 0..rows make the loss NaN, and rewards
    and gradient undefined."""
    return PreferenceLoss(*_loss(_preference, logits, (actions, legal_mask, offsets, ref_logits),
                                 (float(beta), float(label_smoothing))))


def preference_loss_and_grad(logits, actions, legal_mask, offsets, ref_logits=None, beta=0.1, label_smoothing=0.0,
                             grad_scale=None) -> PreferenceLossAndGrad:
    """preference_loss and its gradient in the logits in one call, outside
    autograd (hand the gradient on with logits.backward(grad)).  grad_scale: as
    in policy_loss_and_grad."""
    if forward_ad._current_level >= 0:
        _refuse_duals(logits, ref_logits, grad_scale)
    out, grad, *_ = _preference(True, logits, actions, legal_mask, offsets, ref_logits, beta, label_smoothing, grad_scale)
    return PreferenceLossAndGrad(*out, grad)
