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
are made contiguous.

Everything runs on the tensors' device, on torch's current stream of it,
without a synchronisation or a memory that outlives the call.  All calls may be
captured into a HIP graph except the losses with logits that require a
gradient, which raise there: capture the *_and_grad form and hand its gradient
on (`logits.backward(grad)`).
"""
import ctypes
from typing import NamedTuple, Optional

import torch
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
class _on:
    """The device of `t` current (a no-op where it is); .stream is torch's
    current stream of it."""

    def __init__(self, t):
        self.index = t.device.index
        self.before = torch.cuda.current_device()

    def __enter__(self):
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(self.index))

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _arg(t, name, like, shape, *dtypes):
    """`t` checked and contiguous."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d)[6:] for d in dtypes)}, not {str(t.dtype)[6:]}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is held constant: detach() it")
    return t.contiguous()


def _table(t, name):
    """(the rows of a [..., A] tensor of logits, their stride in elements)"""
    if not isinstance(t, torch.Tensor) or t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be a float32, float16 or bfloat16 tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on a HIP device")
    A = t.shape[-1] if t.dim() else 0
    if not 1 <= A <= _native.MAX_POLICY_ACTIONS:
        raise ValueError(f"{name} must have 1..{_native.MAX_POLICY_ACTIONS} actions in the last dimension")
    rows = t.detach()
    if rows.dim() != 2:
        rows = rows.reshape(-1, A)
    if (A > 1 and rows.stride(1) != 1) or (rows.shape[0] > 1 and rows.stride(0) < A):
        rows = rows.contiguous()
    return rows, max(rows.stride(0), A)


def _decisions(logits, legal_mask, actions=None, ref_logits=None):
    """A coup_decisions of the arguments, and the tensors it points into."""
    rows, stride = _table(logits, "logits")
    lead = logits.shape[:-1]
    mask = _arg(legal_mask, "legal_mask", logits, lead, torch.int32, torch.uint32)
    keep = [rows, mask]
    ref, ref_stride, acts = None, 0, None
    if actions is not None:
        acts = _arg(actions, "actions", logits, lead, torch.int8)
        keep.append(acts)
    if ref_logits is not None:
        _arg_ref(ref_logits, logits)
        ref, ref_stride = _table(ref_logits, "ref_logits")
        keep.append(ref)
    d = _native.Decisions(rows.data_ptr(), stride, ref.data_ptr() if ref is not None else None, ref_stride,
                          acts.data_ptr() if acts is not None else None, mask.data_ptr(), rows.shape[0], rows.shape[1],
                          _DTYPES[rows.dtype])
    return d, keep


def _arg_ref(ref, logits):
    if not isinstance(ref, torch.Tensor) or ref.dtype != logits.dtype or ref.shape != logits.shape:
        raise ValueError("ref_logits must have the type and shape of logits")
    if ref.device != logits.device:
        raise ValueError(f"ref_logits is on {ref.device}, not on {logits.device}")
    if ref.requires_grad and torch.is_grad_enabled():
        raise ValueError("ref_logits is held constant: detach() it")


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
    d, keep = _decisions(logits, legal_mask)
    u = _arg(uniform, "uniform", logits, logits.shape[:-1], torch.float32)
    lib = _native.load()
    actions = torch.empty(u.shape, dtype=torch.int8, device=u.device)
    log_probs = torch.empty(u.shape, dtype=torch.float32, device=u.device)
    with _on(u) as stream:
        _native.check(lib.coup_sample_actions(ctypes.byref(d), u.data_ptr(), actions.data_ptr(), log_probs.data_ptr(),
                                              stream))
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
    the window (None: 0).  Each player's decisions are one chain: its rewards
    up to its next decision, that one's value discounted by gamma, advantages
    decayed by gamma * lam; a LAST step ends every chain, a FIRST step cuts.
    Returns (advantages, targets = advantages + values), float32 [T, B], 0 at
    steps that are no decision (FIRST, SKIPPED, no acting player)."""
    if not isinstance(values, torch.Tensor) or values.dtype not in _DTYPES:
        raise ValueError("values must be a float32, float16 or bfloat16 tensor")
    if values.device.type != "cuda":
        raise ValueError("values must be on a HIP device")
    if values.requires_grad and torch.is_grad_enabled():
        raise ValueError("values is held constant: detach() it")
    if values.dim() != 2:
        raise ValueError("values must be [T, B]")
    T, B = values.shape
    if not isinstance(rewards, torch.Tensor) or rewards.dim() != 3 or not 2 <= rewards.shape[2] <= _native.MAX_PLAYERS:
        raise ValueError(f"rewards must be [T, B, P] with 2..{_native.MAX_PLAYERS} players")
    P = rewards.shape[2]
    gamma, lam = float(gamma), float(lam)
    if not (0.0 <= gamma <= 1.0 and 0.0 <= lam <= 1.0):
        raise ValueError("gamma and lam must be in 0..1")
    r = _arg(rewards, "rewards", values, (T, B, P), torch.int8)
    st = _arg(step_type, "step_type", values, (T, B), torch.uint8)
    pl = _arg(players, "players", values, (T, B), torch.int8)
    v = values.contiguous()
    boot = None if bootstrap is None else _arg(bootstrap, "bootstrap", values, (B, P), values.dtype)
    lib = _native.load()
    adv = torch.empty(T, B, dtype=torch.float32, device=v.device)
    target = torch.empty(T, B, dtype=torch.float32, device=v.device)
    w = _native.Window(r.data_ptr(), st.data_ptr(), pl.data_ptr(), v.data_ptr(),
                       None if boot is None else boot.data_ptr(), T, B, P, _DTYPES[v.dtype])
    with _on(v) as stream:
        _native.check(lib.coup_advantages(ctypes.byref(w), gamma, lam, adv.data_ptr(), target.data_ptr(), stream))
    return adv, target


# ------------------------------------------------------------ losses
class _LossOf(torch.autograd.Function):
    """A loss whose call also wrote its gradient: backward hands that out,
    times the incoming derivative (one pass over it in place, or none where it
    is 1).  A second backward over a retained graph makes the call again."""

    @staticmethod
    def forward(ctx, logits, call, *inputs):
        out, grad = call(True)
        ctx.save_for_backward(logits, *inputs)  # their versions are checked where a second backward reads them
        ctx.call, ctx.grad = call, grad
        ctx.mark_non_differentiable(*out[1:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, incoming, *_):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the backward pass of this loss cannot be captured into a graph: capture its "
                               "_and_grad form and hand the gradient on")
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            ctx.saved_tensors
            grad = ctx.call(True)[1]
        scale = incoming.contiguous()
        lib = _native.load()
        with _on(grad) as stream:
            _native.check(lib.coup_scale_grad(grad.data_ptr(), _DTYPES[grad.dtype], grad.numel(), scale.data_ptr(), stream))
        return (grad,) + (None,) * (len(ctx.needs_input_grad) - 1)


def _loss(logits, call, inputs):
    if not (logits.requires_grad and torch.is_grad_enabled()):
        return call(False)[0]
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a loss whose logits require a gradient cannot be captured into a graph: capture its "
                           "_and_grad form and hand the gradient on")
    return _LossOf.apply(logits, call, *[t for t in inputs if t is not None])


def _scratch(nbytes, device):
    return torch.empty((nbytes + 7) // 8, dtype=torch.int64, device=device)


def _policy_call(logits, actions, legal_mask, old_log_probs, advantages, ref_logits, active, clip_low, clip_high, kl_coef,
                 entropy_coef):
    d, keep = _decisions(logits, legal_mask, actions, ref_logits)
    lead, dev = logits.shape[:-1], logits.device
    old = _arg(old_log_probs, "old_log_probs", logits, lead, torch.float32)
    adv = _arg(advantages, "advantages", logits, lead, torch.float32)
    act = None if active is None else _arg(active, "active", logits, lead, torch.bool, torch.uint8)
    clip_low, clip_high, kl_coef, entropy_coef = float(clip_low), float(clip_high), float(kl_coef), float(entropy_coef)
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < float("inf")):
        raise ValueError("clip_low must be in 0..1, clip_high finite and not negative")
    if not (-1e4 <= kl_coef <= 1e4 and -1e4 <= entropy_coef <= 1e4):
        raise ValueError("kl_coef and entropy_coef must be finite, within 1e4")
    terms = _native.PolicyTerms(old.data_ptr(), adv.data_ptr(), None if act is None else act.data_ptr(), clip_low,
                                clip_high, kl_coef, entropy_coef)
    lib = _native.load()

    def call(want_grad):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        stats = torch.empty(4, dtype=torch.float32, device=dev)
        count = torch.empty((), dtype=torch.int64, device=dev)
        log_probs = torch.empty(lead, dtype=torch.float32, device=dev)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
        nbytes = lib.coup_policy_workspace(d.rows)
        scratch = _scratch(nbytes, dev)
        out = _native.PolicyOutputs(loss.data_ptr(), stats.data_ptr(), count.data_ptr(), log_probs.data_ptr(),
                                    None if grad is None else grad.data_ptr())
        with _on(logits) as stream:
            _native.check(lib.coup_policy_loss(ctypes.byref(d), ctypes.byref(terms), ctypes.byref(out),
                                               scratch.data_ptr(), nbytes, stream))
        return (loss, stats, count, log_probs), grad

    call.keep = (keep, old, adv, act)  # what d and terms point into
    return call


def policy_loss(logits, actions, legal_mask, old_log_probs, advantages, ref_logits=None, active=None, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, entropy_coef=0.0) -> PolicyLoss:
    """The clipped policy loss with a KL term, differentiable in logits:

        mean of -min(rho adv, clip(rho, 1 - clip_low, 1 + clip_high) adv)
                + kl_coef KL(pi || pi_ref) - entropy_coef H(pi)

    over the decisions that count, rho = exp(log pi(action) - old_log_probs).

    logits [..., A]; actions int8 [...] and legal_mask int32 [...]: the action
    taken and the legal-action word it was taken under; old_log_probs,
    advantages float32 [...]; ref_logits [..., A]: the reference policy's, in
    the logits' type (None: the KL is 0, whatever kl_coef); active bool [...]: which rows to train on
    (e.g. one player's; None: all).  Everything but logits is held constant.
    The loss is 0, with zero gradients, where nothing counts.  A ratio exactly
    on a border is not clipped.  A legal action that the reference gives no
    probability makes the KL infinite."""
    call = _policy_call(logits, actions, legal_mask, old_log_probs, advantages, ref_logits, active, clip_low, clip_high,
                        kl_coef, entropy_coef)
    return PolicyLoss(*_loss(logits, call, (actions, legal_mask, old_log_probs, advantages, ref_logits, active)))


def policy_loss_and_grad(logits, actions, legal_mask, old_log_probs, advantages, ref_logits=None, active=None,
                         clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0) -> PolicyLossAndGrad:
    """policy_loss and its gradient in the logits in one pass, outside
    autograd (hand the gradient on with logits.backward(grad))."""
    out, grad = _policy_call(logits, actions, legal_mask, old_log_probs, advantages, ref_logits, active, clip_low,
                             clip_high, kl_coef, entropy_coef)(True)
    return PolicyLossAndGrad(*out, grad)


def _preference_call(logits, actions, legal_mask, offsets, ref_logits, beta, label_smoothing):
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("logits must be [rows, A]: the sequences' decisions one after another")
    d, keep = _decisions(logits, legal_mask, actions, ref_logits)
    dev = logits.device
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.numel() % 2 == 0:
        raise ValueError("offsets must be [2 * pairs + 1]")
    off = _arg(offsets, "offsets", logits, offsets.shape, torch.int32, torch.int64)
    pairs = off.numel() // 2
    beta, label_smoothing = float(beta), float(label_smoothing)
    if beta - beta != 0.0:
        raise ValueError("beta must be finite")
    if not 0.0 <= label_smoothing <= 0.5:
        raise ValueError("label_smoothing must be in 0..0.5")
    terms = _native.PreferenceTerms(off.data_ptr(), off.element_size(), pairs, beta, label_smoothing)
    lib = _native.load()

    def call(want_grad):
        loss = torch.empty((), dtype=torch.float32, device=dev)
        rewards = torch.empty(2 * pairs, dtype=torch.float32, device=dev)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
        nbytes = lib.coup_preference_workspace(d.rows, pairs)
        scratch = _scratch(max(nbytes, 8), dev)
        out = _native.PreferenceOutputs(loss.data_ptr(), rewards.data_ptr(), None if grad is None else grad.data_ptr())
        with _on(logits) as stream:
            _native.check(lib.coup_preference_loss(ctypes.byref(d), ctypes.byref(terms), ctypes.byref(out),
                                                   scratch.data_ptr(), nbytes, stream))
        return (loss, rewards), grad

    call.keep = (keep, off)  # what d and terms point into
    return call


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
    Offsets that do not ascend from 0..rows make the loss NaN."""
    call = _preference_call(logits, actions, legal_mask, offsets, ref_logits, beta, label_smoothing)
    return PreferenceLoss(*_loss(logits, call, (actions, legal_mask, offsets, ref_logits)))


def preference_loss_and_grad(logits, actions, legal_mask, offsets, ref_logits: Optional[torch.Tensor] = None, beta=0.1,
                             label_smoothing=0.0) -> PreferenceLossAndGrad:
    """preference_loss and its gradient in the logits in one call, outside
    autograd (hand the gradient on with logits.backward(grad))."""
    out, grad = _preference_call(logits, actions, legal_mask, offsets, ref_logits, beta, label_smoothing)(True)
    return PreferenceLossAndGrad(*out, grad)
