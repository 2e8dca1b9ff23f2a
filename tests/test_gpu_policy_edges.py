"""The learner-side operators at the edges of their definitions: infinite
margins and divergences, nearly sure decisions, offsets that do not ascend,
long read-ons behind a part of a window, saved-tensor hooks and forward-mode
derivatives.  Tolerances as in test_gpu_policy.py: H = 2^-24 is half a step of
a 32-bit value of 1."""
import math

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

from open_spiel_coup_amd import BatchedCoupEnv, policy
from tests import policy_oracle as oracle
from tests import test_gpu_policy as base

pytestmark = pytest.mark.gpu

H, DEV = base.H, base.DEV
_np, _close = base._np, base._close


# ------------------------------------------------------------ infinite margins
@pytest.mark.parametrize("pairs,each", [(3, 4), (600, 30), (3, 400)], ids=["short-few", "short", "long"])
@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_a_margin_of_plus_infinity_costs_nothing(pairs, each, eps):
    """A rejected decision of probability 0 makes its pair's margin +inf: -log sigmoid(inf) = 0, and with smoothing
    -eps log sigmoid(-inf) = inf; a chosen one makes the cost inf either way.  The other pairs lie at a margin of 0 and
    cost log 2; a sure pair's gradient is eps beta / pairs ([b = a] - p_b) in the chosen rows."""
    n = pairs * each
    x = torch.zeros(n, 3)
    mask, actions = torch.full((n,), 7, dtype=torch.int32), torch.zeros(n, dtype=torch.int8)
    off = torch.tensor([k * each // 2 for k in range(2 * pairs + 1)], device=DEV)
    x[each // 2] = torch.tensor([-math.inf, 0.0, 0.0])  # pair 0's first rejected row
    args = (actions.to(DEV), mask.to(DEV), off)
    got = policy.preference_loss_and_grad(x.to(DEV), *args, beta=0.25, label_smoothing=eps)
    assert float(got.rewards[1]) == -math.inf and bool(torch.isfinite(got.rewards[2:]).all())
    if eps:
        assert float(got.loss) == math.inf
    else:
        _close(float(got.loss), (pairs - 1) * math.log(2) / pairs, 16 * H, "loss")
    c = eps * 0.25 / pairs
    want = np.tile(c * np.array([2 / 3, -1 / 3, -1 / 3]), (each // 2, 1))
    _close(_np(got.grad[:each // 2]), want, 16 * H * c, "grad of the chosen rows")
    assert torch.isfinite(got.grad).all()
    y = x.clone()
    y[0], y[each // 2] = x[each // 2], x[0]
    assert float(policy.preference_loss(y.to(DEV), *args, beta=0.25, label_smoothing=eps).loss) == math.inf


# ------------------------------------------------------------ references without a share
def _one_decision(x, ref, n):
    """Row n // 2 of n like rows is the decision of logits x against ref; the others' KL is 0."""
    A = x.numel()
    rows, refs = torch.zeros(n, A, dtype=x.dtype), torch.zeros(n, A, dtype=x.dtype)
    rows[n // 2], refs[n // 2] = x, ref
    words = torch.full((n,), (1 << A) - 1, dtype=torch.int32)
    return rows, refs, words, torch.ones(n, dtype=torch.int8), torch.full((n,), -math.log(A)), torch.ones(n)


@pytest.mark.parametrize("dtype", base.DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("n", [5, 70001])
@pytest.mark.parametrize("A", [3, 18, 24])
def test_an_action_only_the_policy_takes_makes_the_kl_infinite(A, n, dtype):
    """However small its share is (e^-25 to e^-700): the KL and the loss are infinite, and the row has no gradient.
    Where the share is 0 (a logit of -inf, or 800 below), or the loss does not weigh the KL, all is finite."""
    for gap in (1.0, 25.0, 60.0, 80.0, 150.0, 700.0):
        x, ref = torch.zeros(A, dtype=dtype), torch.zeros(A, dtype=dtype)
        x[A - 1], ref[A - 1] = -gap, -math.inf
        rows, refs, words, acts, old, adv = (t.to(DEV) for t in _one_decision(x, ref, n))
        got = policy.policy_loss_and_grad(rows, acts, words, old, adv, ref_logits=refs, kl_coef=0.1)
        assert float(got.stats[1]) == math.inf and float(got.loss) == math.inf, gap
        assert got.grad[n // 2].isnan().all() and int(got.grad.isnan().sum()) == A
        assert float(policy.policy_loss(rows, acts, words, old, adv, ref_logits=refs, kl_coef=0.1).loss) == math.inf
        free = policy.policy_loss_and_grad(rows, acts, words, old, adv, ref_logits=refs)
        none = policy.policy_loss_and_grad(rows, acts, words, old, adv)
        assert float(free.stats[1]) == math.inf and torch.equal(free.loss, none.loss) and torch.equal(free.grad, none.grad)
    for gap in (800.0, math.inf):
        x[A - 1] = -gap
        rows, refs, words, acts, old, adv = (t.to(DEV) for t in _one_decision(x, ref, n))
        got = policy.policy_loss_and_grad(rows, acts, words, old, adv, ref_logits=refs, kl_coef=0.1)
        # both policies are uniform over the other A - 1 actions
        assert abs(float(got.stats[1])) <= 100 * H and torch.isfinite(got.grad).all()
        assert float(got.grad[n // 2, A - 1]) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("n", [5, 70001])
def test_a_references_lowest_values_have_a_finite_kl(n, dtype):
    """Logits of the type's lowest value, -1e30 and -1e34 at actions the policy takes: finite distances, weighed as such.
    64-bit sums, rounded: the KL is off by a rounding of the row's and one of the mean (2 H), a gradient entry by the
    scale's, its own (2 H of its terms) and its type's."""
    low = torch.finfo(dtype).min
    # (logit, reference's) of an action; the first is acted
    for far in ([(-1.0, low)], [(-30.0, low)], [(-1.0, low), (0.5, low / 4), (0.25, -1e30)], [(-60.0, -1e34)], [(0.0, -3e32)]):
        x, ref = torch.zeros(9), torch.zeros(9)
        x[1], ref[1], x[2], ref[2] = 0.75, -0.5, -1.5, 0.25
        for k, (a, b) in enumerate(far):
            x[4 + k], ref[4 + k] = a, b
        rows, refs, words, acts, old, adv = _one_decision(x.to(dtype), ref.to(dtype), n)
        one = [t[n // 2:n // 2 + 1] for t in (rows, acts, words, old, adv, refs)]
        o = oracle.policy(_np(one[0]), one[1].numpy(), one[2].numpy(), _np(one[3]), _np(one[4]), _np(one[5]), None, 0.2, 0.2,
                          0.25, 0.01)
        got = policy.policy_loss_and_grad(*(t.to(DEV) for t in (rows, acts, words, old, adv)), ref_logits=refs.to(DEV),
                                          kl_coef=0.25, entropy_coef=0.01)
        kl = o["stats"][1] / n
        # below kLowest / 2 the row is taken in 32 bits as every other: 9 terms, each a few roundings
        _close(float(got.stats[1]), kl, 50 * H * abs(kl), "kl")
        info = torch.finfo(dtype)
        lim = 50 * H * o["size"] + info.eps / 2 * np.abs(o["grad"])
        _close(_np(got.grad[n // 2]), o["grad"][0] / n, lim[0] / n, "grad")


# ------------------------------------------------------------ many sequences
def _preference64(x, actions, mask, offsets, ref, beta, eps):
    """oracle.preference over many rows at once (torch, 64 bits), as a dict of the same names."""
    n, A = x.shape
    legal = ((mask[:, None] >> torch.arange(A)) & 1).bool() & (mask >= 0)[:, None]
    a = actions.long()
    real = (a >= 0) & (a < A) & legal.gather(1, a.clamp(0, A - 1)[:, None])[:, 0]
    hot = (torch.arange(A) == a[:, None]) & real[:, None]

    def logs(t):
        return torch.log_softmax(t.double().masked_fill(~legal, -math.inf), 1).masked_fill(~legal | ~real[:, None], 0.0)

    lp = logs(x)
    ratio = (lp * hot).sum(1) - ((logs(ref) * hot).sum(1) if ref is not None else 0.0)
    off = torch.as_tensor(offsets)
    lens = off[1:] - off[:-1]
    owner = torch.repeat_interleave(torch.arange(lens.numel()), lens)
    inside = slice(int(off[0]), int(off[-1]))
    rewards = beta * torch.zeros(lens.numel(), dtype=torch.float64).index_add(0, owner, ratio[inside])
    m = rewards[0::2] - rewards[1::2]
    pairs = m.numel()
    loss = ((1 - eps) * torch.nn.functional.softplus(-m) + eps * torch.nn.functional.softplus(m)).mean()
    c = (eps - torch.sigmoid(-m)) * beta / pairs
    coef = torch.zeros(n, dtype=torch.float64)
    coef[inside] = torch.stack((c, -c), 1).flatten()[owner]
    p = lp.exp().masked_fill(~legal | ~real[:, None], 0.0)
    length = torch.zeros(lens.numel(), dtype=torch.float64).index_add(0, owner, real[inside].double())
    return dict(loss=float(loss), rewards=rewards.numpy(), grad=(coef[:, None] * (hot.double() - p)).numpy(),
                size=(coef.abs()[:, None] * (hot.double() + p)).numpy(), length=length.numpy())


def _many(seed, n, A, dtype, with_ref):
    """base._table's kinds of rows, 660 of them over and over, with waste of their own."""
    gen = torch.Generator().manual_seed(seed)
    x, mask, actions = base._table(gen, 660, A, dtype)
    k = (n + 659) // 660
    x, mask, actions = (t.repeat(k, *[1] * (t.dim() - 1))[:n] for t in (x, mask, actions))
    x = torch.where(torch.isfinite(x.float()), x.float() + torch.randn(n, A, generator=gen), x.float()).to(dtype)
    ref = (x.float() + 0.5 * torch.randn(n, A, generator=gen)).to(dtype) if with_ref else None
    return x, mask, actions, ref


def test_the_vector_form_is_the_oracle():
    x, mask, actions, ref = _many(3, 900, 7, torch.float32, True)
    offsets = [2, 9, 9, 120, 400, 640, 899]
    for r in (ref, None):
        want = oracle.preference(_np(x), actions.numpy(), mask.numpy(), offsets, None if r is None else _np(r), 0.2, 0.1)
        got = _preference64(x, actions, mask, offsets, r, 0.2, 0.1)
        for k in want:
            _close(got[k], want[k], 1e-12, k)


@pytest.mark.parametrize("n,pairs", [(20000, 400), (70000, 150)], ids=["short", "long"])
def test_one_long_sequence_among_many(n, pairs):
    """A sequence of most of the call's rows, which the kernels ask the offsets for, among short ones and empty ones, at
    the head, in the middle and at the end."""
    x, mask, actions, ref = _many(n, n, 5, torch.float32, True)
    short = [0, 3, 11, 0, 7]
    for at in (0, pairs, 2 * pairs - 1):
        lens = [short[k % 5] for k in range(2 * pairs)]
        lens[at] = n - 50 - (sum(lens) - lens[at])
        offsets = np.concatenate(([20], 20 + np.cumsum(lens)))
        o = _preference64(x, actions, mask, offsets, ref, 0.01, 0.1)
        got = policy.preference_loss_and_grad(*(t.to(DEV) for t in (x, actions, mask)), torch.tensor(offsets, device=DEV),
                                              ref_logits=ref.to(DEV), beta=0.01, label_smoothing=0.1)
        base._check_preference(got, o, x, mask, 0.01, torch.float32)


@pytest.mark.parametrize("pairs", [30000, 24000], ids=["short", "long"])
@pytest.mark.parametrize("wide", [False, True], ids=["int32", "int64"])
def test_offsets_that_do_not_ascend_are_not_walked(pairs, wide):
    """2^22 rows; every other pair is 0, n / 2, n, or every sequence all the rows, so that walking them all would be 10^10
    rows and more: the loss is NaN, in about the time of a good call's."""
    n, A = 1 << 22, 2
    x = torch.zeros(n, A, dtype=torch.float16, device=DEV)
    words = torch.full((n,), 3, dtype=torch.int32, device=DEV)
    acts = torch.zeros(n, dtype=torch.int8, device=DEV)
    good = torch.arange(2 * pairs + 1) * (n // (2 * pairs))
    alternate = torch.tensor([0, n // 2, n, 0] * (pairs // 2) + [0])
    whole = torch.tensor([0, n] * pairs + [0])
    started, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for offsets in (good, good, alternate, whole, n - whole):
        off = offsets.to(torch.int64 if wide else torch.int32).to(DEV)
        started.record()
        got = policy.preference_loss_and_grad(x, acts, words, off)
        ended.record()
        ended.synchronize()
        assert math.isnan(float(got.loss)) == (offsets is not good)
        assert started.elapsed_time(ended) < (1000 if offsets is good else 4)


# ------------------------------------------------------------ trajectories
def test_policy_trajectory_buffers_are_checked_before_a_step():
    """Buffers that a step would write past, of another type or layout, or missing: refused, the env as it was; longer
    buffers are filled as far as asked."""
    B, T = 24, 3
    env = BatchedCoupEnv(B, seed=6, auto_reset=True, obs=True)
    logits, values = torch.zeros(B, 18, device=DEV), torch.zeros(B, device=DEV)
    before = env.export_state().clone()
    good = env.policy_trajectory_buffers(T)
    bad = [dict(good, actions=good["actions"][:2]), dict(good, rewards=good["rewards"][:, :8].contiguous()),
           dict(good, legal_mask=good["legal_mask"].long()), dict(good, obs=good["obs"].half()),
           dict(good, step_type=good["step_type"].cpu()), dict(good, log_probs=good["log_probs"][0]),
           dict(good, current_player=good["current_player"].t().contiguous().t()),
           dict(good, decision_obs=good["obs"][:, :, :1]), {k: v for k, v in good.items() if k != "decision_player"},
           dict(good, values=torch.zeros(T, B, dtype=torch.float64, device=DEV))]
    for buf in bad:
        with pytest.raises(ValueError, match="buf"):
            env.collect_policy_trajectory(T, lambda ts: logits, buf)
    for wrong in (values[:1], values[:, None], values.repeat(2)):
        with pytest.raises(ValueError, match="values must be"):
            env.collect_policy_trajectory(T, lambda ts: (logits, wrong))
    assert torch.equal(env.export_state(), before)
    longer = env.policy_trajectory_buffers(T + 2)
    longer["actions"].fill_(99)
    assert env.collect_policy_trajectory(T, lambda ts: logits, longer) is longer
    assert (longer["actions"][:T] < 18).all() and (longer["actions"][T:] == 99).all()
    few = {k: good[k] for k in ("legal_mask", "current_player", "decision_mask", "decision_player", "log_probs")}
    env.collect_policy_trajectory(T, lambda ts: logits, few)  # what else a step writes need not be recorded
    assert env.error_count() == 0


# ------------------------------------------------------------ derivatives
def test_forward_mode_derivatives_are_refused():
    """A dual tensor in any place raises, with and without logits that require a gradient, and so does a derivative that
    comes in as one: their tangents would be lost without a word.  Detached, and outside the dual level, all is as ever."""
    n, A = 16, 18
    x, mask, actions, ref, old, adv = (t.to(DEV) for t in base._policy_inputs(2, n, A, torch.float32))
    off, u = torch.tensor([0, 4, 16], device=DEV), torch.rand(n, device=DEV)
    window = [t.to(DEV) for t in base._window(torch.Generator().manual_seed(1), 4, 5, 2, torch.float32)]
    one = torch.ones((), device=DEV)
    dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    leaf = x.clone().requires_grad_()
    with torch.autograd.forward_ad.dual_level():
        for logits in (x, leaf):
            for call in (lambda x: policy.policy_loss(x, actions, mask, old, adv),
                         lambda x: policy.preference_loss(x, actions, mask, off)):
                with pytest.raises(ValueError, match="forward-mode"):
                    call(dual(logits))
            for kw in (dict(old_log_probs=dual(old)), dict(advantages=dual(adv)), dict(ref_logits=dual(ref))):
                with pytest.raises(ValueError, match="forward-mode|held constant"):
                    policy.policy_loss(logits, actions, mask, **{**dict(old_log_probs=old, advantages=adv), **kw})
            with pytest.raises(ValueError, match="forward-mode|held constant"):
                policy.preference_loss(logits, actions, mask, off, ref_logits=dual(ref))
        for call in (lambda: policy.sample_actions(dual(x), mask, u), lambda: policy.sample_actions(x, mask, dual(u)),
                     lambda: policy.policy_loss_and_grad(dual(x), actions, mask, old, adv),
                     lambda: policy.policy_loss_and_grad(x, actions, mask, old, adv, grad_scale=dual(one)),
                     lambda: policy.preference_loss_and_grad(dual(x), actions, mask, off),
                     lambda: policy.advantages(*window[:3], dual(window[3]), window[4]),
                     lambda: policy.advantages(*window[:4], dual(window[4]))):
            with pytest.raises(ValueError, match="forward-mode|held constant"):
                call()
        out = policy.policy_loss(leaf, actions, mask, old, adv)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out.loss, leaf, dual(one))
        inside = policy.policy_loss(dual(x).detach(), actions, mask, old, adv)
        policy.policy_loss(leaf, actions, mask, old, adv, ref_logits=dual(ref).detach()).loss.backward()
    assert torch.equal(inside.loss, policy.policy_loss(x, actions, mask, old, adv).loss) and leaf.grad is not None


@pytest.mark.parametrize("dtype", base.DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("hooks", ["save_on_cpu", "clone", "checkpoint"])
def test_losses_under_saved_tensor_hooks(hooks, dtype):
    """Hooks that hand out equal tensors at other addresses (and of other strides), and a checkpoint that computes them
    again: the gradients without hooks, in the first backward pass and in a second one."""
    n, A = 300, 18
    x, mask, actions, ref, old, adv = (t.to(DEV) for t in base._policy_inputs(7, n, A, dtype))
    off = torch.tensor([0, 30, 100, 180, 300], device=DEV)
    wide = torch.zeros(n, 40, dtype=dtype, device=DEV)
    wide[:, 3:21] = x
    twice = [t.repeat_interleave(2)[::2] for t in (actions, mask, old, adv)]

    def both(table):
        logits = table[:, 3:21]
        return (policy.policy_loss(logits, *twice, ref_logits=ref, kl_coef=0.1).loss
                + policy.preference_loss(logits, twice[0], twice[1], off, ref_logits=ref).loss)

    def gradients(call):
        leaf = wide.clone().requires_grad_()
        loss = call(leaf)
        return [torch.autograd.grad(loss, leaf, retain_graph=True)[0] for _ in range(2)]

    want = gradients(both)
    assert want[0].any() and torch.equal(want[0], want[1])
    if hooks == "checkpoint":
        got = gradients(lambda t: torch.utils.checkpoint.checkpoint(both, t, use_reentrant=False))
    else:
        with (torch.autograd.graph.save_on_cpu() if hooks == "save_on_cpu" else
              torch.autograd.graph.saved_tensors_hooks(torch.clone, torch.clone)):
            got = gradients(both)
    for g in got:
        assert torch.equal(g, want[0])


# ------------------------------------------------------------ nearly sure decisions
def _sure(seed, n, A, dtype):
    """Rows whose acted action is 10 to 20 above all others, two of them legal at least."""
    gen = torch.Generator().manual_seed(seed)
    actions = torch.randint(A, (n,), generator=gen)
    legal = torch.rand(n, A, generator=gen) < 0.5
    row = torch.arange(n)
    legal[row, actions] = legal[row, (actions + 1) % A] = True
    x = 3.0 - 10.0 - 10.0 * torch.rand(n, A, generator=gen)
    x[row, actions] = 3.0
    mask = (legal.long() << torch.arange(A)).sum(1).to(torch.int32)
    return x.to(dtype), mask, actions.to(torch.int8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("A", [4, 18, 31])
@pytest.mark.parametrize("times", [1, 30, 170], ids=lambda k: f"{400 * k} rows")
def test_nearly_sure_decisions_keep_their_digits(times, A, dtype):
    """1 - p of 1e-3 to 1e-9: the log probability and every gradient entry, the acted action's too, to the softmax's
    relative error (the logits' z = 20) of themselves.  Ratios of about 1 and a surrogate weight of either sign; pairs of
    short sequences, and one pair of long ones."""
    n, z = 400, 20
    x, mask, actions = _sure(A, n, A, dtype)
    old, adv = torch.full((n,), -0.01), torch.where(torch.arange(n) % 2 == 0, 1.0, -0.5)
    o = oracle.policy(_np(x), actions.numpy(), mask.numpy(), _np(old), _np(adv), None, None, 0.2, 0.2, 0.0, 0.05)
    assert -A * math.exp(-10) < o["log_probs"].min() and o["log_probs"].max() < 0  # A - 1 others of e^-10 at most
    info, rel = torch.finfo(dtype), 8 * (48 + 2 * z) * H
    many = lambda t: t.to(DEV).repeat(times, *[1] * (t.dim() - 1))  # noqa: E731
    xm, am, mm = many(x), many(actions), many(mask)
    got = policy.policy_loss_and_grad(xm, am, mm, many(old), many(adv), entropy_coef=0.05)
    where = slice((times - 1) * n, times * n)
    _close(got.log_probs[where].cpu().numpy(), o["log_probs"], rel * np.abs(o["log_probs"]), "log_probs")
    want = o["grad"] / times
    _close(_np(got.grad[where]), want, (rel + info.eps / 2) * np.abs(want) + info.smallest_normal * info.eps, "policy grad")
    u = torch.full((n * times,), 0.5, device=DEV)
    acts, lp = policy.sample_actions(xm, mm, u)
    assert torch.equal(acts, am)
    _close(lp[where].cpu().numpy(), o["log_probs"], rel * np.abs(o["log_probs"]), "sample's log_probs")
    short = [n * k // 8 for k in range(9)]
    for offsets in ([*(r * n + v for r in range(times) for v in short[:-1]), times * n], [0, times * n // 2, times * n]):
        o = _preference64(x.repeat(times, 1), actions.repeat(times), mask.repeat(times), offsets, None, 0.1, 0.1)
        got = policy.preference_loss_and_grad(xm, am, mm, torch.tensor(offsets, device=DEV), label_smoothing=0.1)
        # 1 - p of the vector form's own log_softmax is good to 2^-53 of 1 only
        p = x.repeat(times, 1).double().masked_fill(((mask.repeat(times)[:, None] >> torch.arange(A)) & 1) == 0, -math.inf)
        p = torch.softmax(p, 1).numpy()
        acted = np.arange(A) == actions.repeat(times).numpy()[:, None]
        rest = np.where(acted, 0.0, p).sum(1)
        want = np.where(acted, -(o["grad"] * ~acted).sum(1, keepdims=True), o["grad"])
        assert (rest > 1e-10).all() and np.abs(want[acted]).min() > 0
        # the pair's weight moves by its difference's error, beta * rows * 32-bit roundings of a log ratio near 0
        lim = (rel + 0.1 * o["length"].max() * 8 * H + info.eps / 2) * np.abs(want) + info.smallest_normal * info.eps
        _close(_np(got.grad), want, lim, "preference grad")


def test_a_very_sure_pairs_small_loss():
    """Pairs 40 to 85 apart, where the constant's part that log2(e) rounds off weighs 85 * 1.3e-8: e^-x to a few 2^-24.
    The rows' other action is 40 below or more: its e leaves no trace in the log probabilities, which are then 32-bit
    numbers, and their 64-bit sums are exact."""
    depth = torch.tensor([40.0, 55.5, 70.25, 84.875])
    x = torch.zeros(8, 2)
    x[1::2, 1] = -depth  # the rejected row takes it; the chosen one is certain
    actions = (torch.arange(8) % 2).to(torch.int8)
    mask = torch.tensor([1, 3] * 4, dtype=torch.int32)
    for k in range(4):
        off = torch.tensor([2 * k, 2 * k + 1, 2 * k + 2], device=DEV)
        got = policy.preference_loss_and_grad(x.to(DEV), actions.to(DEV), mask.to(DEV), off, beta=1.0)
        want = math.exp(-float(depth[k]))
        assert abs(float(got.loss) / want - 1) <= 8 * H
        assert abs(float(got.grad[2 * k + 1, 1]) / want - 1) <= 16 * H


@pytest.mark.parametrize("dtype", base.DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("scale", [math.inf, math.nan])
def test_masked_entries_stay_zero_under_a_scale_without_bound(scale, dtype):
    """A loss scaler's infinite factor, or a NaN that comes in: rows that do not count and actions outside the word get 0
    all the same, the others something that is no number."""
    n, A = 200, 18
    x, mask, actions, ref, old, adv = (t.to(DEV) for t in base._policy_inputs(9, n, A, dtype))
    x[0] = torch.arange(A, device=DEV) / 4  # a row of the loss whose every legal action has a share
    mask[0], actions[0], old[0], adv[0], ref[0] = 0x155, 2, -1.5, 1.0, 0.0
    off = torch.tensor([0, 20, 60, 90, 180], device=DEV)
    factor = torch.tensor(scale, device=DEV)
    kw = dict(ref_logits=ref, kl_coef=0.1, entropy_coef=0.01)
    legal = ((mask[:, None] >> torch.arange(A, device=DEV)) & 1).bool() & (mask >= 0)[:, None]
    counts = legal.gather(1, actions.long().clamp(0, A - 1)[:, None])[:, 0] & (actions >= 0) & (actions < A)
    live = legal & counts[:, None]
    leaf = x.clone().requires_grad_()
    for loss, both in ((lambda t, **k: policy.policy_loss(t, actions, mask, old, adv, **kw),
                        lambda t, **k: policy.policy_loss_and_grad(t, actions, mask, old, adv, **kw, **k)),
                       (lambda t, **k: policy.preference_loss(t, actions, mask, off, ref_logits=ref),
                        lambda t, **k: policy.preference_loss_and_grad(t, actions, mask, off, ref_logits=ref, **k))):
        first = torch.autograd.grad(loss(leaf).loss, leaf, factor)[0]
        for g in (first, both(x, grad_scale=factor).grad):
            assert not g[~live].any() and not torch.isfinite(g[0][live[0]]).any()


# ------------------------------------------------------------ forms that larger calls take
@pytest.mark.parametrize("dtype", base.DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("A", [5, 16, 18, 31])
@pytest.mark.parametrize("with_ref", [True, False], ids=["ref", "none"])
def test_short_sequences_of_many_rows(with_ref, A, dtype):
    """More than 16,384 rows in short sequences (32-bit sums within a tile): groups of one tile and of several, empty
    sequences, rows outside every one; the loss alone, with its gradient and through autograd."""
    pairs = 300
    x, mask, actions, ref = _many(A, 18003, A, dtype, with_ref)
    gen = torch.Generator().manual_seed(A)
    lens = torch.randint(0, 55, (2 * pairs,), generator=gen)
    lens[100], lens[301], lens[302], lens[7:12] = 300, 700, 520, 0
    offsets = (11 + torch.cat((torch.zeros(1, dtype=torch.int64), lens.cumsum(0)))).tolist()
    assert 16384 < offsets[-1] < 18000 and 18003 // pairs <= 160
    o = _preference64(x, actions, mask, offsets, ref, 0.05, 0.1)
    args = [t.to(DEV) for t in (actions, mask)] + [torch.tensor(offsets, device=DEV)]
    kw = dict(ref_logits=None if ref is None else ref.to(DEV), beta=0.05, label_smoothing=0.1)
    got = policy.preference_loss_and_grad(x.to(DEV), *args, **kw)
    base._check_preference(got, o, x, mask, 0.05, dtype)
    assert not got.grad[:11].any() and not got.grad[offsets[-1]:].any()
    leaf = x.to(DEV).requires_grad_()
    out = policy.preference_loss(leaf, *args, **kw)
    grad, = torch.autograd.grad(out.loss, leaf)
    only = policy.preference_loss(x.to(DEV), *args, **kw)
    for a, b in zip((out.loss, out.rewards, grad, only.loss, only.rewards), (*got, got.loss, got.rewards)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cuts", [0, 1, 3])
@pytest.mark.parametrize("T,B,P", [(2305, 9, 2), (5000, 130, 2), (700, 250, 6), (500, 1500, 2), (300, 5, 3), (1000, 600, 6),
                                   (257, 2100, 2), (130, 8000, 4), (4000, 300, 2), (70, 33000, 2), (200, 16500, 3),
                                   (9, 140000, 2), (40, 140000, 2)])
def test_what_lies_far_behind_reaches_every_step(T, B, P, cuts):
    """gamma = lam = 1: an advantage is every reward up to the lane's next cut (or the bootstrap) less the value, however
    many rounds behind a block's part they lie.  Whole rewards, values in eighths: every sum is exact in 32 bits
    (3 T + 4 < 2^17), so is the comparison."""
    gen = torch.Generator().manual_seed(T + B + cuts)
    st = torch.ones(T, B, dtype=torch.uint8)
    lane = torch.arange(B)
    for k in range(cuts):
        st[torch.randint(0, T, (B,), generator=gen), lane] = 2 if k != 1 else 0
    pl = torch.randint(0, P, (T, B), generator=gen).to(torch.int8)
    r = torch.randint(-3, 4, (T, B, P), generator=gen).to(torch.int8)
    v = torch.randint(-32, 33, (T, B), generator=gen).float() / 8
    b = torch.randint(-32, 33, (B, P), generator=gen).float() / 8
    togo, want = b.clone(), torch.zeros(T, B)
    for t in range(T - 1, -1, -1):
        togo[st[t] != 1] = 0
        togo += r[t] * (st[t] != 0)[:, None]
        want[t] = torch.where(st[t] != 0, togo[lane, pl[t].long()], 0.0)
    for dtype in (torch.float32, torch.bfloat16):
        adv, target = policy.advantages(r.to(DEV), st.to(DEV), pl.to(DEV), v.to(dtype).to(DEV), b.to(dtype).to(DEV),
                                        gamma=1.0, lam=1.0)
        assert torch.equal(target.cpu(), want)
        assert torch.equal(adv.cpu(), torch.where(st != 0, want - v, 0.0))


# ------------------------------------------------------------ the documented round
@pytest.mark.parametrize("auto_reset", [True, False])
def test_a_round_with_open_games(auto_reset):
    """The guide's policy update: acting seats' observations, and the last step's as each seat's bootstrap for the games
    left open; advantages and loss against the oracle."""
    B, T = 40, 30
    env = BatchedCoupEnv(B, seed=5, auto_reset=auto_reset, obs=True, num_players=3)
    torch.manual_seed(1)
    model = torch.nn.Linear(env.obs_size, 18 + 1, device=DEV)

    def act(ts):
        seat = ts["current_player"].long().clamp(min=0)
        out = model(ts["obs"][torch.arange(env.batch, device=env.device), seat]).detach()
        return out[:, :18], out[:, 18]

    buf = env.collect_policy_trajectory(T, act)
    bootstrap = model(buf["obs"][-1])[..., 18].detach()
    assert bootstrap.shape == (B, 3)
    given = (buf["rewards"], buf["step_type"], buf["decision_player"], buf["values"])
    adv, target = policy.advantages(*given, bootstrap, gamma=0.99)
    want, _ = oracle.advantages(*(t.cpu().numpy() for t in given[:3]), _np(buf["values"]), _np(bootstrap), 0.99, 0.95)
    # sums of at most T terms, below T (3 + 2 * 4) in size, 4 roundings a term
    _close(adv.cpu().numpy(), want, 4 * T * H * T * 11, "advantages")
    unopened = policy.advantages(*given, gamma=0.99)[0]
    still = buf["step_type"][-1] == 1
    assert still.any() and (unopened - adv)[-1][still].abs().max() > 0.01
    seat = buf["decision_player"].long().clamp(min=0)[:, :, None, None].expand(-1, -1, 1, env.obs_size)
    logits = model(buf["decision_obs"].gather(2, seat)[:, :, 0])[..., :18]
    kw = dict(kl_coef=0.05, ref_logits=logits.detach() * 0.9, active=buf["decision_player"] == 0)
    out = policy.policy_loss(logits, buf["actions"], buf["decision_mask"], buf["log_probs"], adv, **kw)
    out.loss.backward()
    flat = lambda t: _np(t).reshape(T * B, -1).squeeze()  # noqa: E731
    o = oracle.policy(flat(logits), flat(buf["actions"]), buf["decision_mask"].flatten().cpu().numpy(), flat(buf["log_probs"]),
                      flat(adv), flat(kw["ref_logits"]), flat(kw["active"]) > 0, 0.2, 0.2, 0.05, 0.0)
    assert int(out.count) == o["count"] > 0 and torch.isfinite(model.weight.grad).all() and model.weight.grad.any()
    z = base._reach(logits.detach().reshape(T * B, 18).cpu(), buf["decision_mask"].flatten().cpu())
    assert abs(float(out.loss.detach()) - o["loss"]) <= 8 * (48 + 2 * z) * H * (o["mass"].sum() + 3 * z)


@pytest.mark.parametrize("auto_reset", [True, False])
def test_policy_trajectory_of_information_states(auto_reset):
    """An env that writes information states: each decision's is the state's before the step, and what the policy got; a
    lane whose logits are no numbers is skipped."""
    B, T = 50, 12
    kw = dict(seed=3, auto_reset=auto_reset, obs=False, info_state=True, history=True)
    env, ref = BatchedCoupEnv(B, **kw), BatchedCoupEnv(B, **kw)
    seen = []

    def act(ts):
        assert "obs" not in ts
        seen.append(ts["info_state"].clone())
        logits = torch.zeros(B, 18, device=DEV)
        logits[7] = math.nan
        return logits

    buf = env.collect_policy_trajectory(T, act, generator=torch.Generator(DEV).manual_seed(1))
    now = ref.query(obs=False, info_state=True)
    for t in range(T):
        assert torch.equal(buf["decision_info_state"][t], now["info_state"]) and torch.equal(seen[t], now["info_state"])
        over = now["terminal"].bool()
        ref.step(buf["actions"][t].masked_fill(over, 0))
        now = ref.query(obs=False, info_state=True)
    assert (buf["actions"][:, 7] == -1).all() and (buf["step_type"][:, 7] == 3).all() and buf["log_probs"][:, 7].isnan().all()
    assert torch.equal(env.export_state(), ref.export_state()) and env.error_count() == 0


@pytest.mark.parametrize("dtype", base.DTYPES, ids=lambda d: str(d)[6:])
def test_excluded_actions_in_strided_tables_and_graphs(dtype):
    """Rows whose reference excludes an action the policy takes, in strided tables, captured and replayed: the contiguous,
    eager call's results."""
    n, A = 700, 18
    x, mask, actions, ref, old, adv = (t.to(DEV) for t in base._policy_inputs(13, n, A, dtype))
    rows = torch.arange(n, device=DEV)
    ref[rows[::3], rows[::3] % A] = -math.inf
    ref[rows[1::3], rows[1::3] % A] = torch.finfo(dtype).min
    wide = torch.zeros(n, 2, 41, dtype=dtype, device=DEV)
    wide[:, 0, 5:23], wide[:, 1, 3:21] = x, ref
    kw = dict(kl_coef=0.1, entropy_coef=0.01)
    want = policy.policy_loss_and_grad(x, actions, mask, old, adv, ref_logits=ref, **kw)
    # a row whose one legal action the reference excludes has no reference at all: NaN, and so is the mean
    assert math.isnan(float(want.loss)) and want.grad.isnan().any() and (want.grad == 0).any()
    strided = lambda: policy.policy_loss_and_grad(wide[:, 0, 5:23], actions, mask, old, adv,  # noqa: E731
                                                  ref_logits=wide[:, 1, 3:21], **kw)
    held = [strided()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.append(strided())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for got in held:
            for a, b in zip(got, want):
                assert torch.equal(a.nan_to_num(5), b.nan_to_num(5))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("n", [64, 70000])
def test_decisions_of_a_types_lowest_logit(n, dtype):
    """An acted action of the type's lowest logit, 3.4e38 below the others: its ratio is 0 (clipped for a negative
    advantage), without a gradient; a rejected sequence that holds one costs nothing, a chosen one 3.4e38, in calls of few
    rows and of many."""
    low = torch.finfo(dtype).min
    x = torch.zeros(n, 3, dtype=dtype, device=DEV)
    x[:, 1] = low
    words = torch.full((n,), 7, dtype=torch.int32, device=DEV)
    acts = torch.ones(n, dtype=torch.int8, device=DEV)
    old = torch.full((n,), -1.0, device=DEV)
    for adv, loss in ((1.0, 0.0), (-1.0, 0.8)):
        got = policy.policy_loss_and_grad(x, acts, words, old, torch.full((n,), adv, device=DEV))
        assert abs(float(got.loss) - loss) <= 4 * H and not got.grad.any()
        assert (got.log_probs == float(low)).all()
    for each in (1, n // 2):  # short sequences, and (of 70,000 rows) long ones
        taken = torch.zeros(n, dtype=torch.int8, device=DEV)
        off = torch.arange(0, n + 1, each, device=DEV)
        taken[each] = 1  # the first rejected row
        got = policy.preference_loss_and_grad(x, taken, words, off, beta=1.0)
        pairs = n // each // 2
        assert abs(float(got.loss) - (pairs - 1) * math.log(2) / pairs) <= 16 * H and torch.isfinite(got.grad).all()
        taken[each], taken[0] = 0, 1
        got = policy.preference_loss_and_grad(x, taken, words, off, beta=1.0)
        _close(float(got.loss), -low / pairs, 4 * H * -low / pairs, "loss")
        assert torch.isfinite(got.grad).all()


@pytest.mark.parametrize("pairs,each", [(4, 50), (600, 50), (200, 400)], ids=["short-few", "short", "long"])
def test_sums_of_lowest_logits_keep_their_range(pairs, each):
    """Two acted actions of float32's lowest logit in each of a pair's sequences: sums of -6.8e38, past 32 bits' range,
    whose difference is 0; 0.1 of them is a reward within it."""
    n, low = pairs * each, torch.finfo(torch.float32).min
    x = torch.zeros(n, 3, device=DEV)
    x[:, 1] = low
    words = torch.full((n,), 7, dtype=torch.int32, device=DEV)
    taken = torch.zeros(n, dtype=torch.int8, device=DEV)
    taken[[0, 1, each // 2, each // 2 + 1]] = 1
    off = torch.arange(0, n + 1, each // 2, device=DEV)
    got = policy.preference_loss_and_grad(x, taken, words, off, beta=0.1)
    _close(got.rewards[:2].cpu().numpy(), np.full(2, 0.2 * low), 2 * H * 0.2 * -low, "rewards")
    assert abs(float(got.loss) - math.log(2)) <= 16 * H and torch.isfinite(got.grad).all()
