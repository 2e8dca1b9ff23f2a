"""The learner-side operators over the batched environment's trajectories, as cases to measure.

Four operators work on what `BatchedCoupEnv` hands a learner -- logits over the game's actions, legal-action words,
acted actions, rewards, step types and acting players:

  sample      an action and its log probability from masked logits and given uniform numbers (the acting side);
  advantages  generalised advantages and value targets over [T, B] trajectories in which the players take turns;
  policy      the clipped policy loss with a KL term to a reference policy and an entropy bonus, and its gradient;
  preference  the paired log-ratio loss over packed chosen / rejected sequences of decisions, and its gradient.

`run` computes them from elementary torch operations where `own` is false, and through open_spiel_coup_amd.policy where
it is true.  A row is a decision where its action is legal: bit `action` of its mask word is set, the action is one of
the A, and bit 31 (a chance node) is clear.  Other rows count for nothing, whatever they hold.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CHANCE = -(1 << 31)


# ------------------------------------------------------------------ cases
def listed():
    return [
        # acting: one game answered (a served opponent: only the latency counts)
        {"name": "act-1", "op": "sample", "rows": 1, "actions": 18, "dtype": "f32"},
        # acting: every lane of the 2^20-lane batch, logits as a bf16 network leaves them
        {"name": "act-1048576-bf16", "op": "sample", "rows": 1 << 20, "actions": 18, "dtype": "bf16"},
        # advantages: few lanes over a long window (evaluation games, one lane a wave or less)
        {"name": "adv-4096x33", "op": "advantages", "steps": 4096, "lanes": 33, "players": 2, "dtype": "f32",
         "gamma": 0.99, "lam": 0.95},
        # advantages: the ordinary window of a learner over the 65,536-lane batch
        {"name": "adv-64x65536", "op": "advantages", "steps": 64, "lanes": 65536, "players": 2, "dtype": "f32",
         "gamma": 0.99, "lam": 0.95},
        # advantages: 20 steps of the 6-player 2^20-lane batch, values of a bf16 critic
        {"name": "adv-20x1048576-6p", "op": "advantages", "steps": 20, "lanes": 1 << 20, "players": 6, "dtype": "bf16",
         "gamma": 1.0, "lam": 0.9},
        # policy update: a small odd minibatch, through autograd
        {"name": "ppo-777", "op": "policy", "rows": 777, "actions": 18, "dtype": "f32", "ref": True, "active": False,
         "grad": "autograd", "kl": 0.05, "entropy": 0.01, "low": 0.2, "high": 0.2},
        # a held-out window scored without a gradient (early stopping by its KL)
        {"name": "ppo-262145-eval-f16", "op": "policy", "rows": 262145, "actions": 18, "dtype": "f16", "ref": True,
         "active": False, "grad": "none", "kl": 0.05, "entropy": 0.01, "low": 0.2, "high": 0.2},
        # policy update: 20 steps x 65,536 lanes, one player's decisions of them, a bf16 network
        {"name": "ppo-20x65536-bf16", "op": "policy", "rows": 20 * 65536, "actions": 18, "dtype": "bf16", "ref": True,
         "active": True, "grad": "call", "kl": 0.05, "entropy": 0.01, "low": 0.2, "high": 0.28},
        # policy update: 4 steps x 2^20 lanes, float logits
        {"name": "ppo-4x1048576", "op": "policy", "rows": 4 << 20, "actions": 18, "dtype": "f32", "ref": True,
         "active": False, "grad": "call", "kl": 0.05, "entropy": 0.01, "low": 0.2, "high": 0.2},
        # preferences: a few pairs of games
        {"name": "pref-24-f16", "op": "preference", "pairs": 24, "rows": 1031, "actions": 18, "dtype": "f16", "ref": True,
         "grad": "autograd", "beta": 0.1, "smoothing": 0.0},
        # preferences: 8192 games, the winner's decisions against the loser's
        {"name": "pref-8192-bf16", "op": "preference", "pairs": 8192, "rows": 327680, "actions": 18, "dtype": "bf16",
         "ref": True, "grad": "call", "beta": 0.1, "smoothing": 0.1},
        # preferences: few pairs of long runs of decisions (whole sessions of one policy against another's)
        {"name": "pref-8-long", "op": "preference", "pairs": 8, "rows": 1500007, "actions": 18, "dtype": "f32",
         "ref": True, "grad": "call", "beta": 0.02, "smoothing": 0.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["sample", "advantages", "policy", "preference"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    actions = 18 if rng.random() < 0.5 else rng.randint(2, 31)
    if op == "sample":
        return {"op": op, "rows": _log_int(rng, 1, 1 << 20), "actions": actions, "dtype": dtype}
    if op == "advantages":
        steps = _log_int(rng, 1, 2048)
        return {"op": op, "steps": steps, "lanes": _log_int(rng, 1, min(1 << 20, (20 << 20) // steps)),
                "players": rng.choice([2, 2, 3, 4, 5, 6]), "dtype": dtype, "gamma": rng.choice([1.0, 0.99]),
                "lam": rng.choice([1.0, 0.95, 0.5])}
    if op == "policy":
        return {"op": op, "rows": _log_int(rng, 1, 1 << 20), "actions": actions, "dtype": dtype,
                "ref": rng.random() < 0.7, "active": rng.random() < 0.4, "grad": rng.choice(["none", "autograd", "call"]),
                "kl": rng.choice([0.02, 0.2]), "entropy": rng.choice([0.0, 0.01]), "low": rng.choice([0.1, 0.2]),
                "high": rng.choice([0.2, 0.3])}
    pairs = _log_int(rng, 1, 16384)
    return {"op": op, "pairs": pairs, "rows": _log_int(rng, 2 * pairs, min(1 << 20, 20000 * pairs)), "actions": actions,
            "dtype": dtype, "ref": rng.random() < 0.7, "grad": rng.choice(["autograd", "call"]),
            "beta": rng.choice([0.02, 0.1]), "smoothing": rng.choice([0.0, 0.1])}


# ------------------------------------------------------------------ inputs
def _decisions(gen, rows, A, dtype, dev):
    """Logits, mask words and actions of `rows` decisions: about five of the A actions legal; one row in 32 terminal
    (no legal action), one in 64 a chance node, one in 64 acted outside its mask; masked logits hold anything."""
    legal = torch.rand(rows, A, generator=gen, device=dev) < min(0.9, 5.0 / A)
    score = torch.rand(rows, A, generator=gen, device=dev)
    legal |= score == score.amax(1, keepdim=True)  # one at least
    kind = torch.rand(rows, generator=gen, device=dev)
    legal &= (kind >= 1 / 32)[:, None]
    actions = torch.where(legal, score, -1.0).argmax(1)
    actions = torch.where(kind < 1 / 32, -1, actions)
    stray = (kind >= 1 / 32) & (kind < 1 / 32 + 1 / 64)
    actions = torch.where(stray, (~legal).int().argmax(1), actions)
    bits = (legal.long() << torch.arange(A, device=dev)).sum(1)
    bits = torch.where((kind >= 1 / 32 + 1 / 64) & (kind < 1 / 32 + 2 / 64), bits - (1 << 31), bits)
    logits = 2.0 * torch.randn(rows, A, generator=gen, device=dev)
    waste = torch.randint(0, 8, (rows, A), generator=gen, device=dev)
    logits = torch.where(~legal & (waste == 0), float("nan"), logits)
    logits = torch.where(~legal & (waste == 1), float("inf"), logits)
    logits = torch.where(~legal & (waste == 2), torch.finfo(dtype).min, logits)
    return logits.to(dtype), bits.to(torch.int32), actions.to(torch.int8)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "advantages":
        T, B, P = case["steps"], case["lanes"], case["players"]
        kind = torch.rand(T, B, generator=gen, device=dev)
        first = kind < 1 / 64
        skipped = (kind >= 1 / 64) & (kind < 2 / 64)
        last = (kind >= 2 / 64) & (kind < 2 / 64 + 1 / 16)
        s["step_type"] = torch.where(first, 0, torch.where(skipped, 3, torch.where(last, 2, 1))).to(torch.uint8)
        player = torch.randint(0, P, (T, B), generator=gen, device=dev)
        s["players"] = torch.where(first | skipped, -1, player).to(torch.int8)
        loser = torch.randint(0, 4 * P, (T, B, 1), generator=gen, device=dev)  # a card lost in one step of four
        seat = torch.arange(P, device=dev)
        rewards = torch.where(loser < P, torch.where(loser == seat, 1 - P, 1), 0)
        s["rewards"] = (rewards * ~(first | skipped)[:, :, None]).to(torch.int8)
        values = 0.7 * torch.randn(T, B, generator=gen, device=dev)
        s["values"] = torch.where(first | skipped, float("nan"), values).to(dtype)
        s["bootstrap"] = (0.7 * torch.randn(B, P, generator=gen, device=dev)).to(dtype)
        return s
    s["logits"], s["mask"], s["actions"] = _decisions(gen, case["rows"], case["actions"], dtype, dev)
    if case["op"] == "sample":
        s["uniform"] = torch.rand(case["rows"], generator=gen, device=dev)
        return s
    s["ref"] = None
    if case["ref"]:
        noise = 0.3 * torch.randn(case["rows"], case["actions"], generator=gen, device=dev)
        s["ref"] = (s["logits"].float() + noise).to(dtype)
    if case["op"] == "policy":
        legal = _legal(s["mask"], case["actions"])
        logp = _log_softmax(s["logits"].float(), legal)
        taken = logp.gather(1, s["actions"].long().clamp(0)[:, None])[:, 0]
        moved = taken + 0.2 * torch.randn(case["rows"], generator=gen, device=dev)
        real = _decided(legal, s["actions"])
        s["old"] = torch.where(real, moved, float("nan"))
        s["adv"] = torch.where(real, torch.randn(case["rows"], generator=gen, device=dev), float("inf"))
        s["active"] = torch.rand(case["rows"], generator=gen, device=dev) < 0.5 if case["active"] else None
    else:
        used = case["rows"] - case["rows"] // 37  # rows behind the last sequence belong to none
        cuts = torch.randint(0, used + 1, (2 * case["pairs"] - 1,), generator=gen, device=dev).sort().values
        ends = torch.tensor([0, used], device=dev)
        s["offsets"] = torch.cat((ends[:1], cuts, ends[1:])).to(torch.int32)
    s["train"] = s["logits"].clone().requires_grad_() if case["grad"] == "autograd" else None
    return s


# ------------------------------------------------------------------ the plain forms
def _legal(mask, A):
    bits = (mask[:, None] >> torch.arange(A, device=mask.device, dtype=torch.int32)) & 1
    return (bits != 0) & (mask >= 0)[:, None]


def _decided(legal, actions):
    A = legal.shape[1]
    a = actions.long()
    return (a >= 0) & (a < A) & legal.gather(1, a.clamp(0, A - 1)[:, None])[:, 0]


def _log_softmax(x, legal):
    """log softmax over the legal actions; 0 where an action is not legal."""
    x = torch.where(legal, x, float("-inf"))
    m = x.amax(1, keepdim=True)
    m = torch.where(legal.any(1, keepdim=True), m, 0.0)
    z = x - m
    return torch.where(legal, z - z.exp().sum(1, keepdim=True).log(), 0.0)


def _plain_sample(s):
    A = s["case"]["actions"]
    legal = _legal(s["mask"], A)
    x = torch.where(legal, s["logits"].double(), float("-inf"))  # next to a border of the distribution 32 bits lose it
    any_legal = legal.any(1)
    e = torch.where(legal, (x - torch.where(any_legal, x.amax(1), 0.0)[:, None]).exp(), 0.0)
    c = e.cumsum(1)
    a = (c > s["uniform"].double()[:, None] * c[:, -1:]).int().argmax(1)
    logp = _log_softmax(s["logits"].float(), legal).gather(1, a[:, None])[:, 0]
    return torch.where(any_legal, a, -1).to(torch.int8), torch.where(any_legal, logp, 0.0)


def _plain_advantages(s):
    c = s["case"]
    T, B, P = c["steps"], c["lanes"], c["players"]
    g, gl = c["gamma"], c["gamma"] * c["lam"]
    v, st, pl = s["values"].float(), s["step_type"], s["players"].long()
    seat = torch.arange(P, device=v.device)
    adv, target = torch.zeros_like(v), torch.zeros_like(v)
    z = g * s["bootstrap"].float()  # what a player's next decision is worth, discounted, with the rewards up to it
    for t in range(T - 1, -1, -1):
        step = (st[t] == 1) | (st[t] == 2)
        z = torch.where(((st[t] == 0) | (st[t] == 2))[:, None], 0.0, z)
        z = z + torch.where(step[:, None], s["rewards"][t].float(), 0.0)
        mine = step[:, None] & (pl[t][:, None] == seat)
        acted = mine.any(1)
        value = torch.where(acted, v[t], 0.0)
        a = torch.where(mine, z, 0.0).sum(1) - value
        adv[t] = torch.where(acted, a, 0.0)
        target[t] = torch.where(acted, a + value, 0.0)
        z = torch.where(mine, gl * z + ((g - gl) * value)[:, None], z)
    return adv, target


def _plain_policy(s):
    c = s["case"]
    A, rows = c["actions"], c["rows"]
    legal = _legal(s["mask"], A)
    real = _decided(legal, s["actions"])
    if s["active"] is not None:
        real = real & s["active"]
    a = torch.where(real, s["actions"].long(), 0)[:, None]
    n = real.sum().clamp(min=1).float()
    # the ratio in 64 bits: which side of the clip border it is on decides a whole gradient
    d = _log_softmax(s["logits"].double(), legal).gather(1, a)[:, 0] - torch.where(real, s["old"], 0.0).double()
    ratio = d.exp()
    adv = torch.where(real, s["adv"], 0.0)
    clipped = ((adv > 0) & (ratio > 1 + c["high"])) | ((adv < 0) & (ratio < 1 - c["low"]))
    ratio = ratio.float()
    surrogate = -torch.where(adv == 0, 0.0, torch.minimum(ratio * adv, ratio.clamp(1 - c["low"], 1 + c["high"]) * adv))
    logp = _log_softmax(s["logits"].float(), legal)
    p = torch.where(legal, logp.exp(), 0.0)
    entropy = -(p * logp).sum(1)
    diff = logp - _log_softmax(s["ref"].float(), legal) if s["ref"] is not None else torch.zeros_like(logp)
    kl = (p * diff).sum(1)
    mean = [torch.where(real, x, 0.0).double().sum().float() / n for x in (surrogate, kl, entropy, clipped.float())]
    loss = mean[0] + c["kl"] * mean[1] - c["entropy"] * mean[2]
    stats, count = torch.stack(mean), real.sum()
    taken = torch.where(real, logp.gather(1, a)[:, 0], 0.0)
    if c["grad"] == "none":
        return loss, stats, count, taken
    w = torch.where(clipped | (adv == 0), 0.0, -ratio * adv)[:, None]
    grad = w * (torch.zeros_like(p).scatter_(1, a, 1.0) - p)
    grad = grad + p * (c["kl"] * (diff - kl[:, None]) + c["entropy"] * (logp + entropy[:, None]))
    grad = torch.where(real[:, None] & legal, grad / n, 0.0).to(s["logits"].dtype)
    return loss, stats, count, taken, grad


def _plain_preference(s):
    c = s["case"]
    A, rows, pairs = c["actions"], c["rows"], c["pairs"]
    legal = _legal(s["mask"], A)
    real = _decided(legal, s["actions"])
    a = torch.where(real, s["actions"].long(), 0)[:, None]
    logp = _log_softmax(s["logits"].float(), legal)
    lr = logp.gather(1, a)[:, 0]
    if s["ref"] is not None:
        lr = lr - _log_softmax(s["ref"].float(), legal).gather(1, a)[:, 0]
    run_sum = torch.cat((torch.zeros(1, device=lr.device, dtype=torch.float64),
                         torch.where(real, lr, 0.0).double().cumsum(0)))
    off = s["offsets"].long()
    total = run_sum[off[1:]] - run_sum[off[:-1]]
    reward = c["beta"] * total
    x = reward[0::2] - reward[1::2]
    soft = lambda y: torch.clamp(-y, min=0) + torch.log1p(torch.exp(-y.abs()))  # noqa: E731  (-log sigmoid)
    eps = c["smoothing"]
    loss = ((1 - eps) * soft(x) + eps * soft(-x)).sum() / pairs
    if c["grad"] == "none":
        return loss.float(), reward.float()
    dx = eps - 1 + 1 / (1 + torch.exp(-x))
    coef = torch.stack((dx, -dx), 1).reshape(-1) * c["beta"] / pairs
    index = torch.arange(rows, device=off.device)
    seq = torch.searchsorted(off, index, right=True) - 1
    inside = (seq >= 0) & (seq < 2 * pairs)
    g = torch.where(inside & real, coef[seq.clamp(0, 2 * pairs - 1)], 0.0).float()[:, None]
    p = torch.where(legal, logp.exp(), 0.0)
    grad = g * (torch.zeros_like(p).scatter_(1, a, 1.0) - p)
    return loss.float(), reward.float(), torch.where(real[:, None] & legal, grad, 0.0).to(s["logits"].dtype)


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if not own:
        return {"sample": _plain_sample, "advantages": _plain_advantages, "policy": _plain_policy,
                "preference": _plain_preference}[case["op"]](state)
    from open_spiel_coup_amd import policy
    s = state
    if case["op"] == "sample":
        return policy.sample_actions(s["logits"], s["mask"], s["uniform"])
    if case["op"] == "advantages":
        return policy.advantages(s["rewards"], s["step_type"], s["players"], s["values"], s["bootstrap"],
                                 gamma=case["gamma"], lam=case["lam"])
    if case["op"] == "policy":
        rest = (s["actions"], s["mask"], s["old"], s["adv"])
        more = dict(ref_logits=s["ref"], active=s["active"], clip_low=case["low"], clip_high=case["high"],
                    kl_coef=case["kl"], entropy_coef=case["entropy"])
        loss, both = policy.policy_loss, policy.policy_loss_and_grad
    else:
        rest = (s["actions"], s["mask"], s["offsets"])
        more = dict(ref_logits=s["ref"], beta=case["beta"], label_smoothing=case["smoothing"])
        loss, both = policy.preference_loss, policy.preference_loss_and_grad
    if case["grad"] == "call":
        return both(s["logits"], *rest, **more)
    if case["grad"] == "none":
        return loss(s["logits"], *rest, **more)
    out = loss(s["train"], *rest, **more)
    grad, = torch.autograd.grad(out[0], s["train"])
    return (out[0].detach(), *out[1:], grad)


def work(case):
    if case["op"] == "advantages":
        cells = case["steps"] * case["lanes"]
        e, P = BYTES[case["dtype"]], case["players"]
        return {"bytes": cells * (P + 2 + e + 8) + case["lanes"] * P * e, "flops": cells * (P + 6)}
    rows, A, e = case["rows"], case["actions"], BYTES[case["dtype"]]
    if case["op"] == "sample":
        return {"bytes": rows * (A * e + 4 + 4 + 1 + 4), "flops": rows * A * 4}
    tables = 1 + case["ref"] + (case["grad"] != "none")
    if case["op"] == "policy":
        return {"bytes": rows * (tables * A * e + 1 + 4 + 4 + 4 + 4 + case["active"]) + 28, "flops": rows * A * 8 * tables}
    return {"bytes": rows * (tables * A * e + 1 + 4) + (2 * case["pairs"] + 1) * 4 + 8 * case["pairs"] + 4,
            "flops": rows * A * 6 * tables}


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _legal_table(mask, A):
    table = torch.zeros(mask.shape[0], A, dtype=torch.bool, device=mask.device)
    for a in range(A):
        table[:, a] = (mask.bitwise_and(1 << a) != 0) & (mask.bitwise_and(CHANCE) == 0)
    return table


def _taken(legal, actions):
    """(rows that are decisions, one-hot of their actions)"""
    hot = (torch.arange(legal.shape[1], device=legal.device) == actions.long()[:, None]) & legal
    return hot.any(1), hot


def _probabilities(x, legal):
    """softmax over the legal actions of every row that has one (elsewhere 0), differentiable in x."""
    shift = x.detach().masked_fill(~legal, -math.inf).amax(1, keepdim=True)
    e = (x - shift.masked_fill(~torch.isfinite(shift), 0.0)).masked_fill(~legal, -math.inf).exp()
    total = e.sum(1, keepdim=True)
    return e / total.masked_fill(total == 0, 1.0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "advantages":
        T, B, P = case["steps"], case["lanes"], case["players"]
        v = s["values"].double().nan_to_num(0.0)
        adv, target = torch.zeros_like(v), torch.zeros_like(v)
        for p in range(P):
            # player p's decisions, backwards: delta = rewards until its next one + gamma V(next) - V
            ahead = s["bootstrap"][:, p].double()
            carried, earned = torch.zeros_like(ahead), torch.zeros_like(ahead)
            for t in reversed(range(T)):
                kind = s["step_type"][t]
                over = (kind == 2) | (kind == 0)
                ahead, carried, earned = (x.masked_fill(over, 0.0) for x in (ahead, carried, earned))
                earned = earned + s["rewards"][t, :, p].double() * ((kind == 1) | (kind == 2))
                here = ((kind == 1) | (kind == 2)) & (s["players"][t] == p)
                delta = earned + case["gamma"] * ahead - v[t]
                value = delta + case["gamma"] * case["lam"] * carried
                adv[t] = torch.where(here, value, adv[t])
                target[t] = torch.where(here, value + v[t], target[t])
                ahead = torch.where(here, v[t], ahead)
                carried = torch.where(here, value, carried)
                earned = earned.masked_fill(here, 0.0)
        return adv, target
    A = case["actions"]
    legal = _legal_table(s["mask"], A)
    x = s["logits"].double().masked_fill(~legal, 0.0).requires_grad_()
    p = _probabilities(x, legal)
    if case["op"] == "sample":
        e = p.detach()
        some = legal.any(1)
        edge = torch.zeros_like(s["uniform"], dtype=torch.float64)
        action = torch.full_like(edge, -1.0)
        for a in range(A):
            edge = edge + e[:, a]
            action = torch.where((action < 0) & legal[:, a] & (edge > s["uniform"].double()), float(a), action)
        final = A - 1 - (e > 0).flip(1).int().argmax(1)  # rounding left the whole below the number: the last one
        action = torch.where(some & (action < 0), final.double(), action).long()
        logp = e.gather(1, action.clamp(0)[:, None])[:, 0].log()
        return action.to(torch.int8), torch.where(some, logp, 0.0)
    real, hot = _taken(legal, s["actions"])
    if case["op"] == "policy" and s["active"] is not None:
        real = real & s["active"]
    logs = p.masked_fill(p.detach() == 0, 1.0).log()
    taken = (logs * hot).sum(1)
    q_logs = torch.zeros_like(logs)
    if s["ref"] is not None:
        q = _probabilities(s["ref"].double().masked_fill(~legal, 0.0), legal)
        q_logs = q.masked_fill(q == 0, 1.0).log()
    if case["op"] == "policy":
        count = max(1, int(real.sum()))
        ratio = (taken - s["old"].double().masked_fill(~real, 0.0)).exp()
        adv = s["adv"].double().masked_fill(~real, 0.0)
        low, high = 1 - case["low"], 1 + case["high"]
        capped = ((adv > 0) & (ratio.detach() > high)) | ((adv < 0) & (ratio.detach() < low))
        bound = torch.where(adv > 0, high, low)
        gain = torch.where(capped, bound, ratio) * adv
        kl = (p * (logs - q_logs)).sum(1) if s["ref"] is not None else torch.zeros_like(gain)
        spread = -(p * logs).sum(1)
        mean = [(t.double() * real).sum() / count for t in (-gain, kl, spread, capped)]
        loss = mean[0] + case["kl"] * mean[1] - case["entropy"] * mean[2]
        info = (torch.stack([m.detach() for m in mean]), real.sum(), taken.detach() * real)
    else:
        score = ((taken - (q_logs * hot).sum(1)) * real)
        off = s["offsets"].long()
        lens = off[1:] - off[:-1]
        owner = torch.repeat_interleave(torch.arange(lens.numel(), device=off.device), lens)
        total = torch.zeros(lens.numel(), dtype=torch.float64, device=off.device)
        total = total.index_add(0, owner, score[int(off[0]):int(off[-1])])
        reward = case["beta"] * total
        margin = reward[0::2] - reward[1::2]
        zero = torch.zeros_like(margin)
        loss = ((1 - case["smoothing"]) * torch.logaddexp(zero, -margin)
                + case["smoothing"] * torch.logaddexp(zero, margin)).mean()
        info = (reward.detach(),)
    if case["grad"] == "none":
        return (loss.detach(), *info)
    grad, = torch.autograd.grad(loss, x)
    return (loss.detach(), *info, grad)
