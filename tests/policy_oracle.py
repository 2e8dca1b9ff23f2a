"""The learner-side operators (open_spiel_coup_amd.policy) from their
definitions, in numpy float64, one row / one lane / one pair at a time: the
oracle of tests/test_gpu_policy.py.  Nothing here uses the package."""
import math

import numpy as np


def legal_actions(word, A):
    """Legal actions of a mask word, ascending; none at a chance node (bit 31)."""
    word = int(word) & 0xFFFFFFFF
    return [] if word >> 31 else [a for a in range(A) if (word >> a) & 1]


def log_softmax(row, legal):
    """{action: log probability} over the legal actions (NaN where undefined)."""
    x = [float(row[a]) for a in legal]
    if any(math.isnan(v) or v == math.inf for v in x) or all(v == -math.inf for v in x):
        return {a: math.nan for a in legal}
    m = max(x)
    total = math.fsum(math.exp(v - m) for v in x)
    rest = math.fsum(math.exp(v - m) for v in x) - 1.0
    lse = math.log1p(rest) if rest < 0.5 else math.log(total)
    return {a: (v - m) - lse for a, v in zip(legal, x)}


def sample(logits, mask, uniform):
    """(actions, log_probs)"""
    n, A = logits.shape
    actions, logp = np.full(n, -1, np.int8), np.zeros(n)
    for i in range(n):
        legal = legal_actions(mask[i], A)
        if not legal:
            continue
        lp = log_softmax(logits[i], legal)
        if math.isnan(lp[legal[0]]):
            logp[i] = math.nan
            continue
        m = max(float(logits[i][a]) for a in legal)
        e = [math.exp(float(logits[i][a]) - m) for a in legal]
        total = 0.0
        for v in e:
            total += v
        run, pick = 0.0, None
        for a, v in zip(legal, e):
            run += v
            if run > float(uniform[i]) * total:
                pick = a
                break
        if pick is None:
            pick = [a for a, v in zip(legal, e) if v > 0][-1]
        actions[i], logp[i] = pick, lp[pick]
    return actions, logp


def advantages(rewards, step_type, players, values, bootstrap, gamma, lam):
    """(advantages, targets): each player's decisions of each lane, forwards."""
    T, B, P = rewards.shape
    adv, target = np.zeros((T, B)), np.zeros((T, B))
    for b in range(B):
        for p in range(P):
            mine = [t for t in range(T) if step_type[t, b] in (1, 2) and players[t, b] == p]
            carried = 0.0
            for k in range(len(mine) - 1, -1, -1):
                t = mine[k]
                end = mine[k + 1] if k + 1 < len(mine) else T
                gain, ahead, linked = 0.0, None, True
                for s in range(t, end):
                    if s > t and step_type[s, b] == 0:  # the game was restarted: nothing behind it counts
                        linked = False
                        break
                    if step_type[s, b] in (1, 2):
                        gain += float(rewards[s, b, p])
                    if step_type[s, b] == 2:
                        linked = False
                        break
                if linked:
                    if end < T:
                        ahead = float(values[end, b])
                    else:
                        ahead = 0.0 if bootstrap is None else float(bootstrap[b, p])
                v = float(values[t, b])
                delta = gain + (gamma * ahead if linked else 0.0) - v
                carried = delta + (gamma * lam * carried if linked and end < T else 0.0)
                adv[t, b], target[t, b] = carried, carried + v
    return adv, target


def policy(logits, actions, mask, old, adv, ref, active, low, high, kl, ent):
    """dict: loss, stats [4], count, log_probs, grad, and for tolerances the
    size of every gradient entry's terms (`size`) and of the loss's (`mass`)."""
    n, A = logits.shape
    logp_out, grad, size = np.zeros(n), np.zeros((n, A)), np.zeros((n, A))
    terms, rows = [], []
    for i in range(n):
        legal = legal_actions(mask[i], A)
        a = int(actions[i])
        if a not in legal or (active is not None and not active[i]):
            continue
        l = log_softmax(logits[i], legal)
        p = {b: math.exp(l[b]) for b in legal}
        d = {b: 0.0 for b in legal}
        if ref is not None:
            lr = log_softmax(ref[i], legal)
            d = {b: l[b] - lr[b] if p[b] > 0 else 0.0 for b in legal}
        H = -sum(p[b] * l[b] for b in legal if p[b] > 0)
        K = sum(p[b] * d[b] for b in legal)
        Z = float(adv[i])
        dl = l[a] - float(old[i])
        over = (Z > 0 and dl > math.log1p(high)) or (Z < 0 and low < 1 and dl < math.log1p(-low))
        rho = math.exp(min(dl, 700.0))
        held = (1 + high) if Z > 0 else (1 - low)
        s = 0.0 if Z == 0 else -(held if over else rho) * Z
        w = 0.0 if over or Z == 0 else -rho * Z
        logp_out[i] = l[a]
        terms.append((s, K, H, float(over)))
        rows.append(i)
        for b in legal:
            g = w * ((b == a) - p[b])
            m = abs(w) * ((b == a) + p[b])
            if p[b] > 0:
                g += p[b] * (kl * (d[b] - K) + ent * (l[b] + H))
                m += p[b] * (abs(kl) * (abs(d[b]) + abs(K)) + abs(ent) * (abs(l[b]) + H))
            grad[i, b], size[i, b] = g, m
    c = max(1, len(rows))
    t = np.array(terms).reshape(-1, 4)
    stats = t.sum(0) / c
    loss = stats[0] + kl * stats[1] - ent * stats[2]
    mass = np.abs(t).sum(0) / c
    return dict(loss=loss, stats=stats, count=len(rows), log_probs=logp_out, grad=grad / c, size=size / c, mass=mass)


def neg_log_sigmoid(x):
    return math.log1p(math.exp(-abs(x))) + max(-x, 0.0)


def preference(logits, actions, mask, offsets, ref, beta, eps):
    """dict: loss, rewards, grad, and for tolerances `size` as above and each
    sequence's decisions (`length`)."""
    n, A = logits.shape
    S = len(offsets) - 1
    rewards, grad, size = np.zeros(S), np.zeros((n, A)), np.zeros((n, A))
    lps, length = {}, np.zeros(S, int)
    for s in range(S):
        for i in range(int(offsets[s]), int(offsets[s + 1])):
            legal = legal_actions(mask[i], A)
            a = int(actions[i])
            if a not in legal:
                continue
            lps[i] = (s, a, log_softmax(logits[i], legal))
            rewards[s] += lps[i][2][a] - (log_softmax(ref[i], legal)[a] if ref is not None else 0.0)
            length[s] += 1
    rewards *= beta
    pairs = S // 2
    cost, coef = 0.0, np.zeros(S)
    for k in range(pairs):
        x = rewards[2 * k] - rewards[2 * k + 1]
        cost += (1 - eps) * neg_log_sigmoid(x) + eps * neg_log_sigmoid(-x)
        down = 1 / (1 + math.exp(x)) if x < 700 else 0.0
        coef[2 * k] = (eps - down) * beta / pairs
        coef[2 * k + 1] = -coef[2 * k]
    for i, (s, a, l) in lps.items():
        for b in l:
            grad[i, b] = coef[s] * ((b == a) - math.exp(l[b]))
            size[i, b] = abs(coef[s]) * ((b == a) + math.exp(l[b]))
    return dict(loss=cost / max(1, pairs), rewards=rewards, grad=grad, size=size, length=length)
