"""Plain float64 forms of the long-history policy operators (layer norm, relative position bias, grouped-query
attention, the clipped policy loss), written from their definitions on CPU tensors, and the tolerances they are held to.

Tolerances. u is the unit roundoff of a type (half a step: fp32 2^-24, bf16 2^-8, relative to the value). An fp32 result that
is a sum of n terms in a tree or chain, of magnitude sum m, is off by at most about (depth) u m; the bounds below use the
probabilistic constant 32 for m (chains of up to 1000 terms) beside 8 u of the value. A bf16 result adds its own rounding,
2^-8 of the value, once per rounding that its path makes.
"""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8


def close(got, ref, mag, rounds=0, name="", k=32.0):
    """|got - ref| <= rounds 2^-8 |ref| + k 2^-24 mag + 8 2^-24 |ref| (rounds: bf16 roundings of the value)."""
    got, ref, mag = (torch.as_tensor(t, dtype=torch.float64) for t in (got, ref, mag))
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)} against {tuple(ref.shape)}"
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), f"{name}: infinities differ"
    err = (got - ref).abs()
    bound = (rounds * U16 + 8 * U32) * ref.abs() + k * U32 * mag + 1e-37
    bad = fin & ~(err <= bound)
    if bad.any():
        i = int(torch.argmax(torch.where(fin, err / bound, torch.zeros_like(err))))
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} out of bounds; worst at {i}: got "
                             f"{got.reshape(-1)[i]:.9g} ref {ref.reshape(-1)[i]:.9g} err {err.reshape(-1)[i]:.3g} "
                             f"bound {bound.expand_as(err).reshape(-1)[i]:.3g}")


def layernorm(x, w, b, dy, eps):
    """y, mean, rstd, dx, dw, db."""
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    h = dy * w
    dx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    return xh * w + b, mean[:, 0], rstd[:, 0], dx, (dy * xh).sum(0), dy.sum(0)


def bucket(d, buckets, max_distance, both):
    """The bucket of distance d by whole-number comparisons: n >= E (M / E)^(t / L) as n^L E^t >= M^t E^L."""
    side = buckets // 2 if both else buckets
    n, few = (abs(d) if both else max(0, -d)), side // 2
    b = n
    if n >= few:
        steps, t = side - few, 0
        if n >= max_distance:
            t = steps - 1
        else:
            while t < steps - 1 and n ** steps * few ** (t + 1) >= max_distance ** (t + 1) * few ** steps:
                t += 1
        b = few + t
    return b + (side if both and d > 0 else 0)


def policy_loss(x, actions, adv, old, ref, weight, low, high, kl_coef):
    """loss, logp, dlogits and the five statistics; ref and weight may be None."""
    rows, vocab = x.shape
    w = torch.full((rows,), 1.0 / rows, dtype=torch.float64) if weight is None else weight
    loss, stats = 0.0, [0.0] * 5
    logps, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros_like(x)
    for t in range(rows):
        if w[t] == 0:
            continue
        a = int(actions[t])
        if a < 0 or a >= vocab:
            loss, logps[t] = math.nan, math.nan
            stats = [math.nan, math.nan, math.nan if ref is not None else stats[2], stats[3], stats[4] + 1]
            continue
        lp = torch.log_softmax(x[t], 0)
        diff = float(lp[a] - old[t])
        ratio = math.exp(diff)
        plain, held = ratio * float(adv[t]), min(max(ratio, 1 - low), 1 + high) * float(adv[t])
        gain = min(plain, held)
        clipped = ratio > 1 + high if adv[t] >= 0 else ratio < 1 - low
        kl = dkl = 0.0
        if ref is not None:
            gap = float(ref[t] - lp[a])
            kl, dkl = math.exp(gap) - gap - 1, 1 - math.exp(gap)
        loss += float(w[t]) * (kl_coef * kl - gain)
        slope = float(w[t]) * (kl_coef * dkl - (0.0 if clipped else plain))
        grad[t] = -slope * lp.exp()
        grad[t, a] += slope
        logps[t] = lp[a]
        stats = [s + v for s, v in zip(stats, (ratio - 1 - diff, gain, kl, float(clipped), 1.0))]
    return loss, logps, grad, stats
