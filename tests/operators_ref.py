"""Plain float64 forms of the long-history policy operators (layer norm, relative position bias, grouped-query
attention, the clipped policy loss), written from their definitions on CPU tensors, and the tolerances they are held to.

Tolerances. u is the unit roundoff of a type (half a step: fp32 2^-24, bf16 2^-8, relative to the value). An fp32 result that
is a sum of n terms in a tree or chain, of magnitude sum m, is off by at most about (depth) u m; the bounds below use the
probabilistic constant 32 for m (chains of up to 1000 terms) beside 8 u of the value. A bf16 result adds its own rounding,
2^-8 of the value, once per rounding that its path makes.
"""
import math

import pytest
import torch


@pytest.fixture(autouse=True)
def float32_default():
    """The sizes of the buffers made here do not depend on the default that another test module set."""
    kept = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(kept)


U32, U16 = 2.0 ** -24, 2.0 ** -8


def close(got, ref, mag, rounds=0, name="", k=32.0, tiny=8.0):
    """|got - ref| <= rounds 2^-8 |ref| + k 2^-24 mag + 8 2^-24 |ref| + 2^-126 tiny (rounds: bf16 roundings of the value;
    tiny: the sum of its terms' magnitudes were every factor that may underflow one)."""
    got, ref, mag, tiny = (torch.as_tensor(t, dtype=torch.float64) for t in (got, ref, mag, tiny))
    assert got.shape == ref.shape, f"{name}: {tuple(got.shape)} against {tuple(ref.shape)}"
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), f"{name}: infinities differ"
    err = (got - ref).abs()
    bound = (rounds * U16 + 8 * U32) * ref.abs() + k * U32 * mag + 2.0 ** -126 * tiny
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


def attention(q, k, v, scale, causal, qlens, klens, bias=None, do=None):
    """Grouped-query attention of [B, S, heads, d] tensors and its gradients, with what the tolerances need.

    Returns a dict: o, lse (and dq, dk, dv, dbias with do), each beside its magnitudes: "<name>.f", the sum of the
    magnitudes of its fp32 terms times one plus that of the scores (an error e of a score changes its probability by the
    share e), and "<name>.h", the sum of the magnitudes of the terms that bf16 kernels round to bf16 (probabilities, their
    gradients, and o inside D = rowsum(do o)), and "<name>.u", the sum of the terms' magnitudes with every probability one
    (a probability below 2^-126, the least normal fp32 number, is taken for zero)."""
    B, Sq, H, _ = q.shape
    Sk, KV, dv = k.shape[1], k.shape[2], v.shape[3]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    r = {"o": z(B, Sq, H, dv), "lse": torch.full((B, H, Sq), -math.inf, dtype=torch.float64)}
    shapes = {"o": (B, Sq, H, dv), "lse": (B, H, Sq)}
    if do is not None:
        shapes.update(dq=tuple(q.shape), dk=tuple(k.shape), dv=tuple(v.shape))
        if bias is not None:
            shapes["dbias"] = tuple(bias.shape)
        r.update({n: z(*s) for n, s in shapes.items() if n not in r})
    r.update({n + e: z(*s) for n, s in shapes.items() for e in (".f", ".h", ".u")})
    for b in range(B):
        ql = Sq if qlens is None else min(max(int(qlens[b]), 0), Sq)
        kl = Sk if klens is None else min(max(int(klens[b]), 0), Sk)
        if ql == 0 or kl == 0:
            continue
        apart = torch.arange(kl)[None, :] - (torch.arange(ql)[:, None] + kl - ql)
        for h in range(H):
            g = h // (H // KV)
            Q, K, V = q[b, :ql, h], k[b, :kl, g], v[b, :kl, g]
            s, sm = scale * Q @ K.t(), scale * Q.abs() @ K.abs().t()
            if bias is not None:
                M = bias.shape[1] // 2
                at = apart.clamp(-M, M) + M
                hidden = bias[h][at] < -3.4e30  # such entries hide the keys at their distance
                near = torch.where(hidden, 0.0, bias[h][at])
                s, sm = s + near, sm + near.abs()
            see = apart <= 0 if causal else torch.ones_like(apart, dtype=torch.bool)
            if bias is not None:
                see = see & ~hidden
            some = see.any(1)
            s = s.masked_fill(~see, -math.inf)
            top = torch.where(some, s.max(1).values, 0.0)
            e = torch.exp(s - top[:, None])
            zsum = e.sum(1)
            p = e / torch.where(some, zsum, 1.0)[:, None]
            lse = torch.where(some, top + torch.log(zsum), torch.tensor(-math.inf, dtype=torch.float64))
            w = 1 + torch.where(see, sm, 0.0).max(1).values + torch.where(some, lse.abs(), 0.0)  # of a row's scores
            O = p @ V
            pv = p @ V.abs()
            r["o"][b, :ql, h], r["lse"][b, h, :ql] = O, lse
            r["o.f"][b, :ql, h], r["o.h"][b, :ql, h] = pv * w[:, None], pv
            r["lse.f"][b, h, :ql] = w
            one = see.double()
            r["o.u"][b, :ql, h] = one @ V.abs()
            if do is None:
                continue
            G = do[b, :ql, h]
            D = (G * O).sum(1, keepdim=True)
            Dh = (G.abs() * (pv + O.abs())).sum(1, keepdim=True)  # what a rounded o puts into D
            ds = p * (G @ V.t() - D)
            dsf = p * (G.abs() @ V.abs().t() + Dh) * w[:, None]
            dsh = ds.abs() + p * Dh
            r["dq"][b, :ql, h] = scale * ds @ K
            r["dq.f"][b, :ql, h], r["dq.h"][b, :ql, h] = scale * dsf @ K.abs(), scale * dsh @ K.abs()
            r["dk"][b, :kl, g] += scale * ds.t() @ Q
            r["dk.f"][b, :kl, g] += scale * dsf.t() @ Q.abs()
            r["dk.h"][b, :kl, g] += scale * dsh.t() @ Q.abs()
            r["dv"][b, :kl, g] += p.t() @ G
            r["dv.f"][b, :kl, g] += (p * w[:, None]).t() @ G.abs()
            r["dv.h"][b, :kl, g] += p.t() @ G.abs()
            dsu = one * (G.abs() @ V.abs().t() + Dh)
            r["dq.u"][b, :ql, h] = scale * dsu @ K.abs()
            r["dk.u"][b, :kl, g] += scale * dsu.t() @ Q.abs()
            r["dv.u"][b, :kl, g] += one.t() @ G.abs()
            if bias is not None:
                r["dbias.u"][h].index_add_(0, at.reshape(-1), dsu.reshape(-1))
                for n, t in (("dbias", ds), ("dbias.f", dsf), ("dbias.h", p * Dh)):
                    r[n][h].index_add_(0, at.reshape(-1), t.reshape(-1))
    return r


def close_attention(got, r, ty, names):
    """fp32: 32 u of the terms; bf16 also half a step of the result and of each rounded term (o's rounding inside D alone
    for dbias, whose terms are not rounded)."""
    for n in names:
        h = r[n + ".h"] if ty == "bf16" else torch.zeros(())
        mag = r[n + ".f"] + h * (U16 / (32 * U32))
        close(got[n], r[n], mag, 1 if ty == "bf16" and n not in ("lse", "dbias") else 0, n, tiny=r[n + ".u"] + 8)
