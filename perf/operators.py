"""What the operators of a policy over long histories are measured on: one training or decoding pass each, in the
plain form (torch, 32 bits, written from the formulas) or through the C ABI (include/talos_hip.h).

Kinds of case, each with the sizes it is used at:

* norm   -- layer norm, forward and backward (talos_layernorm_fwd_*, _bwd_*): y, the row statistics, dx, dw, db.
* attn   -- grouped-query attention (talos_gqa_fwd_*, _bwd_*): any length, per-sample query and key lengths, causal or
            not; forward alone (decoding a token or a chunk against a long context) or with the backward pass, which
            recomputes the probabilities.
* relpos -- the same attention with a learned relative position bias by buckets: the table expanded to a bias by
            distance (talos_relpos_bias_fwd_f32), attention forward and backward, and the table's gradient
            (talos_relpos_bias_bwd_f32).
* loss   -- the clipped policy loss with a KL term over wide rows of logits and its gradient
            (talos_policy_loss_bwd_*): loss, the rows' log-probabilities, dlogits.

Queries and keys of a sample end together: query i of a sample of q_len queries and k_len keys stands at position
i + k_len - q_len, causal attention lets it see keys j <= that, and the bias goes by j minus that position. Rows past a
sample's length are padding; their outputs are zero (log-sum-exp: -inf).
"""
import math

import torch
import torch.nn.functional as F

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-5
_CLIP_LOW, _CLIP_HIGH, _KL = 0.2, 0.28, 0.04


def listed():
    return [
        # the reference policy's width over a replay batch: launch latency is all of it
        {"name": "norm_256x64", "kind": "norm", "rows": 256, "dim": 64, "type": "f32"},
        # every token of the headline minibatch (4096 samples of 32 tokens, d 128)
        {"name": "norm_131072x128", "kind": "norm", "rows": 131072, "dim": 128, "type": "f32"},
        # a wide model's activations over a batch of tokens
        {"name": "norm_8192x4096_bf16", "kind": "norm", "rows": 8192, "dim": 4096, "type": "bf16"},
        # a few environments, one new token each, against a short context: latency
        {"name": "decode_4x1x512", "kind": "attn", "B": 4, "Sq": 1, "Sk": 512, "H": 8, "KV": 8, "dk": 64, "dv": 64,
         "causal": 1, "ragged": 0, "grad": 0, "type": "f32"},
        # a full set of requests, one token each, against long contexts of different lengths
        {"name": "decode_64x1x4096_bf16", "kind": "attn", "B": 64, "Sq": 1, "Sk": 4096, "H": 32, "KV": 8, "dk": 128,
         "dv": 128, "causal": 1, "ragged": 1, "grad": 0, "type": "bf16"},
        # training over histories longer than the 256 tokens of the block kernels, right-padded, no round length
        {"name": "train_8x1000_ragged", "kind": "attn", "B": 8, "Sq": 1000, "Sk": 1000, "H": 8, "KV": 8, "dk": 64,
         "dv": 64, "causal": 1, "ragged": 1, "grad": 1, "type": "f32"},
        # training at a long context, grouped heads
        {"name": "train_4x4096_16kv4_bf16", "kind": "attn", "B": 4, "Sq": 4096, "Sk": 4096, "H": 16, "KV": 4,
         "dk": 128, "dv": 128, "causal": 1, "ragged": 0, "grad": 1, "type": "bf16"},
        # the d 128 policy's heads over ragged histories of an odd length, causal bias
        {"name": "relpos_16x333_ragged", "kind": "relpos", "B": 16, "Sq": 333, "Sk": 333, "H": 4, "KV": 4, "dk": 32,
         "dv": 32, "causal": 1, "ragged": 1, "grad": 1, "type": "f32", "buckets": 32, "max_distance": 128},
        # an encoder's layer: both directions, whole sequences
        {"name": "relpos_2x2048_bf16", "kind": "relpos", "B": 2, "Sq": 2048, "Sk": 2048, "H": 16, "KV": 16, "dk": 64,
         "dv": 64, "causal": 0, "ragged": 0, "grad": 1, "type": "bf16", "buckets": 32, "max_distance": 128},
        # the reference's five actions over the headline minibatch
        {"name": "loss_4096x5", "kind": "loss", "rows": 4096, "vocab": 5, "type": "f32"},
        # a wide action set of no round number, fp32 logits
        {"name": "loss_1021x50021", "kind": "loss", "rows": 1021, "vocab": 50021, "type": "f32"},
        # a batch of tokens over a vocabulary
        {"name": "loss_4096x32768_bf16", "kind": "loss", "rows": 4096, "vocab": 32768, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "attn", "attn", "attn", "relpos", "relpos", "loss", "loss"])
    kind_type = rng.choice(["f32", "bf16"])
    if kind == "norm":
        dim = _log_int(rng, 16, 8192)
        return {"kind": kind, "rows": min(_log_int(rng, 64, 131072), (1 << 25) // dim), "dim": dim, "type": kind_type}
    if kind == "loss":
        vocab = _log_int(rng, 2, 65536)
        return {"kind": kind, "rows": min(_log_int(rng, 16, 8192), (1 << 27) // vocab), "vocab": vocab,
                "type": kind_type}
    dk, dv = rng.choice([(32, 32), (64, 64), (64, 64), (80, 80), (96, 64), (128, 128), (128, 128), (40, 56)])
    H, KV = rng.choice([(4, 4), (8, 8), (16, 16), (8, 2), (16, 4), (6, 2), (8, 1)])
    c = {"kind": kind, "H": H, "KV": KV, "dk": dk, "dv": dv, "causal": rng.randint(0, 1), "ragged": rng.randint(0, 1),
         "grad": 1, "type": kind_type}
    decode = kind == "attn" and rng.random() < 0.4
    if decode:
        c["Sq"] = rng.choice([1, 1, 1, rng.randint(2, 16), rng.randint(17, 200)])
        c["Sk"] = _log_int(rng, max(64, c["Sq"]), 8192)
        c["causal"], c["grad"] = 1, 0
        c["B"] = max(1, min(_log_int(rng, 1, 64), (1 << 18) // c["Sk"]))
    else:
        c["Sq"] = c["Sk"] = _log_int(rng, 16, 4096)
        if rng.random() < 0.25:
            c["Sk"] = _log_int(rng, 16, 4096)  # queries of one sequence on the keys of another
        c["B"] = max(1, min(_log_int(rng, 1, 64), 32768 // c["Sq"], (1 << 28) // (H * c["Sq"] * c["Sk"])))
    if kind == "relpos":
        c["buckets"] = rng.choice([8, 16, 32, 64])
        c["max_distance"] = c["buckets"] * rng.choice([2, 4, 8])
    return c


# ---------------------------------------------------------------------------------------------------------
# Inputs (made on the GPU from the seed; the same tensors for run and exact)
# ---------------------------------------------------------------------------------------------------------

class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1000003 * (seed + 1))

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def spread(self, lo, hi, n):
        """n lengths spread evenly over lo..hi, in a random order."""
        v = torch.linspace(lo, hi, n, device="cuda", dtype=torch.float64).round().to(torch.int32)
        return v[torch.randperm(n, generator=self.g, device="cuda")]


def _lengths(case):
    """(lowest query length, lowest key length) of a ragged case; the highest are Sq and Sk."""
    return (1, 1) if case["Sq"] == case["Sk"] else (max(1, case["Sq"] // 2), 1)


def _inputs(case, seed):
    g, dt = _Draws(seed), _DTYPES[case["type"]]
    if case["kind"] == "norm":
        R, D = case["rows"], case["dim"]
        x = g.normal(R, D) * g.uniform(0.5, 2.0, R, 1) + g.normal(R, 1, std=0.5)  # a residual stream's rows differ
        return {"x": x.to(dt), "w": g.uniform(0.9, 1.1, D), "b": g.normal(D, std=0.1), "dy": g.normal(R, D).to(dt)}
    if case["kind"] == "loss":
        R, V = case["rows"], case["vocab"]
        logits = g.normal(R, V, std=2.0).to(dt)
        actions = torch.randint(0, V, (R,), generator=g.g, device="cuda", dtype=torch.int32)
        # half of the rows take a likely action, as sampling does
        actions = torch.where(g.uniform(0, 1, R) < 0.5, logits.argmax(-1).int(), actions)
        logp = torch.log_softmax(logits.float(), -1).gather(1, actions.long()[:, None])[:, 0]
        # the rollout's policy and the reference policy, somewhat apart from this one; an eighth of the rows is padding
        weight = (g.uniform(0, 1, R) < 0.875).float()
        return {"logits": logits, "actions": actions, "adv": g.normal(R), "old": logp + g.normal(R, std=0.3),
                "ref": logp + g.normal(R, std=0.3), "weight": weight / R}
    B, Sq, Sk, H, KV, dk, dv = (case[k] for k in ("B", "Sq", "Sk", "H", "KV", "dk", "dv"))
    i = {"q": g.normal(B, Sq, H, dk).to(dt), "k": g.normal(B, Sk, KV, dk).to(dt), "v": g.normal(B, Sk, KV, dv).to(dt)}
    if case["grad"]:
        i["do"] = g.normal(B, Sq, H, dv).to(dt)
    i["qlen"] = i["klen"] = None
    if case["ragged"]:
        lq, lk = _lengths(case)
        i["klen"] = g.spread(lk, Sk, B)
        i["qlen"] = i["klen"] if Sq == Sk else g.spread(lq, Sq, B)
    if case["kind"] == "relpos":
        i["table"] = g.normal(case["buckets"], H, std=0.5)
    return i


def prepare(case, seed):
    i, c = _inputs(case, seed), case
    new = lambda *shape, dtype=torch.float32: torch.empty(*shape, device="cuda", dtype=dtype)  # noqa: E731
    if c["kind"] == "norm":
        o = {"y": torch.empty_like(i["x"]), "mean": new(c["rows"]), "rstd": new(c["rows"]),
             "dx": torch.empty_like(i["x"]), "dw": new(c["dim"]), "db": new(c["dim"])}
    elif c["kind"] == "loss":
        o = {"loss": new(1), "logp": new(c["rows"]), "dlogits": torch.empty_like(i["logits"])}
    else:
        o = {"o": new(c["B"], c["Sq"], c["H"], c["dv"], dtype=i["q"].dtype), "lse": new(c["B"], c["H"], c["Sq"])}
        if c["kind"] == "relpos":
            n = 2 * c["max_distance"] + 1
            o.update(bias=new(c["H"], n), buckets=new(n, dtype=torch.int32))
        if c["grad"]:
            o.update(dq=torch.empty_like(i["q"]), dk=torch.empty_like(i["k"]), dv=torch.empty_like(i["v"]))
            if c["kind"] == "relpos":
                o.update(dbias=torch.empty_like(o["bias"]), dtable=torch.empty_like(i["table"]))
    return {"case": dict(case), "in": i, "out": o}


# ---------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------

def _plain_norm(c, i):
    x, dy, w = i["x"].float(), i["dy"].float(), i["w"]
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + _EPS)
    xh = xc * rstd
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return {"y": (xh * w + i["b"]).to(i["x"].dtype), "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(i["x"].dtype),
            "dw": (dy * xh).sum(0, dtype=torch.float64).float(), "db": dy.sum(0, dtype=torch.float64).float()}


def _plain_loss(c, i):
    x = i["logits"].float()
    a = i["actions"].long()[:, None]
    top = x.max(-1, keepdim=True).values
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True, dtype=torch.float64)
    logp = (x.gather(1, a).double() - top.double() - torch.log(z))[:, 0]
    adv, w = i["adv"].double(), i["weight"].double()
    ratio = torch.exp(logp - i["old"].double())
    clipped = ratio.clamp(1.0 - _CLIP_LOW, 1.0 + _CLIP_HIGH)
    gap = i["ref"].double() - logp
    row = -torch.minimum(ratio * adv, clipped * adv) + _KL * (torch.exp(gap) - gap - 1.0)
    live = torch.where(adv >= 0, ratio <= 1.0 + _CLIP_HIGH, ratio >= 1.0 - _CLIP_LOW)
    slope = torch.where(live, -adv * ratio, torch.zeros_like(adv)) + _KL * (1.0 - torch.exp(gap))
    slope = torch.where(w != 0, w * slope, torch.zeros_like(w))
    d = e * (-slope[:, None] / z).float()
    d.scatter_add_(1, a, slope.float()[:, None])
    loss = torch.where(w != 0, w * row, torch.zeros_like(w)).sum().float()[None]
    return {"loss": loss, "logp": torch.where(w != 0, logp, torch.zeros_like(w)).float(),
            "dlogits": d.to(i["logits"].dtype)}


def _plain_buckets(c):
    """Bucket of the distances -M .. M (key minus query): exact ones up to half a side's buckets, then by logarithm."""
    d = torch.arange(-c["max_distance"], c["max_distance"] + 1, device="cuda")
    both = not c["causal"]
    side = c["buckets"] // 2 if both else c["buckets"]
    n = d.abs() if both else (-d).clamp(min=0)
    few = side // 2
    step = torch.log(n.clamp(min=1).double() / few) / math.log(c["max_distance"] / few) * (side - few)
    far = (few + torch.floor(step + 1e-9).long()).clamp(max=side - 1)
    return (torch.where(n < few, n, far) + (side * (d > 0) if both else 0)).int()


def _plain_attn(c, i):
    B, Sq, Sk, H, KV, dk, dv = (c[k] for k in ("B", "Sq", "Sk", "H", "KV", "dk", "dv"))
    G, scale, dev = H // KV, 1.0 / math.sqrt(dk), i["q"].device
    full = lambda n: torch.full((B,), n, device=dev)  # noqa: E731
    ql = full(Sq) if i["qlen"] is None else i["qlen"].long()
    kl = full(Sk) if i["klen"] is None else i["klen"].long()
    rows, cols = torch.arange(Sq, device=dev), torch.arange(Sk, device=dev)
    # [B, KV, G * S, d]: the heads of a group are rows over their shared keys
    split = lambda t: t.float().reshape(B, Sq, KV, G, -1).permute(0, 2, 3, 1, 4).reshape(B, KV, G * Sq, -1)  # noqa: E731
    join = lambda t: t.reshape(B, H, Sq, -1).permute(0, 2, 1, 3).to(i["q"].dtype)  # noqa: E731
    shared = lambda t: torch.where((cols < kl[:, None])[:, :, None, None], t.float(), 0.0).permute(0, 2, 1, 3)  # noqa: E731
    q, k, v = split(i["q"]), shared(i["k"]), shared(i["v"])
    s = (torch.matmul(q, k.transpose(-1, -2)) * scale).reshape(B, H, Sq, Sk)
    delta = cols[None, None, :] - (rows[None, :] + (kl - ql)[:, None])[:, :, None]  # [B, Sq, Sk]
    see = (rows < ql[:, None])[:, :, None] & (cols < kl[:, None])[:, None, :]
    if c["causal"]:
        see = see & (delta <= 0)
    out = {}
    if c["kind"] == "relpos":
        M = c["max_distance"]
        out["buckets"] = _plain_buckets(c)
        out["bias"] = i["table"][out["buckets"].long()].t().contiguous()
        s = s + out["bias"][:, delta.clamp(-M, M) + M].transpose(0, 1)
    s = s.masked_fill(~see[:, None], -math.inf)
    top = s.max(-1, keepdim=True).values
    p = torch.exp(s - top.clamp(min=-1e38))
    del s
    z = p.sum(-1, keepdim=True)
    p /= torch.where(z > 0, z, 1.0)
    p = p.reshape(B, KV, G * Sq, Sk)
    o = torch.matmul(p, v)
    out["lse"] = (top + torch.log(z)).reshape(B, H, Sq)
    out["o"] = join(o)
    if not c["grad"]:
        return out
    do = split(torch.where((rows < ql[:, None])[:, :, None, None], i["do"], 0.0))
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (do * o).sum(-1, keepdim=True)
    ds *= p
    group = lambda t, like: t.permute(0, 2, 1, 3).to(like.dtype)  # noqa: E731
    out["dv"] = group(torch.matmul(p.transpose(-1, -2), do), i["v"])
    del p
    out["dq"] = join(torch.matmul(ds, k) * scale)
    out["dk"] = group(torch.matmul(ds.transpose(-1, -2), q) * scale, i["k"])
    if c["kind"] == "relpos":
        # the diagonals' sums: in rows of n - 1 values read again as rows of n, entry (r, j) stands in column j - r
        n = Sq + Sk
        skew = F.pad(ds.reshape(B, H, Sq, Sk), (0, Sq - 1)).reshape(B, H, -1)
        by = F.pad(skew, (0, Sq)).reshape(B, H, Sq, n).sum(2, dtype=torch.float64)
        at = torch.arange(n, device=dev)
        at = (torch.where(at < Sk, at, at - n)[None, :] - (kl - ql)[:, None]).clamp(-M, M) + M  # [B, n]
        grad = torch.zeros(H, 2 * M + 1, device=dev, dtype=torch.float64)
        grad.index_add_(1, at.reshape(-1), by.permute(1, 0, 2).reshape(H, -1))
        out["dbias"] = grad.float()
        table = torch.zeros(c["buckets"], H, device=dev, dtype=torch.float64)
        out["dtable"] = table.index_add_(0, out["buckets"].long(), grad.t()).float()
    return out


# ---------------------------------------------------------------------------------------------------------
# The framework's calls
# ---------------------------------------------------------------------------------------------------------

_WORKSPACE_BYTES = 1 << 30
_th = None
_workspace = None


def _library():
    """The binding, with the thread in the asynchronous mode and a workspace bound, as a training loop sets itself up."""
    global _th, _workspace
    if _th is None:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "talos-xii_amd"))
        import talos_hip
        _workspace = torch.empty(_WORKSPACE_BYTES, device="cuda", dtype=torch.uint8)
        talos_hip.call("talos_set_async", 1)
        talos_hip.call("talos_workspace_bind", _workspace.data_ptr(), _WORKSPACE_BYTES)
        _th = talos_hip
    return _th


def _p(t):
    return None if t is None else t.data_ptr()


def _own(c, i, o):
    th, st, ty = _library(), torch.cuda.current_stream().cuda_stream, c["type"]
    if c["kind"] == "norm":
        R, D = c["rows"], c["dim"]
        th.call("talos_layernorm_fwd_" + ty, R, D, _EPS, _p(i["x"]), _p(i["w"]), _p(i["b"]), _p(o["y"]), _p(o["mean"]),
                _p(o["rstd"]), st)
        th.call("talos_layernorm_bwd_" + ty, R, D, _p(i["x"]), _p(i["w"]), _p(o["mean"]), _p(o["rstd"]), _p(i["dy"]),
                0.0, _p(o["dx"]), 0.0, _p(o["dw"]), _p(o["db"]), st)
        return o
    if c["kind"] == "loss":
        V = c["vocab"]
        th.call("talos_policy_loss_bwd_" + ty, c["rows"], V, _CLIP_LOW, _CLIP_HIGH, _KL, _p(i["logits"]), V,
                _p(i["actions"]), _p(i["adv"]), _p(i["old"]), _p(i["ref"]), _p(i["weight"]), _p(o["dlogits"]), V,
                _p(o["loss"]), _p(o["logp"]), None, 0, st)
        return o
    H, KV, dk, dv = (c[k] for k in ("H", "KV", "dk", "dv"))
    bias, M = None, 0
    if c["kind"] == "relpos":
        bias, M = o["bias"], c["max_distance"]
        th.call("talos_relpos_bias_fwd_f32", c["buckets"], H, M, 1 - c["causal"], _p(i["table"]), _p(bias),
                _p(o["buckets"]), st)
    cfg = th.GqaCfg(c["B"], c["Sq"], c["Sk"], H, KV, dk, dv, c["causal"], M, 1.0 / math.sqrt(dk))
    at = [cfg, _p(i["qlen"]), _p(i["klen"]), _p(bias), _p(i["q"]), H * dk, _p(i["k"]), KV * dk, _p(i["v"]), KV * dv,
          _p(o["o"]), H * dv, _p(o["lse"])]
    th.call("talos_gqa_fwd_" + ty, *at, st)
    if c["grad"]:
        th.call("talos_gqa_bwd_" + ty, *at, _p(i["do"]), H * dv, _p(o["dq"]), H * dk, _p(o["dk"]), KV * dk,
                _p(o["dv"]), KV * dv, 0.0, _p(o.get("dbias")), st)
        if c["kind"] == "relpos":
            th.call("talos_relpos_bias_bwd_f32", c["buckets"], H, M, 1 - c["causal"], _p(o["dbias"]), 0.0,
                    _p(o["dtable"]), st)
    return o


def run(state):
    c, i = state["case"], state["in"]
    if own:
        return _own(c, i, state["out"])
    if c["kind"] == "norm":
        return _plain_norm(c, i)
    if c["kind"] == "loss":
        return _plain_loss(c, i)
    return _plain_attn(c, i)


# ---------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------

def work(case):
    c, el = case, 2 if case["type"] == "bf16" else 4
    if c["kind"] == "norm":
        # x and dy in, y and dx out; the forward and the backward pass are two calls, so x is read by both
        n = c["rows"] * c["dim"]
        return {"bytes": 5 * n * el + 16 * c["dim"] + 16 * c["rows"], "flops": 20 * n}
    if c["kind"] == "loss":
        n = c["rows"] * c["vocab"]
        return {"bytes": 2 * n * el + 24 * c["rows"], "flops": 8 * n}
    B, Sq, Sk, H, KV, dk, dv = (c[k] for k in ("B", "Sq", "Sk", "H", "KV", "dk", "dv"))
    lq, lk = _lengths(c)
    spread = [j / max(1, B - 1) for j in range(B)]
    kl = [round(lk + (Sk - lk) * t) if c["ragged"] else Sk for t in spread]
    ql = kl if Sq == Sk else [round(lq + (Sq - lq) * t) if c["ragged"] else Sq for t in spread]
    pairs = nq = nk = 0
    for a, b in zip(ql, kl):
        # query i sees the first i + 1 + b - a keys where causal, else all b
        full, short = min(a, b), max(0, b - a)
        pairs += full * short + full * (full + 1) // 2 if c["causal"] else a * b
        nq, nk = nq + a, nk + b
    n_in = nq * H * dk + nk * KV * (dk + dv)
    n_out = B * Sq * H * dv
    total, flops = (n_in + n_out) * el + 4 * B * H * Sq, 2 * pairs * H * (dk + dv)
    if c["grad"]:
        total += (n_in + 2 * nq * H * dv) * el + 4 * nq * H + (B * Sq * H * dk + B * Sk * KV * (dk + dv)) * el
        flops += 2 * pairs * H * (3 * dk + 2 * dv)
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------

def _exact_bucket(c, d):
    """The bucket of distance d (key minus query) in whole numbers: the logarithm's steps compared as powers."""
    both = not c["causal"]
    side = c["buckets"] // 2 if both else c["buckets"]
    n, few, far = (abs(d) if both else max(0, -d)), side // 2, c["max_distance"]
    b = n
    if n >= few:
        steps = side - few
        t = 0
        while t < steps - 1 and n ** steps * few ** (t + 1) >= far ** (t + 1) * few ** steps:
            t += 1
        b = few + t
    return b + (side if both and d > 0 else 0)


def exact(case, seed):
    c, i = case, _inputs(case, seed)
    if c["kind"] == "norm":
        x, w, b = (i[k].double().requires_grad_() for k in ("x", "w", "b"))
        mean, var = x.mean(1), x.var(1, unbiased=False)
        y = (x - mean[:, None]) / torch.sqrt(var + _EPS)[:, None] * w + b
        dx, dw, db = torch.autograd.grad(y, (x, w, b), i["dy"].double())
        return {"y": y.detach(), "mean": mean.detach(), "rstd": (var + _EPS).rsqrt().detach(), "dx": dx, "dw": dw,
                "db": db}
    if c["kind"] == "loss":
        keep = i["weight"] != 0
        x = i["logits"].double().requires_grad_()
        logp = torch.log_softmax(x, 1)[torch.arange(c["rows"], device="cuda"), i["actions"].long()]
        adv = i["adv"].double()
        ratio = (logp - i["old"].double()).exp()
        gain = torch.minimum(ratio * adv, ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * adv)
        gap = i["ref"].double() - logp
        loss = ((_KL * (gap.exp() - gap - 1) - gain) * i["weight"].double())[keep].sum()
        d = torch.autograd.grad(loss, x)[0]
        return {"loss": loss.detach()[None], "logp": torch.where(keep, logp.detach(), 0.0), "dlogits": d}
    B, Sq, Sk, H, KV, dk, dv = (c[k] for k in ("B", "Sq", "Sk", "H", "KV", "dk", "dv"))
    wide = dict(dtype=torch.float64, device="cuda")
    out = {"o": torch.zeros(B, Sq, H, dv, **wide), "lse": torch.full((B, H, Sq), -math.inf, **wide)}
    table = None
    if c["kind"] == "relpos":
        M = c["max_distance"]
        out["buckets"] = torch.tensor([_exact_bucket(c, d) for d in range(-M, M + 1)], device="cuda", dtype=torch.int32)
        out["bias"] = i["table"].double()[out["buckets"].long()].t().contiguous()
    if c["grad"]:
        out.update(dq=torch.zeros(B, Sq, H, dk, **wide), dk=torch.zeros(B, Sk, KV, dk, **wide),
                   dv=torch.zeros(B, Sk, KV, dv, **wide))
        if c["kind"] == "relpos":
            out.update(dbias=torch.zeros(H, 2 * M + 1, **wide))
    for b in range(B):
        ql = Sq if i["qlen"] is None else int(i["qlen"][b])
        kl = Sk if i["klen"] is None else int(i["klen"][b])
        if not ql or not kl:
            continue
        place = torch.arange(ql, device="cuda") + kl - ql
        apart = torch.arange(kl, device="cuda") - place[:, None]
        hide = apart > 0 if c["causal"] else torch.zeros_like(apart, dtype=torch.bool)
        none = hide.all(1)
        if c["kind"] == "relpos":
            near = apart.clamp(-M, M) + M
        for h in range(H):
            q, k, v = (t.double().requires_grad_() for t in
                       (i["q"][b, :ql, h], i["k"][b, :kl, h // (H // KV)], i["v"][b, :kl, h // (H // KV)]))
            a = (q @ k.t()) / math.sqrt(dk)
            if c["kind"] == "relpos":
                table = out["bias"][h].clone().requires_grad_()
                a = a + table[near]
            a = a.masked_fill(hide, -math.inf)[~none]
            o = torch.softmax(a, 1) @ v
            out["o"][b, :ql, h][~none] = o.detach()
            out["lse"][b, h, :ql][~none] = torch.logsumexp(a.detach(), 1)
            if c["grad"]:
                leaves = [q, k, v] + ([] if table is None else [table])
                g = torch.autograd.grad(o, leaves, i["do"][b, :ql, h].double()[~none])
                out["dq"][b, :ql, h] += g[0]
                out["dk"][b, :kl, h // (H // KV)] += g[1]
                out["dv"][b, :kl, h // (H // KV)] += g[2]
                if table is not None:
                    out["dbias"][h] += g[3]
    if "dbias" in out:
        out["dtable"] = torch.zeros(c["buckets"], H, **wide).index_add_(0, out["buckets"].long(), out["dbias"].t())
    return out
