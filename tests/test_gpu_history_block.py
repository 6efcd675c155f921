"""The long-history operators run together as a training step of a policy uses them, beside the library's GEMM: layer norm,
q | k | v products, a relative position bias by buckets, grouped-query attention over right-padded histories past 256
tokens, output product and residual, layer norm, logits, the clipped policy loss with a KL term, and all of it backwards.
The gradients are compared with torch's autograd of the same step in float64 on the CPU, eagerly and from a captured graph
that is replayed with other work between."""
import math

import pytest
import torch

import operators_ref as ref
import talos_hip as th
from operators_ref import float32_default  # noqa: F401

B, S, D, H, KV, HD, V, NB, FAR = 3, 300, 64, 4, 2, 16, 1003, 16, 64
EPS, CLIP, KL = 1e-5, (0.2, 0.28), 0.05
LENS = [300, 41, 177]
R, N = B * S, 2 * FAR + 1
SHAPES = {"x": (R, D), "g1": (D,), "b1": (D,), "wq": (D, H * HD), "wk": (D, KV * HD), "wv": (D, KV * HD),
          "wo": (H * HD, D), "table": (NB, H), "g2": (D,), "b2": (D,), "wl": (D, V)}


def p(t):
    return None if t is None else t.data_ptr()


def inputs():
    g = torch.Generator().manual_seed(3)
    t = {}
    for n, s in SHAPES.items():
        t[n] = torch.randn(s, generator=g) * (1.0 if n == "x" else 0.3 if n == "table" else s[0] ** -0.5 if len(s) == 2 else 0.1)
        if n in ("g1", "g2"):
            t[n] += 1
    t["actions"] = torch.randint(0, V, (R,), generator=g, dtype=torch.int32)
    t["adv"] = torch.randn(R, generator=g)
    live = (torch.arange(S)[None, :] < torch.tensor(LENS)[:, None]).reshape(-1)
    t["weight"] = torch.where(live, 1.0 / sum(LENS), 0.0)
    return t


def forward64(t, old, rp):
    x = t["x"]
    norm = lambda a, g, b: ref.layernorm(a, g, b, a.detach(), EPS)[0]  # noqa: E731
    a = norm(x, t["g1"], t["b1"])
    q, k, v = ((a @ t[w]).reshape(B, S, -1, HD) for w in ("wq", "wk", "wv"))
    idx = torch.tensor([ref.bucket(d, NB, FAR, 0) for d in range(-FAR, FAR + 1)])
    bias = t["table"][idx].t()
    place = torch.arange(S)
    apart = place[None, :] - place[:, None]
    rows = []
    for b in range(B):
        n = LENS[b]
        s = torch.einsum("ihd,jhd->hij", q[b, :n], k[b, :n].repeat_interleave(H // KV, 1)) / math.sqrt(HD)
        s = s + bias[:, apart[:n, :n].clamp(-FAR, FAR) + FAR]
        o = torch.softmax(s.masked_fill(apart[:n, :n] > 0, -math.inf), -1)
        o = torch.einsum("hij,jhd->ihd", o, v[b, :n].repeat_interleave(H // KV, 1)).reshape(n, H * HD)
        rows.append(torch.cat([o, o.new_zeros(S - n, H * HD)]))
    logits = norm(x + torch.cat(rows) @ t["wo"], t["g2"], t["b2"]) @ t["wl"]
    logp = torch.log_softmax(logits, 1)[torch.arange(R), t["actions"].long()]
    ratio = torch.exp(logp - old)
    gain = torch.minimum(ratio * t["adv"], ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * t["adv"])
    gap = rp - logp
    return (t["weight"] * (KL * (torch.exp(gap) - gap - 1) - gain)).sum(), logp


@pytest.mark.gpu
def test_training_step_of_a_policy_over_histories():
    t = inputs()
    d = {n: v.double() if v.dtype == torch.float32 else v for n, v in t.items()}
    with torch.no_grad():
        lp = forward64(d, torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64))[1]
    g = torch.Generator().manual_seed(4)
    old, rp = (lp + 0.4 * torch.randn(R, generator=g)).float(), (lp + 0.2 * torch.randn(R, generator=g)).float()
    leaves = {n: d[n].requires_grad_() for n in SHAPES}
    loss, _ = forward64(d, old.double(), rp.double())
    want = dict(zip(SHAPES, torch.autograd.grad(loss, list(leaves.values()))))

    c = {n: v.cuda() for n, v in t.items()}
    c["old"], c["rp"] = old.cuda(), rp.cuda()
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    new = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    grad = {n: new(*s) for n, s in SHAPES.items()}
    a, a_mean, a_rstd, q, k, v = new(R, D), new(R), new(R), new(R, H * HD), new(R, KV * HD), new(R, KV * HD)
    bias, dbias, o, lse, y, z = new(H, N), new(H, N), new(R, H * HD), new(B, H, S), new(R, D), new(R, D)
    z_mean, z_rstd, logits, dz, dy = new(R), new(R), new(R, V), new(R, D), new(R, D)
    do, dq, dk, dv, da, out = new(R, H * HD), new(R, H * HD), new(R, KV * HD), new(R, KV * HD), new(R, D), new(1)
    cfg = th.GqaCfg(B, S, S, H, KV, HD, HD, 1, FAR, 1 / math.sqrt(HD))
    heads = [p(q), H * HD, p(k), KV * HD, p(v), KV * HD, p(o), H * HD, p(lse)]
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")

    def gemm(ta, tb, m, n, kk, x, lda, w, ldb, beta, r, ldr, s):
        th.call("talos_gemm_f32", ta, tb, m, n, kk, 1.0, p(x), lda, p(w), ldb, beta, p(r), ldr, s)

    def step(s):
        th.call("talos_layernorm_fwd_f32", R, D, EPS, p(c["x"]), p(c["g1"]), p(c["b1"]), p(a), p(a_mean), p(a_rstd), s)
        for w, r, n in (("wq", q, H * HD), ("wk", k, KV * HD), ("wv", v, KV * HD)):
            gemm(0, 0, R, n, D, a, D, c[w], n, 0.0, r, n, s)
        th.call("talos_relpos_bias_fwd_f32", NB, H, FAR, 0, p(c["table"]), p(bias), None, s)
        th.call("talos_gqa_fwd_f32", cfg, p(lens), p(lens), p(bias), *heads, s)
        th.call("talos_unary_fwd_f32", th.COPY, R * D, 0.0, 0.0, p(c["x"]), p(y), s)
        gemm(0, 0, R, D, H * HD, o, H * HD, c["wo"], D, 1.0, y, D, s)
        th.call("talos_layernorm_fwd_f32", R, D, EPS, p(y), p(c["g2"]), p(c["b2"]), p(z), p(z_mean), p(z_rstd), s)
        gemm(0, 0, R, V, D, z, D, c["wl"], V, 0.0, logits, V, s)
        # the logits' gradient over the logits themselves
        th.call("talos_policy_loss_bwd_f32", R, V, *CLIP, KL, p(logits), V, p(c["actions"]), p(c["adv"]), p(c["old"]),
                p(c["rp"]), p(c["weight"]), p(logits), V, p(out), None, None, 0, s)
        gemm(1, 0, D, V, R, z, D, logits, V, 0.0, grad["wl"], V, s)
        gemm(0, 1, R, D, V, logits, V, c["wl"], V, 0.0, dz, D, s)
        th.call("talos_layernorm_bwd_f32", R, D, p(y), p(c["g2"]), p(z_mean), p(z_rstd), p(dz), 0.0, p(dy), 0.0,
                p(grad["g2"]), p(grad["b2"]), s)
        gemm(1, 0, H * HD, D, R, o, H * HD, dy, D, 0.0, grad["wo"], D, s)
        gemm(0, 1, R, H * HD, D, dy, D, c["wo"], D, 0.0, do, H * HD, s)
        th.call("talos_gqa_bwd_f32", cfg, p(lens), p(lens), p(bias), *heads, p(do), H * HD, p(dq), H * HD, p(dk), KV * HD,
                p(dv), KV * HD, 0.0, p(dbias), s)
        th.call("talos_relpos_bias_bwd_f32", NB, H, FAR, 0, p(dbias), 0.0, p(grad["table"]), s)
        for i, (w, r, n) in enumerate((("wq", dq, H * HD), ("wk", dk, KV * HD), ("wv", dv, KV * HD))):
            gemm(1, 0, D, n, R, a, D, r, n, 0.0, grad[w], n, s)
            gemm(0, 1, R, D, n, r, n, c[w], n, float(i > 0), da, D, s)
        th.call("talos_unary_fwd_f32", th.COPY, R * D, 0.0, 0.0, p(dy), p(grad["x"]), s)
        th.call("talos_layernorm_bwd_f32", R, D, p(c["x"]), p(c["g1"]), p(a_mean), p(a_rstd), p(da), 1.0, p(grad["x"]), 0.0,
                p(grad["g1"]), p(grad["b1"]), s)

    torch.cuda.synchronize()
    step(None)
    torch.cuda.synchronize()
    assert abs(out.item() - loss.item()) <= 1e-6 * (1 + abs(loss.item()))
    first = {n: grad[n].clone() for n in grad}
    for n in grad:
        # some ten stages, each good to 32 u of its terms in norm
        err = (grad[n].cpu().double() - want[n]).norm() / want[n].norm()
        assert err < 10 * 32 * ref.U32, (n, float(err))
    stream = th.stream_create()
    th.call("talos_workspace_bind", ws.data_ptr(), ws.numel())
    try:
        graph = th.Graph(stream, lambda: step(stream))
        for turn in range(4):
            for n in grad:
                grad[n].zero_()
            ws.fill_(255)
            junk = torch.randn(1 << 20, device="cuda").sum()
            torch.cuda.synchronize()
            graph.launch()
            th.call("talos_stream_sync", stream)
            for n in grad:
                # the library's GEMM may split its K otherwise with a workspace bound; the new operators do not
                err = (grad[n] - first[n]).norm() / first[n].norm()
                assert err < 10 * 32 * ref.U32, (turn, n, float(err))
            assert torch.isfinite(junk)
    finally:
        th.call("talos_workspace_bind", None, 0)
        th.stream_destroy(stream)
