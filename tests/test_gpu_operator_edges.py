"""The long-history operators where sizes and sharing are extreme: rows a gigabyte apart in a cache that 32-bit offsets do
not reach, rows of a million values, results in an input's place, two streams at work at once."""
import math

import pytest
import torch

import operators_ref as ref
import test_gpu_norm_loss as norm
import talos_hip as th
from operators_ref import float32_default  # noqa: F401

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
pytestmark = pytest.mark.gpu


def p(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_cache_past_32_bit_offsets(ty):
    """A token against 1.2 million keys in rows of 2048 values (keys and values of 64 in each): 2.5e9 elements a sample."""
    Sk, ld, H, d = 1_200_000, 2048, 4, 64
    rows = torch.empty(Sk, ld, dtype=DT[ty], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    rows[:, :2 * d] = torch.randn(Sk, 2 * d, generator=g, device="cuda")
    q, do = (torch.randn(H, d, generator=g, device="cuda").to(DT[ty]) for _ in range(2))
    o, dq = torch.empty_like(q), torch.empty_like(q)
    dk, dv = (torch.empty(Sk, d, dtype=DT[ty], device="cuda") for _ in range(2))
    lse = torch.empty(H, device="cuda")
    cfg = th.GqaCfg(1, 1, Sk, H, 1, d, d, 1, 0, 0.125)
    ins = [p(q), H * d, p(rows), ld, p(rows) + d * rows.element_size(), ld, p(o), H * d, p(lse)]
    th.call("talos_gqa_fwd_" + ty, cfg, None, None, None, *ins, None)
    th.call("talos_gqa_bwd_" + ty, cfg, None, None, None, *ins, p(do), H * d, p(dq), H * d, p(dk), d, p(dv), d, 0.0, None,
            None)
    K, V, Q, G = rows[:, :d].double(), rows[:, d:2 * d].double(), q.double(), do.double()
    s = 0.125 * Q @ K.t().contiguous()
    P = torch.softmax(s, 1)
    O = P @ V
    D = (G * O).sum(1, keepdim=True)
    dS = P * (G @ V.t().contiguous() - D)
    w = 1 + (0.125 * Q.abs() @ K.abs().t().contiguous()).amax(1, keepdim=True)  # a score's error is its probability's share
    Dh = (G.abs() * (P @ V.abs() + O.abs())).sum(1, keepdim=True)
    A = P * (G.abs() @ V.abs().t().contiguous() + Dh)  # the magnitudes of dS's terms
    half = 2.0 ** -8 if ty == "bf16" else 0.0
    for name, got, want, mag, size in (
            ("o", o, O, P @ V.abs() * w, P @ V.abs()),
            ("dq", dq, 0.125 * dS @ K, 0.125 * (A * w) @ K.abs(), 0.125 * (dS.abs() + P * Dh) @ K.abs()),
            ("dk", dk, 0.125 * dS.t() @ Q, 0.125 * (A * w).t() @ Q.abs(), 0.125 * (dS.abs() + P * Dh).t() @ Q.abs()),
            ("dv", dv, P.t() @ G, (P * w).t() @ G.abs(), P.t() @ G.abs())):
        ref.close(got.cpu(), want.cpu(), (mag + size * half / (32 * ref.U32)).cpu(), 1 if ty == "bf16" else 0, name)
    ref.close(lse.cpu(), torch.logsumexp(s, 1).cpu(), w[:, 0].cpu() + 14, name="lse")


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_layernorm_of_rows_of_a_million(ty):
    """The mean of 2^20 + 5 values far from zero: the sums of a lane hold 4096 terms."""
    rows, dim = 3, (1 << 20) + 5
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(rows, dim, generator=g) + 30).to(DT[ty])
    dy, w, b = torch.randn(rows, dim, generator=g).to(DT[ty]), 1 + 0.1 * torch.randn(dim, generator=g), torch.zeros(dim)
    y, mean, rstd, dx, dw, db = ref.layernorm(x.double(), w.double(), b.double(), dy.double(), 1e-5)
    X, DY, W = x.cuda(), dy.cuda(), w.cuda()
    Y, DX, M, R = torch.empty_like(X), torch.empty_like(X), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    DW, DB = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    th.call("talos_layernorm_fwd_" + ty, rows, dim, 1e-5, p(X), p(W), None, p(Y), p(M), p(R), None)
    th.call("talos_layernorm_bwd_" + ty, rows, dim, p(X), p(W), p(M), p(R), p(DY), 0.0, p(DX), 0.0, p(DW), p(DB), None)
    # a lane's sums are f64 and the tree over 256 lanes has 8 levels: 16 steps of fp32 are ample
    far = 31.0 * rstd[:, None]
    rounds = 1 if ty == "bf16" else 0
    ref.close(M.cpu(), mean, torch.full_like(mean, 31.0), name="mean", k=16)
    ref.close(R.cpu(), rstd, rstd, name="rstd", k=16)
    ref.close(Y.cpu(), y, (far + y.abs()) * w.double().abs(), rounds, "y", k=16)
    h = (dy * w).double().abs()
    ref.close(DX.cpu(), dx, rstd[:, None] * (h + 1 + (far + y.abs()) * 2), rounds, "dx", k=16)
    ref.close(DW.cpu(), dw, (dy.double().abs() * (far + y.abs())).sum(0), name="dw")
    ref.close(DB.cpu(), db, dy.double().abs().sum(0), name="db")


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(1300, 40), (700, 1024), (9, 20000)])
def test_layernorm_in_place(rows, dim, ty):
    g = torch.Generator(device="cuda").manual_seed(3)
    x, dy = (torch.randn(rows, dim, generator=g, device="cuda").to(DT[ty]) for _ in range(2))
    w, b = (torch.randn(dim, generator=g, device="cuda") for _ in range(2))
    M, R, DW, DB = (torch.empty(n, device="cuda") for n in (rows, rows, dim, dim))
    y, dx = torch.empty_like(x), torch.empty_like(x)
    th.call("talos_layernorm_fwd_" + ty, rows, dim, 1e-5, p(x), p(w), p(b), p(y), p(M), p(R), None)
    th.call("talos_layernorm_bwd_" + ty, rows, dim, p(x), p(w), p(M), p(R), p(dy), 0.0, p(dx), 0.0, p(DW), p(DB), None)
    want = [DW.clone(), DB.clone()]
    th.call("talos_layernorm_bwd_" + ty, rows, dim, p(x), p(w), p(M), p(R), p(dy), 0.0, p(dy), 0.0, p(DW), p(DB), None)
    th.call("talos_layernorm_fwd_" + ty, rows, dim, 1e-5, p(x), p(w), p(b), p(x), None, None, None)
    torch.cuda.synchronize()
    assert torch.equal(x, y) and torch.equal(dy, dx) and torch.equal(DW, want[0]) and torch.equal(DB, want[1])


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [2, 7, 9, 1540, 2055, 2056, 2057, 2304, 3100, 4100, 5001, 6143, 6145, 8191])
def test_layernorm_where_shapes_change(dim, ty):
    norm.test_layernorm(dim, ty)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(53, 7573), (40, 23), (37, 40001), (700, 6)])
def test_policy_loss_whose_gains_cancel(rows, vocab, ty):
    """A loss of a thousandth of its terms, whose scalars are f64: what is left is the loss's own rounding and the errors of
    the log-probabilities. In long rows an exponential is fp32, off by its own and its piece's roundings (2^-22) and its
    argument's (2^-24 of it), which are independent: a row's sum is off by their root mean square, and the loss by that of
    its rows. In short rows they are f64 (2^-38 is ample). Four deviations."""
    x, a, adv, old, rp, w = norm.loss_inputs(rows, vocab, ty, 12)
    loss0, *_ = ref.policy_loss(x.double(), a, adv.double(), old.double(), None, w.double(), 9.0, 9.0, 0.0)
    lp = torch.log_softmax(x.double(), 1).gather(1, a.long()[:, None])[:, 0]
    ratio = torch.exp(lp - old.double())
    t = int((w * ratio).argmax())
    adv[t] += float(loss0) / float(w[t].double() * ratio[t]) * 0.999  # the largest row balances the rest
    loss, *_ = ref.policy_loss(x.double(), a, adv.double(), old.double(), None, w.double(), 9.0, 9.0, 0.0)
    terms = (w.double() * ratio * adv.double()).abs()
    assert abs(loss) < 0.1 * terms.sum()
    got, *_ = norm.loss_call(ty, x, a, adv, old, None, w, (9.0, 9.0), 0.0)
    gap = x.double() - x.double().max(1, keepdim=True).values
    each = (torch.softmax(gap, 1) * (2.0 ** -22 - 2.0 ** -24 * gap)).norm(dim=1) if vocab > 64 else torch.tensor(2.0 ** -38)
    assert abs(float(got) - loss) <= 2.0 ** -24 * abs(loss) + 4 * float((terms * each).norm())


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_two_streams_at_once(ty):
    """With no workspace bound, calls on two streams take scratch of their own: each result as when it ran alone."""
    B, S, H, KV, d, M, rows, vocab = 2, 300, 4, 2, 64, 60, 96, 5000
    sets = []
    for seed in (4, 5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[ty])  # noqa: E731
        t = {"q": rnd(B, S, H, d), "k": rnd(B, S, KV, d), "v": rnd(B, S, KV, d), "do": rnd(B, S, H, d), "x": rnd(rows, vocab)}
        t["bias"] = torch.randn(H, 2 * M + 1, generator=g, device="cuda")
        t["act"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda").int()
        t["adv"], t["old"] = torch.randn(rows, generator=g, device="cuda"), torch.full((rows,), -math.log(vocab), device="cuda")
        out = {n: torch.zeros_like(t[n]) for n in ("q", "k", "v", "do", "bias", "x")}
        out["lse"], out["loss"] = torch.zeros(B, H, S, device="cuda"), torch.zeros(1, device="cuda")
        sets.append((t, out))

    def go(t, out, s):
        cfg = th.GqaCfg(B, S, S, H, KV, d, d, 1, M, 0.125)
        ins = [None, None, p(t["bias"]), p(t["q"]), H * d, p(t["k"]), KV * d, p(t["v"]), KV * d, p(out["do"]), H * d,
               p(out["lse"])]
        th.call("talos_gqa_fwd_" + ty, cfg, *ins, s)
        th.call("talos_gqa_bwd_" + ty, cfg, *ins, p(t["do"]), H * d, p(out["q"]), H * d, p(out["k"]), KV * d, p(out["v"]),
                KV * d, 0.0, p(out["bias"]), s)
        th.call("talos_policy_loss_bwd_" + ty, rows, vocab, 0.2, 0.2, 0.0, p(t["x"]), vocab, p(t["act"]), p(t["adv"]),
                p(t["old"]), None, None, p(out["x"]), vocab, p(out["loss"]), None, None, 0, s)

    torch.cuda.synchronize()
    want = []
    for t, out in sets:
        go(t, out, None)
        torch.cuda.synchronize()
        want.append({n: v.clone() for n, v in out.items()})
        for v in out.values():
            v.zero_()
    torch.cuda.synchronize()
    streams = [th.stream_create() for _ in sets]
    try:
        for _ in range(3):
            for s, (t, out) in zip(streams, sets):
                go(t, out, s)
        for s in streams:
            th.call("talos_stream_sync", s)
        for (_, out), w in zip(sets, want):
            for n, v in out.items():
                assert torch.equal(v, w[n]), n
    finally:
        for s in streams:
            th.stream_destroy(s)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_wide_heads_in_a_graph(ty):
    """Head dims of 128, whose tiles take more than 64 KB of a workgroup's LDS, captured; eager work between the replays."""
    B, S, H, KV, d, M = 2, 190, 4, 2, 128, 33
    g = torch.Generator(device="cuda").manual_seed(6)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(DT[ty])  # noqa: E731
    q, k, v, do = rnd(B, S, H, d), rnd(B, S, KV, d), rnd(B, S, KV, d), rnd(B, S, H, d)
    bias = torch.randn(H, 2 * M + 1, generator=g, device="cuda")
    out = [torch.zeros_like(t) for t in (do, q, k, v, bias)] + [torch.zeros(B, H, S, device="cuda")]
    o, dq, dk, dv, db, lse = out
    cfg = th.GqaCfg(B, S, S, H, KV, d, d, 1, M, d ** -0.5)

    def go(s):
        ins = [None, None, p(bias), p(q), H * d, p(k), KV * d, p(v), KV * d, p(o), H * d, p(lse)]
        th.call("talos_gqa_fwd_" + ty, cfg, *ins, s)
        th.call("talos_gqa_bwd_" + ty, cfg, *ins, p(do), H * d, p(dq), H * d, p(dk), KV * d, p(dv), KV * d, 0.0, p(db), s)

    keep = torch.empty(32 << 20, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    stream = th.stream_create()
    th.call("talos_workspace_bind", keep.data_ptr(), keep.numel())
    try:
        graph = th.Graph(stream, lambda: go(stream))
        want = None
        for turn in range(3):
            for t in out:
                t.zero_()
            torch.cuda.synchronize()
            go(None)
            torch.cuda.synchronize()
            want = [t.clone() for t in out]
            for t in out:
                t.fill_(7.0)
            torch.cuda.synchronize()
            graph.launch()
            th.call("talos_stream_sync", stream)
            for t, w in zip(out, want):
                assert torch.equal(t, w), turn
    finally:
        th.call("talos_workspace_bind", None, 0)
        th.stream_destroy(stream)
