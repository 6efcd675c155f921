"""Grouped-query attention (talos_gqa_fwd_*, talos_gqa_bwd_*) against its plain float64 form: lengths from none to long
ones, odd head dims, groups, queries and keys of different lengths, rows that see no key, the bias by distance and its
gradient, strided and unaligned tensors, padding full of NaN, graphs, streams, refusals."""
import ctypes
import math

import pytest
import torch

import operators_ref as ref
import talos_hip as th
from operators_ref import float32_default  # noqa: F401

P16 = ctypes.c_void_p(16)  # never dereferenced: the arguments' checks fail first
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def p(t):
    return None if t is None else t.data_ptr()


class Case:
    """Inputs on the CPU and strided copies on the GPU: ld = heads * dim + pad, the first value `offset` into a buffer."""

    def __init__(self, ty, B, Sq, Sk, H, KV, dk, dv, causal, qlens=None, klens=None, M=0, seed=0, pad=0, offset=0):
        g = torch.Generator().manual_seed(seed)
        self.ty, self.dims, self.causal, self.M = ty, (B, Sq, Sk, H, KV, dk, dv), causal, M
        self.qlens, self.klens = qlens, klens
        self.scale = 1 / math.sqrt(dk)
        rnd = lambda *s: torch.randn(*s, generator=g).to(DT[ty])  # noqa: E731
        self.q, self.k, self.v, self.do = rnd(B, Sq, H, dk), rnd(B, Sk, KV, dk), rnd(B, Sk, KV, dv), rnd(B, Sq, H, dv)
        self.bias = torch.randn(H, 2 * M + 1, generator=g) if M else None
        self.pad, self.offset = pad, offset
        self.dev = {n: self.put(t, lens) for n, t, lens in (("q", self.q, qlens), ("k", self.k, klens),
                                                            ("v", self.v, klens), ("do", self.do, qlens))}
        self.out = {n: self.put(torch.full_like(t, 5.0), None) for n, t in
                    (("o", self.do), ("dq", self.q), ("dk", self.k), ("dv", self.v))}
        self.lse = torch.full((B, H, Sq), 5.0, device="cuda")
        self.dbias = None if not M else torch.full((H, 2 * M + 1), 2.0, device="cuda")
        self.Bias = None if not M else self.bias.cuda()
        self.Q = None if qlens is None else torch.tensor(qlens, dtype=torch.int32, device="cuda")
        self.K = None if klens is None else torch.tensor(klens, dtype=torch.int32, device="cuda")
        self.cfg = th.GqaCfg(B, Sq, Sk, H, KV, dk, dv, causal, M, self.scale)

    def put(self, t, lens):
        B, S, n = t.shape[0], t.shape[1], t.shape[2] * t.shape[3]
        full = torch.full((B, S, n + self.pad), math.nan, dtype=t.dtype)  # nothing between rows or past a length is used
        full[:, :, :n] = t.reshape(B, S, n)
        if lens is not None:
            for b, l in enumerate(lens):
                full[b, max(l, 0):] = math.nan
        buf = torch.empty(full.numel() + self.offset + 8, dtype=t.dtype, device="cuda")
        at = buf[self.offset:self.offset + full.numel()].view(full.shape)
        at.copy_(full)
        return at

    def at(self, n):
        t = self.dev[n] if n in self.dev else self.out[n]
        return [p(t), t.shape[2] if t.numel() else 4096]

    def fwd(self, stream=None):
        th.call("talos_gqa_fwd_" + self.ty, self.cfg, p(self.Q), p(self.K), p(self.Bias), *self.at("q"), *self.at("k"),
                *self.at("v"), *self.at("o"), p(self.lse), stream)

    def bwd(self, beta=0.0, stream=None, dbias=True):
        th.call("talos_gqa_bwd_" + self.ty, self.cfg, p(self.Q), p(self.K), p(self.Bias), *self.at("q"), *self.at("k"),
                *self.at("v"), *self.at("o"), p(self.lse), *self.at("do"), *self.at("dq"), *self.at("dk"), *self.at("dv"),
                beta, p(self.dbias) if dbias else None, stream)

    def result(self):
        torch.cuda.synchronize()
        r = {"lse": self.lse.cpu()}
        for n, t in self.out.items():
            like = {"o": self.do, "dq": self.q, "dk": self.k, "dv": self.v}[n]
            w = like.shape[2] * like.shape[3]
            host = t.cpu()
            assert torch.isnan(host[:, :, w:].float()).all(), f"{n}: written between the rows"
            r[n] = host[:, :, :w].reshape(like.shape)
        if self.dbias is not None:
            r["dbias"] = self.dbias.cpu()
        return r

    def reference(self, grad=True):
        dbl = lambda t: None if t is None else t.double()  # noqa: E731
        return ref.attention(dbl(self.q), dbl(self.k), dbl(self.v), self.scale, self.causal, self.qlens, self.klens,
                             dbl(self.bias), dbl(self.do) if grad else None)

    def check(self, grad=True):
        self.fwd()
        if grad:
            self.bwd()
        names = ["o", "lse"] + (["dq", "dk", "dv"] + (["dbias"] if self.M else []) if grad else [])
        ref.close_attention(self.result(), self.reference(grad), self.ty, names)


# B, Sq, Sk, H, KV, dk, dv
SHAPES = [(1, 1, 1, 1, 1, 8, 8), (2, 1, 40, 4, 4, 32, 32), (2, 33, 33, 2, 2, 32, 32), (1, 64, 64, 2, 1, 64, 64),
          (2, 65, 65, 4, 2, 64, 64), (1, 130, 130, 3, 3, 64, 64), (2, 129, 200, 6, 2, 80, 80), (1, 200, 129, 2, 2, 128, 128),
          (3, 31, 95, 8, 1, 128, 128), (1, 300, 300, 4, 4, 96, 64), (2, 70, 70, 2, 2, 5, 3), (1, 97, 101, 4, 2, 40, 56),
          (1, 17, 257, 5, 5, 128, 33), (1, 260, 20, 2, 2, 64, 128), (9, 20, 20, 8, 8, 16, 16), (1, 8, 700, 8, 2, 64, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(shape, causal, ty):
    Case(ty, *shape, causal, seed=sum(shape)).check()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("dk,dv,H,KV", [(32, 32, 4, 4), (64, 64, 4, 2), (128, 128, 2, 1), (72, 24, 3, 3)])
def test_ragged_and_strided(dk, dv, H, KV, causal, ty):
    """Lengths of zero, one and past the padded ones; fewer keys than queries (causal rows that see nothing); NaN in every
    row past a length and between the rows; unaligned buffers."""
    lens = [0, 1, 150, 77, 400, -3, 64, 128]
    Case(ty, 8, 150, 150, H, KV, dk, dv, causal, lens, lens, seed=dk, pad=3, offset=1).check()
    Case(ty, 6, 70, 133, H, KV, dk, dv, causal, [70, 3, 70, 0, 50, 64], [133, 100, 20, 60, 0, 64], seed=dk + 1, pad=8).check()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("shape,causal,lens,M", [
    ((2, 33, 33, 2, 2, 32, 32), 1, None, 4), ((2, 200, 200, 4, 4, 64, 64), 0, [200, 131], 16),
    ((1, 300, 300, 2, 2, 64, 64), 1, None, 128), ((1, 257, 257, 4, 2, 128, 128), 0, None, 32),
    ((2, 90, 90, 8, 2, 80, 48), 1, [90, 17], 1), ((1, 150, 150, 2, 2, 16, 16), 0, None, 512),
    ((3, 1, 70, 4, 4, 64, 64), 1, None, 20), ((1, 40, 500, 2, 1, 32, 32), 0, None, 64)], ids=str)
def test_bias_by_distance(shape, causal, lens, M, ty):
    c = Case(ty, *shape, causal, lens, lens, M=M, seed=M)
    c.check()
    first = c.result()
    c.bwd(beta=1.0)  # accumulates: twice the gradient, every bit of the rest again
    again = c.result()
    for n in ("dq", "dk", "dv"):
        assert torch.equal(again[n], first[n]), n
    assert torch.equal(again["dbias"], (2 * first["dbias"].double()).float())
    c.bwd(dbias=False)
    assert torch.equal(c.result()["dbias"], again["dbias"])


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("Sq,Sk,H,KV,d", [(1, 3000, 4, 1, 128), (1, 2050, 32, 32, 64), (5, 1999, 8, 2, 64), (1, 1500, 40, 1, 32),
                                          (100, 2000, 2, 2, 128)])
def test_decode_against_long_keys(Sq, Sk, H, KV, d, ty):
    """Few rows: the waves split the keys, and so do the workgroups; samples of very different lengths."""
    Case(ty, 2, Sq, Sk, H, KV, d, d, 1, [Sq, Sq], [Sk, 37], seed=d).check(grad=False)
    c = Case(ty, 1, Sq, Sk, H, KV, d, d, 1, M=100, seed=d + 1)
    c.check()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_long_sequences_split_over_heads_and_queries(ty):
    Case(ty, 1, 700, 90, 8, 1, 64, 64, 0, seed=4).check()  # one key tile, many heads and queries
    Case(ty, 1, 1100, 1100, 2, 1, 32, 32, 1, M=50, seed=5).check()


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_scores_of_any_size(ty):
    """Scores of several hundred (one key takes all), equal scores, a bias of minus infinity."""
    c = Case(ty, 1, 70, 150, 2, 2, 64, 64, 0, M=200, seed=6)
    c.scale = c.cfg.scale = 20.0
    c.check()
    c = Case(ty, 1, 70, 150, 2, 2, 64, 64, 0, M=200, seed=7)
    c.bias[:, ::2] = -math.inf
    c.bias[0, :190] = -math.inf  # whole rows of head 0 hidden by the bias alone
    c.Bias.copy_(c.bias)
    c.fwd()
    got, want = c.result(), None
    c.bias = c.bias.clamp(min=-1e30)
    want = c.reference(grad=False)
    seen = want["lse"] > -1e29
    assert torch.equal(torch.isinf(got["lse"]), ~seen)
    rows = seen.permute(0, 2, 1)[..., None].expand_as(got["o"])
    ref.close(torch.where(seen, got["lse"], 0.0), torch.where(seen, want["lse"], 0.0), torch.where(seen, want["lse.f"], 0.0)
              .clamp(max=100), name="lse")
    assert not got["o"][~rows].any()
    keep = lambda t: torch.where(rows, t.double(), 0.0)  # noqa: E731
    w = {n: keep(want[n]) for n in ("o", "o.h", "o.u")}
    w["o.f"] = w["o.h"] * 100  # the scores that count are of order 10
    ref.close_attention({"o": keep(got["o"])}, w, ty, ["o"])


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, -3.5e30])
@pytest.mark.parametrize("causal", [0, 1])
def test_distances_hidden_by_the_bias(causal, low, ty):
    """Minus infinity and the type's lowest value hide a distance, on a block's edge, inside it and beyond M; rows that see
    only hidden keys get nothing, and neither they nor those keys get a gradient from them."""
    c = Case(ty, 2, 90, 190, 4, 2, 64, 64, causal, [90, 41], [190, 40], M=70, seed=11)
    c.bias[0, ::2] = low
    c.bias[1, 70] = low  # the query's own position; sample 1's second causal row sees nothing else
    c.bias[2, 0] = low  # everything far behind
    c.bias[3, 0], c.bias[3, 50:] = low, low
    c.Bias.copy_(c.bias)
    c.check()
    c = Case(ty, 1, 5, 40, 2, 2, 32, 32, causal, M=3, seed=12)
    c.bias[1] = low  # a head with nothing to see
    c.Bias.copy_(c.bias)
    c.check()


@pytest.mark.gpu
def test_gradients_against_differences():
    c = Case("f32", 1, 7, 9, 2, 1, 8, 8, 1, M=3, seed=8)
    c.fwd()
    c.bwd()
    got = c.result()
    h = 1e-5
    for n, like in (("dq", "q"), ("dk", "k"), ("dv", "v"), ("dbias", "bias")):
        base = getattr(c, like)
        for i in range(0, base.numel(), max(1, base.numel() // 9)):
            f = []
            for sign in (1, -1):
                t = base.double().clone()
                t.view(-1)[i] += sign * h
                args = {"q": c.q.double(), "k": c.k.double(), "v": c.v.double(), "bias": c.bias.double(), like: t}
                o = ref.attention(args["q"], args["k"], args["v"], c.scale, 1, None, None, args["bias"])["o"]
                f.append(float((o * c.do.double()).sum()))
            # a central difference: h^2 of a third derivative (order 10) and 2^-53 of a sum of order 50 over h
            assert abs((f[0] - f[1]) / (2 * h) - float(got[n].reshape(-1)[i])) < 1e-5, n


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
def test_same_bits_on_a_stream_in_a_graph_and_with_a_workspace(ty):
    c = Case(ty, 2, 150, 600, 4, 2, 64, 64, 1, [150, 33], [600, 90], M=40, seed=9)
    c.check()
    want = c.result()
    keep = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    for t in [c.lse, *c.out.values(), c.dbias]:
        t.zero_()
    for t, like in zip(c.out.values(), (c.do, c.q, c.k, c.v)):
        t[:, :, like.shape[2] * like.shape[3]:] = math.nan
    torch.cuda.synchronize()
    stream = th.stream_create()
    th.call("talos_workspace_bind", keep.data_ptr(), keep.numel())
    try:
        graph = th.Graph(stream, lambda: (c.fwd(stream), c.bwd(stream=stream)))
        for turn in range(4):
            graph.launch()
            th.call("talos_stream_sync", stream)
            got = c.result()
            for n, t in want.items():
                assert torch.equal(got[n], t), (turn, n)
            keep.fill_(255)  # NaN: nothing of the last turn's scratch is used
            c.lse.zero_()
            torch.cuda.synchronize()
        c.fwd(stream)
        c.bwd(stream=stream)
        got = c.result()
        for n, t in want.items():
            assert torch.equal(got[n], t), n
        assert 0 < th.lib().talos_workspace_high_water() <= keep.numel()
    finally:
        th.call("talos_workspace_bind", None, 0)
        th.stream_destroy(stream)


@pytest.mark.gpu
def test_empty_batches_and_lengths():
    c = Case("f32", 2, 5, 7, 2, 2, 16, 16, 0, M=3, seed=10)
    for B, Sq, Sk in ((0, 5, 7), (2, 0, 7), (2, 5, 0)):
        c.cfg.batch, c.cfg.q_len, c.cfg.k_len = B, Sq, Sk
        for t in [c.lse, *c.out.values(), c.dbias]:
            t.fill_(5.0)
        c.fwd()
        c.bwd()
        torch.cuda.synchronize()
        assert not c.dbias.any()
        if B and Sq:
            assert not c.out["o"].any() and not c.out["dq"].any() and torch.isinf(c.lse).all()
        if B and Sk:
            assert not c.out["dk"].any() and not c.out["dv"].any()


def test_refusals():
    L = th.lib()
    good = dict(batch=2, q_len=8, k_len=8, heads=4, kv_heads=2, qk_dim=16, v_dim=16, causal=1, max_distance=8, scale=0.25)

    def cfg(**kw):
        return ctypes.byref(th.GqaCfg(**{**good, **kw}))

    for ty in ("f32", "bf16"):
        fwd, bwd = getattr(L, "talos_gqa_fwd_" + ty), getattr(L, "talos_gqa_bwd_" + ty)
        base = [P16, 64, P16, 32, P16, 32, P16, 64, P16]  # q, k, v, o with their strides, lse
        grads = [P16, 64, P16, 64, P16, 32, P16, 32]

        def both(code, c, args=base, bias=P16):
            assert fwd(c, None, None, bias, *args, None) == code
            assert bwd(c, None, None, bias, *args, *grads, 0.0, P16 if bias else None, None) == code

        both(th.ERR_NULL, None)
        both(th.ERR_SHAPE, cfg(batch=-1))
        both(th.ERR_SHAPE, cfg(q_len=-1))
        both(th.ERR_SHAPE, cfg(heads=0))
        both(th.ERR_SHAPE, cfg(kv_heads=3))
        both(th.ERR_SHAPE, cfg(qk_dim=0))
        both(th.ERR_UNSUPPORTED, cfg(qk_dim=129))
        both(th.ERR_UNSUPPORTED, cfg(v_dim=160))
        both(th.ERR_DTYPE, cfg(causal=2))
        for scale in (0.0, -1.0, math.inf, math.nan):
            both(th.ERR_SHAPE, cfg(scale=scale))
        both(th.ERR_SHAPE, cfg(max_distance=0))
        both(th.ERR_UNSUPPORTED, cfg(scale=1e-31))
        both(th.ERR_UNSUPPORTED, cfg(scale=2e30))
        assert fwd(cfg(max_distance=(1 << 20) + 1), None, None, P16, *base, None) == th.ERR_SHAPE
        both(th.ERR_UNSUPPORTED, cfg(q_len=1 << 29))
        both(th.ERR_UNSUPPORTED, cfg(batch=1 << 29))
        for i in (1, 3, 5, 7):
            both(th.ERR_SHAPE, cfg(), base[:i] + [base[i] - 1] + base[i + 1:])
        for i in (0, 2, 4, 6, 8):
            both(th.ERR_NULL, cfg(), base[:i] + [None] + base[i + 1:])
        for i in (0, 2, 4, 6):
            args = grads[:i] + [None] + grads[i + 1:]
            assert bwd(cfg(), None, None, P16, *base, *args, 0.0, P16, None) == th.ERR_NULL
            args = grads[:i + 1] + [grads[i + 1] - 1] + grads[i + 2:]
            assert bwd(cfg(), None, None, P16, *base, *args, 0.0, P16, None) == th.ERR_SHAPE
        assert bwd(cfg(), None, None, None, *base, *grads, 0.0, P16, None) == th.ERR_NULL  # dbias without bias
        assert bwd(cfg(), None, None, P16, *base, *grads, 0.5, P16, None) == th.ERR_UNSUPPORTED
        assert bwd(cfg(max_distance=513), None, None, P16, *base, *grads, 0.0, P16, None) == th.ERR_UNSUPPORTED
