"""Layer norm, the relative position bias by buckets and the clipped policy loss, against their plain float64 forms: odd
widths, unaligned rows, bf16 and fp32, accumulation, padding rows, refusals."""
import ctypes
import math

import numpy as np
import pytest
import torch

import operators_ref as ref
import talos_hip as th
from operators_ref import float32_default  # noqa: F401

P16 = ctypes.c_void_p(16)  # never dereferenced: the arguments' checks fail first
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def dev(t, offset=0):
    """A copy on the GPU whose storage starts `offset` elements into a buffer (an unaligned tensor)."""
    buf = torch.empty(t.numel() + offset + 8, dtype=t.dtype, device="cuda")
    out = buf[offset:offset + t.numel()].view(t.shape)
    out.copy_(t)
    return out


def p(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------------------- layer norm

def norm_inputs(rows, dim, ty, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, dim, generator=g) * 1.5 + torch.randn(rows, 1, generator=g)).to(DT[ty])
    dy = torch.randn(rows, dim, generator=g).to(DT[ty])
    w, b = 1 + 0.2 * torch.randn(dim, generator=g), 0.3 * torch.randn(dim, generator=g)
    return x, dy, w, b


# widths: one, below a piece, each count of lanes and pieces with its edges, odd ones, past the register kernels
WIDTHS = [1, 3, 8, 31, 32, 33, 64, 65, 127, 128, 200, 256, 257, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 3000, 4096,
          4097, 8192, 8193, 10007]


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("dim", WIDTHS)
def test_layernorm(dim, ty):
    rows, eps, rounds = (37 if dim < 3000 else 9), 1e-5, (1 if ty == "bf16" else 0)
    for offset, beta in ((0, 0.0), (1, 1.0)):  # the second at an unaligned address, gradients accumulated
        x, dy, w, b = norm_inputs(rows, dim, ty, dim + offset)
        y, mean, rstd, dx, dw, db = ref.layernorm(x.double(), w.double(), b.double(), dy.double(), eps)
        X, DY, W, B = dev(x, offset), dev(dy, offset), dev(w, offset), dev(b, offset)
        Y, DX = torch.full_like(X, 7.0), dev(torch.ones_like(x), offset)
        M, R = (torch.empty(rows, device="cuda") for _ in range(2))
        DW, DB = (torch.full((dim,), 2.0, device="cuda") for _ in range(2))
        th.call("talos_layernorm_fwd_" + ty, rows, dim, eps, p(X), p(W), p(B), p(Y), p(M), p(R), None)
        th.call("talos_layernorm_bwd_" + ty, rows, dim, p(X), p(W), p(M), p(R), p(DY), beta, p(DX), beta, p(DW), p(DB),
                None)
        size = x.double().abs().mean(1)
        xa = (x.double().abs() + size[:, None]) * rstd[:, None]  # magnitude of what xh is formed from
        ref.close(M.cpu(), mean, size, name="mean")
        ref.close(R.cpu(), rstd, rstd * (1 + size * rstd), name="rstd")
        ref.close(Y.cpu(), y, xa * w.double().abs() + b.double().abs(), rounds, name="y")
        h = (dy * w).double().abs()
        xm = (h * xa).mean(1, keepdim=True)
        ref.close(DX.cpu(), dx + beta, rstd[:, None] * (h + h.mean(1, keepdim=True) + xa * xm) + beta, rounds, "dx")
        ref.close(DW.cpu(), dw + 2 * beta, (dy.double().abs() * xa).sum(0) + 2, name="dw")
        ref.close(DB.cpu(), db + 2 * beta, dy.double().abs().sum(0) + 2, name="db")


@pytest.mark.gpu
def test_layernorm_many_rows_and_optional_arguments():
    rows, dim = 40000, 24  # more rows than the backward's workgroups take at once
    x, dy, w, b = norm_inputs(rows, dim, "f32", 1)
    y, mean, rstd, dx, dw, db = ref.layernorm(x.double(), w.double(), 0.0, dy.double(), 0.0)
    X, DY, W = dev(x), dev(dy), dev(w)
    Y, M, R = torch.empty_like(X), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    DB = torch.empty(dim, device="cuda")
    th.call("talos_layernorm_fwd_f32", rows, dim, 0.0, p(X), p(W), None, p(Y), p(M), p(R), None)
    xa = (x.double().abs() + x.double().abs().mean(1, keepdim=True)) * rstd[:, None]
    ref.close(Y.cpu(), y, xa * w.double().abs(), name="y")
    first = None
    for _ in range(2):  # dx over dy's own buffer; the same bits twice
        G = dev(dy)
        th.call("talos_layernorm_bwd_f32", rows, dim, p(X), p(W), p(M), p(R), p(G), 0.0, p(G), 0.0, None, p(DB), None)
        h = (dy * w).double().abs()
        bound = rstd[:, None] * (h + h.mean(1, keepdim=True) + xa * (h * xa).mean(1, keepdim=True))
        ref.close(G.cpu(), dx, bound, name="dx")
        ref.close(DB.cpu(), db, dy.double().abs().sum(0), name="db")
        assert first is None or torch.equal(first[0], G) and torch.equal(first[1], DB)
        first = (G, DB.clone())
    th.call("talos_layernorm_fwd_f32", rows, dim, 0.0, p(X), p(W), None, p(X), None, None, None)  # in place
    assert torch.equal(X, Y)
    th.call("talos_layernorm_bwd_f32", 0, dim, p(X), p(W), p(M), p(R), p(DY), 0.0, p(DY), 0.0, p(DB), p(DB), None)
    assert not DB.any()  # no rows: the sums are zero


@pytest.mark.gpu
def test_layernorm_gradient_against_differences():
    x, dy, w, b = norm_inputs(3, 20, "f32", 5)
    X, W, B, DY = (dev(t) for t in (x, w, b, dy))
    M, R, DX, Y = torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty_like(X), torch.empty_like(X)
    th.call("talos_layernorm_fwd_f32", 3, 20, 1e-5, p(X), p(W), p(B), p(Y), p(M), p(R), None)
    th.call("talos_layernorm_bwd_f32", 3, 20, p(X), p(W), p(M), p(R), p(DY), 0.0, p(DX), 0.0, None, None, None)
    h = 1e-5
    for i in range(0, 60, 7):
        step = torch.zeros(60, dtype=torch.float64)
        step[i] = h
        step = step.view(3, 20)
        f = [(ref.layernorm(x.double() + s * step, w.double(), b.double(), dy.double(), 1e-5)[0] * dy.double()).sum()
             for s in (1, -1)]
        # central difference: h^2 of the third derivative (of order 10) and 2^-53 of a sum of order 50 over h
        assert abs(float((f[0] - f[1]) / (2 * h)) - float(DX.view(-1)[i])) < 1e-5


def test_layernorm_refusals():
    L = th.lib()
    for ty in ("f32", "bf16"):
        fwd, bwd = getattr(L, "talos_layernorm_fwd_" + ty), getattr(L, "talos_layernorm_bwd_" + ty)
        assert fwd(4, 8, 1e-5, None, P16, P16, P16, P16, P16, None) == th.ERR_NULL
        assert fwd(4, 8, 1e-5, P16, None, P16, P16, P16, P16, None) == th.ERR_NULL
        assert fwd(-1, 8, 1e-5, P16, P16, P16, P16, P16, P16, None) == th.ERR_SHAPE
        assert fwd(4, 0, 1e-5, P16, P16, P16, P16, P16, P16, None) == th.ERR_SHAPE
        assert fwd(4, 8, -1.0, P16, P16, P16, P16, P16, P16, None) == th.ERR_SHAPE
        assert fwd(1, (1 << 26) + 1, 1e-5, P16, P16, P16, P16, P16, P16, None) == th.ERR_UNSUPPORTED
        assert bwd(4, 8, P16, P16, None, P16, P16, 0.0, P16, 0.0, P16, P16, None) == th.ERR_NULL
        assert bwd(4, 8, P16, P16, P16, P16, P16, 0.5, P16, 0.0, P16, P16, None) == th.ERR_UNSUPPORTED
        assert bwd(4, 8, P16, P16, P16, P16, P16, 0.0, P16, 2.0, P16, P16, None) == th.ERR_UNSUPPORTED
        assert bwd(4, -8, P16, P16, P16, P16, P16, 0.0, P16, 0.0, P16, P16, None) == th.ERR_SHAPE


# ---------------------------------------------------------------------------------------- relative position bias

@pytest.mark.gpu
@pytest.mark.parametrize("buckets,distance,both,heads", [(32, 128, 1, 16), (32, 128, 0, 3), (8, 16, 1, 1), (64, 512, 0, 5),
                                                         (2, 2, 0, 2), (4, 2, 1, 7), (6, 50, 1, 4), (128, 90, 0, 2),
                                                         (10, 4099, 0, 2)])
def test_relpos_bias(buckets, distance, both, heads):
    n = 2 * distance + 1
    g = torch.Generator().manual_seed(buckets)
    table, dbias = torch.randn(buckets, heads, generator=g), torch.randn(heads, n, generator=g)
    want = torch.tensor([ref.bucket(d, buckets, distance, both) for d in range(-distance, distance + 1)])
    T, G = dev(table), dev(dbias)
    bias, idx = torch.empty(heads, n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    th.call("talos_relpos_bias_fwd_f32", buckets, heads, distance, both, p(T), p(bias), p(idx), None)
    assert torch.equal(idx.cpu().long(), want)
    assert torch.equal(bias.cpu(), table[want].t())
    th.call("talos_relpos_bias_fwd_f32", buckets, heads, distance, both, p(T), p(bias), None, None)
    sums = torch.zeros(buckets, heads, dtype=torch.float64).index_add_(0, want, dbias.double().t())
    D = torch.full((buckets, heads), 3.0, device="cuda")
    for beta in (0.0, 1.0):
        th.call("talos_relpos_bias_bwd_f32", buckets, heads, distance, both, p(G), beta, p(D), None)
        # f64 sums, rounded once a call; a bucket that no distance has gets 0
        ref.close(D.cpu(), sums * (1 + beta), torch.zeros(()), name="dtable")


def test_relpos_refusals():
    fwd, bwd = th.lib().talos_relpos_bias_fwd_f32, th.lib().talos_relpos_bias_bwd_f32
    assert fwd(32, 4, 128, 1, None, P16, P16, None) == th.ERR_NULL
    assert fwd(32, 4, 128, 2, P16, P16, P16, None) == th.ERR_DTYPE
    assert fwd(31, 4, 128, 1, P16, P16, P16, None) == th.ERR_SHAPE  # an odd number for two directions
    assert fwd(1, 4, 128, 0, P16, P16, P16, None) == th.ERR_SHAPE
    assert fwd(32, 4, 16, 0, P16, P16, P16, None) == th.ERR_SHAPE  # max_distance within the exact buckets
    assert fwd(32, 0, 128, 0, P16, P16, P16, None) == th.ERR_SHAPE
    assert fwd(5000, 4, 1 << 19, 0, P16, P16, P16, None) == th.ERR_UNSUPPORTED
    assert fwd(32, 4, (1 << 20) + 1, 0, P16, P16, P16, None) == th.ERR_UNSUPPORTED
    assert bwd(32, 4, 128, 1, P16, 0.5, P16, None) == th.ERR_UNSUPPORTED
    assert bwd(32, 4, 128, 1, P16, 0.0, None, None) == th.ERR_NULL


# ---------------------------------------------------------------------------------------------- policy loss

def loss_inputs(rows, vocab, ty, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g) * 2).to(DT[ty])
    a = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    lp = torch.log_softmax(x.double(), 1).gather(1, a.long()[:, None])[:, 0].float()
    adv = torch.randn(rows, generator=g)
    old, rp = lp + 0.4 * torch.randn(rows, generator=g), lp + 0.4 * torch.randn(rows, generator=g)
    w = torch.where(torch.rand(rows, generator=g) < 0.8, torch.rand(rows, generator=g) / rows, torch.zeros(()))
    return x, a, adv, old, rp, w


def loss_call(ty, x, a, adv, old, rp, w, clip, kl, pad=0, offset=0, in_place=False, grad=True, stats=None, acc=0):
    rows, vocab = x.shape
    ld = vocab + pad
    full = torch.full((rows, ld), math.nan, dtype=x.dtype)
    full[:, :vocab] = x
    X = dev(full, offset)
    D = X if in_place else torch.full((rows, ld), 9.0, dtype=x.dtype, device="cuda")
    loss, logp = torch.empty(1, device="cuda"), torch.empty(rows, device="cuda")
    S = torch.zeros(5, dtype=torch.float64, device="cuda") if stats is None else stats
    A, V, O = dev(a), dev(adv), dev(old)
    R, W = None if rp is None else dev(rp), None if w is None else dev(w)
    head = [rows, vocab, *clip, kl, p(X), ld, p(A), p(V), p(O), p(R), p(W)]
    if grad:
        th.call("talos_policy_loss_bwd_" + ty, *head, p(D), ld, p(loss), p(logp), p(S), acc, None)
    else:
        th.call("talos_policy_loss_fwd_" + ty, *head, p(loss), p(logp), p(S), acc, None)
    torch.cuda.synchronize()
    return loss.cpu(), logp.cpu(), D.cpu(), S.cpu()


def loss_check(ty, x, a, adv, old, rp, w, clip, kl, got, grad=True):
    loss, logp, d, stats = ref.policy_loss(x.double(), a, adv.double(), old.double(), None if rp is None else rp.double(),
                                           None if w is None else w.double(), *clip, kl)
    # a log-probability is off by the exponentials' sum (a few u in all, the arguments' rounding u |x - max| of the
    # terms that count) and its own rounding; the other scalars follow it in f64
    ww = torch.full((x.shape[0],), 1 / x.shape[0], dtype=torch.float64) if w is None else w.double()
    ref.close(got[1], logp, torch.ones(()), name="logp")
    rel = 2.0 * (1 + kl) * ww * torch.exp((logp - old.double()).clamp(max=3)) * (1 + adv.double().abs()) + 4 * kl * ww
    ref.close(got[0], torch.tensor([loss]), rel.nansum(), name="loss")
    if grad:
        vocab = x.shape[1]
        soft = torch.softmax(x.double(), 1)
        hot = torch.zeros_like(soft)
        ok = (a >= 0) & (a < vocab)
        hot[ok, a[ok].long()] = 1.0
        rounds = 1 if ty == "bf16" else 0
        ref.close(got[2][:, :vocab], d, (soft + hot).nan_to_num() * rel.nan_to_num()[:, None], rounds, name="dlogits")
    ref.close(got[3], torch.tensor(stats, dtype=torch.float64), torch.tensor([4.0 * x.shape[0]] * 5), name="stats")


VOCABS = [1, 2, 5, 31, 32, 33, 63, 65, 255, 256, 257, 1000, 1025, 4099, 8192, 8193, 16385, 32768, 40001, 65536, 65537,
          131073, 140001]


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_policy_loss(vocab, ty):
    rows = 70 if vocab < 100 else 9
    clip, kl = (0.2, 0.3), 0.05
    args = loss_inputs(rows, vocab, ty, vocab)
    got = loss_call(ty, *args, clip, kl)
    loss_check(ty, *args, clip, kl, got)
    # rows apart and unaligned; padding columns stay as they were; no weights, no KL term
    x, a, adv, old, _, _ = args
    wide = loss_call(ty, x, a, adv, old, None, None, clip, 0.0, pad=3, offset=1)
    loss_check(ty, x, a, adv, old, None, None, clip, 0.0, wide)
    assert (wide[2][:, vocab:] == 9.0).all()
    # in place, and the forward alone: the same bits
    again = loss_call(ty, *args, clip, kl, in_place=True)
    alone = loss_call(ty, *args, clip, kl, grad=False)
    for one in (again, alone):
        assert torch.equal(one[0], got[0]) and torch.equal(one[1], got[1]) and torch.equal(one[3], got[3])
    assert torch.equal(again[2], got[2])


@pytest.mark.gpu
@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [7, 300, 5000, 70000])
def test_policy_loss_masks_and_padding(vocab, ty):
    """Actions that cannot be taken (-infinity), rows of padding full of NaN, every branch of the clip."""
    rows = 24
    x, a, adv, old, rp, w = loss_inputs(rows, vocab, ty, 3)
    w = torch.full((rows,), 0.25)
    for t in range(rows):
        x[t, (int(a[t]) + 1 + t) % vocab] = -math.inf
    x = torch.where(torch.nn.functional.one_hot(a.long(), vocab).bool(), torch.ones((), dtype=x.dtype), x)
    lp = torch.log_softmax(x.double(), 1).gather(1, a.long()[:, None])[:, 0].float()
    old = lp - torch.tensor([0.5, -0.5, 0.05, -0.05] * 6)  # above, below, inside the clip
    adv = torch.tensor([1.5] * 8 + [-0.7] * 8 + [0.0] * 8)
    w[5] = w[16] = 0.0
    clean = x.clone()
    x[5], x[16, 0], adv[5], old[16] = math.nan, math.inf, math.nan, math.inf
    clean[5] = 0
    clean[16] = 0
    got = loss_call(ty, x, a, adv, old, rp, w, (0.2, 0.2), 0.1)
    loss_check(ty, clean, a, torch.nan_to_num(adv), torch.nan_to_num(old, posinf=0.0), rp, w, (0.2, 0.2), 0.1, got)
    assert not got[2][5].any() and not got[2][16].any() and got[1][5] == 0


@pytest.mark.gpu
def test_policy_loss_bad_actions_statistics_and_no_rows():
    x, a, adv, old, rp, w = loss_inputs(6, 11, "f32", 9)
    a[2], a[4] = 11, -1
    w = torch.ones(6)
    got = loss_call("f32", x, a, adv, old, rp, w, (0.2, 0.2), 0.1)
    loss_check("f32", x, a, adv, old, rp, w, (0.2, 0.2), 0.1, got)
    assert math.isnan(got[0]) and not got[2][2].any() and not got[2][4].any()
    ok = loss_inputs(6, 11, "f32", 10)
    S = torch.zeros(5, dtype=torch.float64, device="cuda")
    once = loss_call("f32", *ok, (0.2, 0.2), 0.1, stats=S)[3].clone()
    twice = loss_call("f32", *ok, (0.2, 0.2), 0.1, stats=S, acc=1)[3]
    assert torch.equal(twice, 2 * once)
    loss = torch.full((1,), 5.0, device="cuda")
    th.call("talos_policy_loss_fwd_f32", 0, 11, 0.2, 0.2, 0.0, None, 11, None, None, None, None, None, p(loss), None, p(S),
            0, None)
    assert loss.item() == 0.0 and not S.any()


def test_policy_loss_refusals():
    L = th.lib()
    for ty in ("f32", "bf16"):
        fwd, bwd = getattr(L, "talos_policy_loss_fwd_" + ty), getattr(L, "talos_policy_loss_bwd_" + ty)
        ins = [P16, P16, P16, P16, P16]
        assert fwd(4, 8, 0.2, 0.2, 0.1, P16, 8, *ins, None, None, None, 0, None) == th.ERR_NULL
        assert fwd(4, 8, 0.2, 0.2, 0.1, P16, 7, *ins, P16, None, None, 0, None) == th.ERR_SHAPE
        assert fwd(4, 0, 0.2, 0.2, 0.1, P16, 8, *ins, P16, None, None, 0, None) == th.ERR_SHAPE
        assert fwd(-4, 8, 0.2, 0.2, 0.1, P16, 8, *ins, P16, None, None, 0, None) == th.ERR_SHAPE
        assert fwd(4, 8, -0.2, 0.2, 0.1, P16, 8, *ins, P16, None, None, 0, None) == th.ERR_SHAPE
        assert fwd(4, 8, 0.2, 0.2, 0.1, P16, 8, *ins, P16, None, None, 2, None) == th.ERR_SHAPE
        assert fwd(4, 8, 0.2, 0.2, 0.1, None, 8, *ins, P16, None, None, 0, None) == th.ERR_NULL
        assert fwd(4, 8, 0.2, 0.2, 0.1, P16, 8, P16, P16, P16, None, P16, P16, None, None, 0, None) == th.ERR_NULL
        assert fwd(4, (1 << 26) + 1, 0.2, 0.2, 0.1, P16, 1 << 27, *ins, P16, None, None, 0, None) == th.ERR_UNSUPPORTED
        assert bwd(4, 8, 0.2, 0.2, 0.1, P16, 8, *ins, None, 8, P16, None, None, 0, None) == th.ERR_NULL
        assert bwd(4, 8, 0.2, 0.2, 0.1, P16, 8, *ins, P16, 5, P16, None, None, 0, None) == th.ERR_SHAPE
        assert bwd(4, 8, 0.2, 0.2, 0.1, P16, 12, *ins, P16, 8, P16, None, None, 0, None) == th.ERR_SHAPE  # in place, rows apart
