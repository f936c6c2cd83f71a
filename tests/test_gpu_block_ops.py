"""Attention, rotary positions and layer norm of ``ops`` against 64-bit definitions, element by element (marked gpu).

Every tolerance is a bound worked out from the roundings the kernels make, evaluated in 64 bits from the same inputs:
u is half a step of the tensors' type (finfo.eps / 2), E the relative error of what is summed or exponentiated in fp32.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from crack_detection_federatedlearning_grpc_amd import ops  # noqa: E402

DEV = torch.device("cuda")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Largest error of a rounding below the type's normal range (half the smallest step)."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol everywhere, NaN nowhere."""
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "worst",
                           float((err / tol.clamp_min(1e-300)).nan_to_num(nan=math.inf).max()),
                           "first at", bad.nonzero()[0].tolist())


def rnd(shape, dt, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dt).to(DEV)


# ------------------------------------------------------------------------------------------------------ attention
def allowed(B, Hq, Sq, Sk, mask=None, lengths=None, causal=False):
    ok = torch.ones(B, Hq, Sq, Sk, dtype=torch.bool, device=DEV)
    if mask is not None:
        ok = ok & mask
    if lengths is not None:
        ok = ok & (torch.arange(Sk, device=DEV) < lengths[:, None])[:, None, None]
    if causal:
        ok = ok & (torch.arange(Sk, device=DEV) <= torch.arange(Sq, device=DEV)[:, None] + Sk - Sq)
    return ok


class Exact:
    """The definition in 64 bits, and the bound of each output's error."""

    def __init__(self, q, k, v, go, ok, scale=None):
        dt, (B, Sq, Hq, D), (Sk, Hkv) = q.dtype, q.shape, k.shape[1:3]
        G = Hq // Hkv
        c = 1 / math.sqrt(D) if scale is None else scale
        u, t = half_step(dt), tiny(dt)

        def heads(x, rep):
            return x.double().transpose(1, 2).repeat_interleave(rep, 1)

        def clean(x, used):                       # what no query may attend (no key is attended by) has no effect
            return torch.where(used[..., None], x, torch.zeros_like(x))

        Q, K, V = clean(heads(q, 1), ok.any(3)), clean(heads(k, G), ok.any(2)), clean(heads(v, G), ok.any(2))
        s = (Q @ K.transpose(2, 3) * c).masked_fill(~ok, -math.inf)
        lse = torch.logsumexp(s, 3) if Sk else torch.full((B, Hq, Sq), -math.inf, device=DEV, dtype=torch.float64)
        p = torch.exp(s - lse.nan_to_num(neginf=0.0)[..., None])
        o = p @ V
        # fp32: a score is a sum of D products (D roundings), scaled, less the maximum or lse2 (both below 2^7 in
        # magnitude here, one rounding each); exp2's own error is within 2 steps; a row's sum has at most Sk roundings
        sabs = (Q.abs() @ K.abs().transpose(2, 3)).amax() * c if Sk else torch.zeros((), device=DEV)
        E = float(U32 * ((D + 4) * sabs + 2 * 128 + 8 + Sk))
        E = math.expm1(E)
        # P is rounded to the type (u, or t below its normal range), the output once more
        Ao = p @ V.abs()
        self.out = o.transpose(1, 2)
        self.out_tol = ((2 * u + u * u + 2 * E) * Ao + t * (ok.double() @ V.abs()) + t).transpose(1, 2)
        self.lse = lse
        self.lse_tol = E * (1 + lse.abs().nan_to_num(posinf=0.0))
        if go is None:
            return
        g = clean(heads(go, 1), ok.any(3))
        dp = g @ V.transpose(2, 3)
        dl = (g * o).sum(3, keepdim=True)
        ds = p * (dp - dl)
        # delta is taken from the rounded output; dp and delta are sums of D products; dS is rounded to the type
        e_dl = ((g.abs() * self.out_tol.transpose(1, 2)).sum(3, keepdim=True) + (D + 2) * U32 * (g * o).abs().sum(3, keepdim=True))
        e_dp = (D + 2) * U32 * (g.abs() @ V.abs().transpose(2, 3))
        e_ds = (u + 2 * E) * ds.abs() + p * (1 + 2 * E) * (e_dl + e_dp) * (1 + u) + t * ok
        n = Sk + G * Sq                           # roundings of the longest fp32 sum

        def out(x, tol, mag):
            return x, tol + (u * 1.001 + n * U32) * mag + u * tol + t

        def shared(x):                            # sum over the heads that share a key head
            return x.unflatten(1, (Hkv, G)).sum(2).transpose(1, 2)

        self.dq, self.dq_tol = out((ds @ K * c).transpose(1, 2), (e_ds @ K.abs() * c).transpose(1, 2),
                                   ((ds.abs() + e_ds) @ K.abs() * c).transpose(1, 2))
        dsT, e_dsT, pT = ds.transpose(2, 3), e_ds.transpose(2, 3), p.transpose(2, 3)
        self.dk, self.dk_tol = out(shared(dsT @ Q * c), shared(e_dsT @ Q.abs() * c),
                                   shared((dsT.abs() + e_dsT) @ Q.abs() * c))
        self.dv, self.dv_tol = out(shared(pT @ g), shared(((u + 2 * E) * pT + t * ok.transpose(2, 3)) @ g.abs()),
                                   shared(pT @ g.abs()))
        # the last rounding is relative to the result, the fp32 sums' to the terms
        for n_, x in (("dq", self.dq), ("dk", self.dk), ("dv", self.dv)):
            assert torch.isfinite(x).all(), n_


def check_attention(q, k, v, go, mask=None, lengths=None, causal=False, scale=None, call=None):
    B, Sq, Hq, _ = q.shape
    ok = allowed(B, Hq, Sq, k.shape[1], mask, lengths, causal)
    ex = Exact(q, k, v, go, ok, scale)
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    out, lse = ops.attention(q, k, v, mask, lengths, causal, scale, return_lse=True)
    close(out, ex.out, ex.out_tol, "out")
    none = ex.lse == -math.inf
    assert torch.equal(none, lse == -math.inf)
    close(lse.masked_fill(none, 0), ex.lse.masked_fill(none, 0), ex.lse_tol, "lse")
    assert not out.transpose(1, 2)[none].any()
    # without a gradient the same call takes no lse: the same output, bit for bit
    with torch.no_grad():
        assert torch.equal(ops.attention(q, k, v, mask, lengths, causal, scale), out)
    if go is None:
        return
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), go)
    close(dq, ex.dq, ex.dq_tol, "dq")
    close(dk, ex.dk, ex.dk_tol, "dk")
    close(dv, ex.dv, ex.dv_tol, "dv")
    assert not dq.transpose(1, 2)[none].any()


def qkvg(B, Sq, Sk, Hq, Hkv, D, dt, seed=0):
    return (rnd((B, Sq, Hq, D), dt, seed), rnd((B, Sk, Hkv, D), dt, seed + 1), rnd((B, Sk, Hkv, D), dt, seed + 2),
            rnd((B, Sq, Hq, D), dt, seed + 3))


SHAPES = [  # B, Sq, Sk, Hq, Hkv, D: one token and one key, tile borders, odd lengths, shared heads, every channel tile
    (1, 1, 1, 1, 1, 8), (2, 1, 300, 4, 4, 32), (1, 1, 1537, 8, 2, 128), (3, 5, 64, 6, 2, 64), (1, 33, 65, 1, 1, 24),
    (2, 64, 64, 2, 2, 32), (1, 127, 129, 3, 1, 80), (2, 200, 96, 4, 2, 96), (1, 256, 256, 2, 2, 128),
    (1, 40, 1000, 2, 1, 40), (2, 300, 7, 2, 2, 112), (1, 513, 640, 5, 5, 64)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_matches_definition(shape, causal, dt):
    check_attention(*qkvg(*shape, dt), causal=causal)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["plain", "causal", "mask", "lengths"])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
def test_attention_many_blocks(D, kind, dt):
    """Enough (image, head)s for the blocks of 128 rows and 128 keys that large calls take."""
    B, Hq, Hkv, Sq, Sk = 20, 28, 28, 140, 150
    g = torch.Generator().manual_seed(17)
    kw = {}
    if kind == "mask":
        kw["mask"] = (torch.rand(1, 1, Sq, Sk, generator=g) < 0.5).to(DEV)
    elif kind == "lengths":
        kw["lengths"] = torch.randint(0, Sk + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
    check_attention(*qkvg(B, Sq, Sk, Hq, Hkv, D, dt), causal=kind == "causal", **kw)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", [(4, 70, 70, 4, 2, 64), (4, 1, 700, 4, 4, 32), (4, 150, 260, 2, 2, 128)])
def test_attention_lengths(shape, causal, dt):
    """Images of different sizes in one batch: none, one, some and all of the keys, and values past the ends."""
    Sk = shape[2]
    lengths = torch.tensor([0, 1, Sk - 6, Sk], dtype=torch.int32, device=DEV)
    check_attention(*qkvg(*shape, dt), lengths=lengths, causal=causal)
    q, k, v, _ = qkvg(*shape, dt)
    wild = torch.tensor([-5, 1, Sk - 6, Sk + 1000], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.attention(q, k, v, lengths=wild), ops.attention(q, k, v, lengths=lengths))


MASKS = {
    "keys": lambda B, H, Sq, Sk, r: r(B, 1, 1, Sk) < 0.6,
    "pairs": lambda B, H, Sq, Sk, r: r(1, 1, Sq, Sk) < 0.5,
    "all axes": lambda B, H, Sq, Sk, r: r(B, H, Sq, Sk) < 0.3,
    "heads": lambda B, H, Sq, Sk, r: r(H, 1, Sk) < 0.5,
    "queries": lambda B, H, Sq, Sk, r: r(B, 1, Sq, 1) < 0.5,
    "transposed": lambda B, H, Sq, Sk, r: (r(Sk, Sq) < 0.5).T,
    "sliced": lambda B, H, Sq, Sk, r: (r(B, 1, Sq, 2 * Sk + 3) < 0.5)[..., 3::2],
    "band": lambda B, H, Sq, Sk, r: (torch.arange(Sq)[:, None] - torch.arange(Sk)).abs() <= 20,
    "blocks": lambda B, H, Sq, Sk, r: torch.arange(Sq)[:, None] // 64 == torch.arange(Sk) // 64,
    "none": lambda B, H, Sq, Sk, r: torch.zeros(1, dtype=torch.bool),
    "every": lambda B, H, Sq, Sk, r: torch.ones(Sq, Sk, dtype=torch.bool),
}


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(2, 100, 100, 4, 2, 64), (2, 1, 400, 3, 3, 32), (1, 290, 330, 3, 1, 128)])
@pytest.mark.parametrize("name", list(MASKS))
def test_attention_masks(name, shape, dt):
    B, Sq, Sk, Hq = shape[:4]
    g = torch.Generator().manual_seed(11)
    mask = MASKS[name](B, Hq, Sq, Sk, lambda *n: torch.rand(n, generator=g)).to(DEV)
    check_attention(*qkvg(*shape, dt), mask=mask)


def test_attention_mask_lengths_and_causal_together():
    shape = (3, 180, 200, 4, 2, 64)
    g = torch.Generator().manual_seed(3)
    mask = (torch.rand(3, 4, 180, 200, generator=g) < 0.5).to(DEV)
    lengths = torch.tensor([200, 77, 0], dtype=torch.int32, device=DEV)
    check_attention(*qkvg(*shape, BF), mask=mask, lengths=lengths, causal=True)


@pytest.mark.parametrize("scale", [1e-3, 1.0])
def test_attention_scale(scale):
    check_attention(*qkvg(1, 90, 110, 2, 2, 32, BF), scale=scale)


@pytest.mark.parametrize("kv", [1, 2, 4])
def test_attention_qkv_is_attention_of_its_parts(kv):
    qkv = rnd((2, 150, 4 + 2 * kv, 64), BF, 5)
    go = rnd((2, 150, 4, 64), BF, 6)
    whole = qkv.clone().requires_grad_()
    out = ops.attention_qkv(whole, 4, kv)
    (d,) = torch.autograd.grad(out, whole, go)
    q, k, v = (t.clone().requires_grad_() for t in qkv.split([4, kv, kv], 2))
    want = ops.attention(q, k, v)
    assert torch.equal(out, want)
    assert torch.equal(d, torch.cat(torch.autograd.grad(want, (q, k, v), go), 2))
    check_attention(*qkv.split([4, kv, kv], 2), go)


def test_attention_strides_and_alignment():
    """Any layout gives what its contiguous copy gives: channels or tokens apart, odd offsets, broadcast inputs."""
    q, k, v, go = qkvg(2, 70, 90, 4, 2, 32, BF)
    want = ops.attention(q, k, v)
    flat = torch.zeros(q.numel() + 1, dtype=BF, device=DEV)
    flat[1:] = q.reshape(-1)
    odd = flat[1:].view(q.shape)
    by_head = k.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 90, 2, 35, dtype=BF, device=DEV)
    wide[..., 3:] = v
    by_channel = go.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    ins = [t.detach().requires_grad_() for t in (odd, by_head, wide[..., 3:])]
    out = ops.attention(*ins)
    assert torch.equal(out, want)
    a = torch.autograd.grad(out, ins, by_channel)
    ref = [t.detach().requires_grad_() for t in (q, k, v)]
    b = torch.autograd.grad(ops.attention(*ref), ref, go)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    one = k[:1].expand(2, -1, -1, -1).detach().requires_grad_()
    check_attention(q, one.detach(), v, go)


def test_attention_gradient_against_differences():
    """d<out, go> along a direction, by central differences of the 64-bit definition, and by the kernels' gradients."""
    q, k, v, go = qkvg(1, 40, 50, 2, 1, 16, HF)
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.attention(*ins), ins, go)
    ok = allowed(1, 2, 40, 50)
    ex = Exact(q, k, v, go, ok)

    def f(*t):
        Q, K, V = (x.transpose(1, 2).repeat_interleave(2 // x.shape[2], 1) for x in t)
        return ((torch.softmax(Q @ K.transpose(2, 3) / 4.0, 3) @ V).transpose(1, 2) * go.double()).sum()

    for n, (g, tol) in enumerate(zip(grads, (ex.dq_tol, ex.dk_tol, ex.dv_tol))):
        x = [t.double() for t in (q, k, v)]
        d = torch.randn(x[n].shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64).to(DEV)
        h = 1e-5
        hi, lo = list(x), list(x)
        hi[n], lo[n] = x[n] + h * d, x[n] - h * d
        want = float((f(*hi) - f(*lo)) / (2 * h))
        got = float((g.double() * d).sum())
        assert abs(got - want) <= float((tol * d.abs()).sum()) + 1e-6 * (1 + abs(want))


def test_attention_is_the_same_every_time():
    q, k, v, go = qkvg(2, 500, 700, 4, 2, 64, BF)
    runs = []
    for _ in range(3):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*ins, causal=True)
        runs.append([out.detach(), *torch.autograd.grad(out, ins, go)])
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)


def test_attention_only_wanted_gradients():
    q, k, v, go = qkvg(1, 70, 80, 2, 2, 32, BF)
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    full = torch.autograd.grad(ops.attention(*ins), ins, go)
    for n in range(3):
        part = [t.detach().requires_grad_(i == n) for i, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(ops.attention(*part), part[n], go)
        assert torch.equal(g, full[n])


def test_attention_empty_tensors():
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q = torch.ones(B, Sq, 2, 16, dtype=BF, device=DEV).requires_grad_()
        k = torch.ones(B, Sk, 2, 16, dtype=BF, device=DEV).requires_grad_()
        out, lse = ops.attention(q, k, k, return_lse=True)
        assert out.shape == q.shape and not out.any() and (lse == -math.inf).all()
        gq, gk = torch.autograd.grad(out.sum(), (q, k))
        assert not gq.any() and not gk.any()


def test_attention_refuses_a_second_derivative():
    q = rnd((1, 4, 1, 16), BF, 0).requires_grad_()
    out = ops.attention(q, q, q)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(out.sum(), q, create_graph=True)


# ----------------------------------------------------------------------------------------------------- layer norm
def check_norm(x, w, b, gy, eps=1e-3):
    dt, C = x.dtype, x.shape[-1]
    u, t = half_step(dt), tiny(dt) if dt != FF else 1e-38
    X, g = x.double().reshape(-1, C), gy.double().reshape(-1, C)
    W = torch.ones(C, dtype=torch.float64, device=DEV) if w is None else w.double()
    mu = X.mean(1, keepdim=True)
    r = 1 / torch.sqrt((X - mu).square().mean(1, keepdim=True) + eps)
    xh = (X - mu) * r
    y = xh * W + (0 if b is None else b.double())
    # fp32: a row's sum is at most 32 terms in a lane and 10 exchanges or wave sums, so a mean is off by 48 roundings of
    # its mean magnitude; x - mu by that and one rounding; r by half of the variance's error: e covers each factor
    e = 64 * U32
    mag = 1 + r * X.abs().mean(1, keepdim=True)
    exh = 2 * e * (1 + xh.abs()) * mag
    ytol = u * y.abs() * 1.001 + exh * W.abs() + 4 * U32 * (y.abs() + W.abs() * xh.abs()) + t
    ins = [v.detach().requires_grad_() for v in (x, w, b) if v is not None]
    names = [n for n, v in (("x", x), ("weight", w), ("bias", b)) if v is not None]
    kw = dict(zip(names, ins))
    out = ops.layer_norm(kw["x"], kw.get("weight"), kw.get("bias"), eps)
    assert out.shape == x.shape and out.dtype == dt and out.is_contiguous()
    close(out.reshape(-1, C), y, ytol, "y")
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps), out)
    grads = dict(zip(names, torch.autograd.grad(out, ins, gy)))
    gw = g * W
    m0, m1 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    dx = r * (gw - m0 - xh * m1)
    terms = gw.abs() + gw.abs().mean(1, keepdim=True) + (1 + xh.abs()) * ((1 + xh.abs()) * gw.abs()).mean(1, keepdim=True)
    close(grads["x"].reshape(-1, C), dx, u * 1.001 * dx.abs() + 4 * e * r * terms * mag + t, "dx")
    rows = X.shape[0]
    n = rows + 32                                    # roundings of a column's sum, at most
    if w is not None:
        assert grads["weight"].dtype == FF
        close(grads["weight"], (g * xh).sum(0), (g.abs() * exh).sum(0) + n * U32 * (g * xh).abs().sum(0) + 1e-38, "dw")
    if b is not None:
        close(grads["bias"], g.sum(0), n * U32 * g.abs().sum(0) + 1e-38, "db")


@pytest.mark.parametrize("dt", [FF, BF, HF])
@pytest.mark.parametrize("rows,C", [(1, 1), (1, 8), (3, 5), (70, 32), (33, 33), (130, 64), (17, 100), (9, 128), (50, 250),
                                    (5, 256), (40, 333), (6, 512), (10, 768), (3, 1024), (7, 1000), (3, 2048), (2, 2050),
                                    (5, 4096), (3, 8192), (2, 8191), (2, 4104), (1100, 1000), (3000, 32), (2100, 320)])
def test_layer_norm_matches_definition(rows, C, dt):
    x = rnd((rows, C), dt, rows + C, 1.5, 0.5)
    check_norm(x, rnd((C,), FF, 1, 0.3, 1.0), rnd((C,), FF, 2, 0.3), rnd((rows, C), dt, 3))


@pytest.mark.parametrize("dt", [FF, BF, HF])
def test_layer_norm_layouts(dt):
    """NHWC maps, channel slices of wider maps (aligned and not), transposed maps, rows broadcast, one axis only."""
    w, b = rnd((32,), FF, 1, 0.3, 1.0), rnd((32,), FF, 2, 0.3)
    maps = rnd((2, 5, 7, 64), dt, 0)
    gy = rnd((2, 5, 7, 32), dt, 4)
    for x in (maps[..., :32].contiguous(), maps[..., 32:], maps[..., 3:35], maps[..., ::2], maps[:, ::2, :, :32],
              maps.permute(0, 2, 1, 3)[..., :32], maps[:1, :, :, :32].expand(2, -1, -1, -1)):
        g = gy[:, :x.shape[1], :x.shape[2]] if x.shape != gy.shape and x.shape[1] <= 5 else \
            rnd(tuple(x.shape), dt, 5)
        check_norm(x, w, b, g)
    check_norm(maps[0, 0, 0, :32], w, b, gy[0, 0, 0])
    check_norm(maps[..., :32], w, b, rnd((2, 5, 7, 33), dt, 6)[..., 1:])


@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(w, b):
    x, gy = rnd((20, 48), BF, 0), rnd((20, 48), BF, 1)
    check_norm(x, rnd((48,), FF, 2) if w else None, rnd((48,), FF, 3) if b else None, gy)


def test_layer_norm_large_mean_and_constant_rows():
    """The variance is of x - mean: a mean a thousand times the spread loses nothing but its own rounding."""
    x = rnd((40, 256), FF, 0, 1.0, 1000.0)
    check_norm(x, None, None, rnd((40, 256), FF, 1))
    for C in (1, 3, 64, 100, 333, 700, 5000):
        for dt in (FF, BF, HF):
            x = torch.full((4, C), 3.25, dtype=dt, device=DEV).requires_grad_()
            y = ops.layer_norm(x)
            assert not y.any()
            # equal gradients: nothing is left of them (a row of one column never keeps any)
            g = rnd((4, 1), dt, C).expand(4, C).contiguous()
            (dx,) = torch.autograd.grad(y, x, g)
            assert C > 1 or not dx.any()
            tol = 64 * U32 * float(g.abs().max()) * math.sqrt(1e3) * 2
            assert float(dx.abs().max()) <= tol


@pytest.mark.parametrize("rows,C", [(3, 32), (70, 33), (130, 256), (1, 1000), (5, 4096), (700, 64)])
def test_layer_norm_without_epsilon(rows, C):
    """eps = 0: no part of the card that holds no row may add to the weights' gradients (0 / 0)."""
    check_norm(rnd((rows, C), BF, 1), rnd((C,), FF, 2), rnd((C,), FF, 3), rnd((rows, C), BF, 4), eps=0.0)


def test_layer_norm_frozen_inputs_and_empty_rows():
    x, w, b = rnd((50, 64), BF, 0), rnd((64,), FF, 1), rnd((64,), FF, 2)
    gy = rnd((50, 64), BF, 3)
    ins = [t.detach().requires_grad_() for t in (x, w, b)]
    full = torch.autograd.grad(ops.layer_norm(*ins), ins, gy)
    for n in range(3):
        part = [t.detach().requires_grad_(i == n) for i, t in enumerate((x, w, b))]
        (g,) = torch.autograd.grad(ops.layer_norm(*part), part[n], gy)
        assert torch.equal(g, full[n])
    none = torch.zeros(0, 64, dtype=BF, device=DEV).requires_grad_()
    ww = w.detach().requires_grad_()
    y = ops.layer_norm(none, ww, b)
    assert y.shape == (0, 64)
    gx, gw = torch.autograd.grad(y.sum(), (none, ww))
    assert gx.shape == (0, 64) and not gw.any()


# --------------------------------------------------------------------------------------------------------- rotary
def exact_rotary(x, pos, dims, theta, joint, inter, sign=1):
    n, B, S = sum(dims), x.shape[0], x.shape[1]
    p = pos.double() if pos.dim() == 3 else pos.double()[:, None]
    ang, i0 = [], 0
    for a, m in enumerate(dims):
        for i in range(m // 2):
            ang.append(p[a] * theta ** (-2.0 * ((i0 + i) / n if joint else i / m)))
        i0 += m // 2
    ang = torch.stack(ang, -1)[:, :, None] * sign                   # (B or 1, S, 1, pairs)
    X = x.double()
    a, b = (X[..., 0:n:2], X[..., 1:n:2]) if inter else (X[..., :n // 2], X[..., n // 2:n])
    c, s = ang.cos(), ang.sin()
    y0, y1 = a * c - b * s, b * c + a * s
    y = torch.stack([y0, y1], -1).flatten(-2) if inter else torch.cat([y0, y1], -1)
    mag = a.abs() + b.abs()
    mag = torch.stack([mag, mag], -1).flatten(-2) if inter else torch.cat([mag, mag], -1)
    # angle: a 64-bit product of the position, off by 4 of its own roundings (exp2 among them); sine and cosine fp32
    # from an eighth of a turn (off by 4 steps of 1); two products and a sum in fp32; the result rounded once
    e = 6 * U32 + 2.0 ** -51 * float(pos.double().abs().max() if pos.numel() else 0)
    tol = half_step(x.dtype) * y.abs() * 1.001 + e * mag + (tiny(x.dtype) if x.dtype != FF else 1e-38)
    return torch.cat([y, X[..., n:]], -1), torch.cat([tol, torch.zeros_like(X[..., n:])], -1)


@pytest.mark.parametrize("dt", [FF, BF, HF])
@pytest.mark.parametrize("joint", [False, True])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,S,H,D,dims", [(1, 1, 1, 2, (2,)), (2, 30, 3, 64, (32, 32)), (1, 77, 5, 128, (32, 48, 48)),
                                          (2, 9, 2, 86, (42, 6, 4)), (1, 50, 4, 40, (8, 0, 24)), (3, 20, 1, 24, (2, 4, 6, 8)),
                                          (1, 300, 9, 32, (16, 16))])
def test_rotary_matches_definition(B, S, H, D, dims, joint, inter, dt):
    g = torch.Generator().manual_seed(S)
    pos = torch.randint(-50, 1 << 20, (len(dims), S), generator=g, dtype=torch.int32).to(DEV)
    x, gy = rnd((B, S, H, D), dt, 0), rnd((B, S, H, D), dt, 1)
    xr = x.detach().requires_grad_()
    y = ops.rotary(xr, pos, dims, joint=joint, interleaved=inter)
    close(y, *exact_rotary(x, pos, dims, 1e4, joint, inter), "y")
    (dx,) = torch.autograd.grad(y, xr, gy)
    close(dx, *exact_rotary(gy, pos, dims, 1e4, joint, inter, -1), "dx")


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_rotary_positions(kind):
    """Positions per image and shared, far ones, fractions, strided, another theta; heads read from a wider tensor."""
    x = rnd((2, 40, 6, 32), FF, 0)
    far = {torch.int32: 1 << 30, torch.int64: 1 << 40, torch.float32: 1000}[kind]
    g = torch.Generator().manual_seed(4)
    pos = (torch.rand(2, 2, 40, generator=g, dtype=torch.float64) * far).to(kind).to(DEV)
    close(ops.rotary(x, pos, (16, 16), theta=500.0), *exact_rotary(x, pos, (16, 16), 500.0, False, False), "batch")
    close(ops.rotary(x, pos[:, :1], (16, 16)), *exact_rotary(x, pos[:, :1], (16, 16), 1e4, False, False), "one row")
    wide = torch.zeros(40, 2, dtype=kind, device=DEV)
    wide.copy_(pos[:, 0].T)
    close(ops.rotary(x, wide.T, (16, 16)), *exact_rotary(x, pos[:, 0], (16, 16), 1e4, False, False), "strided")
    part = x[:, :, 1:4, 2:30]
    close(ops.rotary(part, pos, (12, 8)), *exact_rotary(part, pos, (12, 8), 1e4, False, False), "slice")


def test_grid_positions():
    p = ops.grid_positions(2, 3, 4, device=DEV)
    want = torch.tensor([[t, y, x] for t in range(2) for y in range(3) for x in range(4)], dtype=torch.int32).T
    assert torch.equal(p.cpu(), want) and p.dtype == torch.int32


def test_rotary_keeps_products_of_equal_distance():
    """q.k after the turn depends on the distance of the positions only: far along, as near 0."""
    q, k = rnd((1, 1, 1, 64), FF, 0), rnd((1, 1, 1, 64), FF, 1)

    def dot(i, j):
        a = ops.rotary(q, torch.tensor([[i], [i]], device=DEV), (32, 32))
        b = ops.rotary(k, torch.tensor([[j], [j]], device=DEV), (32, 32))
        return float((a.double() * b.double()).sum())

    bound = 64 * 16 * U32 * float(q.abs().max() * k.abs().max())
    assert abs(dot(5, 2) - dot(5 + 10 ** 8, 2 + 10 ** 8)) <= bound


# ------------------------------------------------------------------------------------------------ the block of them
def block_parts(dt=torch.float64):
    C, heads, kv, D = 64, 4, 2, 32
    g = torch.Generator().manual_seed(21)
    mk = {"norm_weight": torch.randn(C, generator=g) * 0.2 + 1, "norm_bias": torch.randn(C, generator=g) * 0.2,
          "w_qkv": torch.randn(1, 1, C, (heads + 2 * kv) * D, generator=g) * 0.1,
          "w_out": torch.randn(1, 1, heads * D, C, generator=g) * 0.1}
    return C, heads, kv, D, {n: t.to(DEV) for n, t in mk.items()}


def test_self_attention2d_runs_its_layers():
    """The block is its layers in a row, forward and backward, and a padded map's invalid pixels reach no valid one."""
    C, heads, kv, D, w = block_parts()
    B, H, W = 2, 6, 9
    x, gy = rnd((B, H, W, C), BF, 0), rnd((B, H, W, C), BF, 1)
    valid = torch.ones(B, H, W, dtype=torch.bool, device=DEV)
    valid[1, 4:] = False
    valid[1, :, 7:] = False
    mask = valid.view(B, 1, 1, H * W)

    def by_hand(x, w):
        t = ops.conv2d(ops.layer_norm(x, w["norm_weight"], w["norm_bias"]), w["w_qkv"]).view(B, H * W, heads + 2 * kv, D)
        p = ops.grid_positions(H, W, device=DEV)
        q = ops.rotary(t[:, :, :heads], p, (D // 2, D // 2))
        k = ops.rotary(t[:, :, heads:heads + kv], p, (D // 2, D // 2))
        y = ops.attention(q, k, t[:, :, heads + kv:], mask).reshape(B, H, W, heads * D)
        return x + ops.conv2d(y, w["w_out"])

    res = []
    for f in (lambda x, w: ops.self_attention2d(x, heads=heads, kv_heads=kv, mask=mask, **w), by_hand):
        xl = x.detach().requires_grad_()
        wl = {n: t.detach().requires_grad_() for n, t in w.items()}
        y = f(xl, wl)
        res.append([y.detach(), *torch.autograd.grad(y, [xl, *wl.values()], gy)])
    # the same kernels in the same order; the 1x1 convolution's weight gradient is a sum of atomics, whose order varies
    names = ["y", "dx", *w]
    for n, a, b in zip(names, *res):
        if n.startswith("w_"):
            assert float((a - b).norm()) <= 1e-5 * float(b.norm()), n
        else:
            assert torch.equal(a, b), n
    other = x.clone()
    other[~valid] = 3.0
    y2 = ops.self_attention2d(other, heads=heads, kv_heads=kv, mask=mask, **w)
    assert torch.equal(y2[valid], res[0][0][valid])


def test_self_attention2d_gradients_match_64_bits():
    C, heads, kv, D, w = block_parts()
    B, H, W = 2, 8, 8
    x, gy = rnd((B, H, W, C), BF, 0), rnd((B, H, W, C), BF, 1)

    def exact(x, w):
        mu = x.mean(-1, keepdim=True)
        n = (x - mu) / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + 1e-3) * w["norm_weight"] + w["norm_bias"]
        t = (n.view(B, H * W, C) @ w["w_qkv"][0, 0]).view(B, H * W, heads + 2 * kv, D)
        pos = ops.grid_positions(H, W, device=DEV)

        def turn(t):
            i = torch.arange(D // 4, device=DEV, dtype=torch.float64)
            ang = torch.cat([pos[a].double()[:, None] * 1e4 ** (-4 * i / D) for a in range(2)], 1)[None, :, None]
            a, b = t[..., :D // 2], t[..., D // 2:]
            return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)

        q, k, v = turn(t[:, :, :heads]), turn(t[:, :, heads:heads + kv]), t[:, :, heads + kv:]
        q, k, v = (z.transpose(1, 2).repeat_interleave(heads // z.shape[2], 1) for z in (q, k, v))
        o = (torch.softmax(q @ k.transpose(2, 3) / math.sqrt(D), 3) @ v).transpose(1, 2).reshape(B, H * W, heads * D)
        return x + (o @ w["w_out"][0, 0]).view(B, H, W, C)

    out = []
    for f, dt in ((lambda x, w: ops.self_attention2d(x, heads=heads, kv_heads=kv, **w), None), (exact, torch.float64)):
        xl = (x if dt is None else x.to(dt)).detach().requires_grad_()
        wl = {n: (t if dt is None else t.to(dt)).detach().requires_grad_() for n, t in w.items()}
        y = f(xl, wl)
        out.append([y.detach(), *torch.autograd.grad(y, [xl, *wl.values()], gy.to(y.dtype))])
    # Five roundings to bf16 between x and y (norm, qkv, turned, attention, projection) and the weights' (bf16 in the
    # convolutions), as many again on the way back: each relative to its tensor at most u = 2^-8, independent, so the
    # norm of an error is within about sqrt(12) u of the norm of what it is added to; 6 u leaves the products' gain.
    for n, a, b in zip(["y", "dx", *w], *out):
        assert float((a.double() - b).norm()) <= 6 * half_step(BF) * float(b.norm()), n


# ------------------------------------------------------------------------- values that are not finite, where not allowed
BAD = [math.nan, math.inf, -math.inf]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("shape", [(2, 90, 130, 4, 2, 64), (2, 1, 300, 2, 2, 32), (1, 150, 200, 2, 1, 128),
                                   (1, 100, 140, 2, 2, 96)])
@pytest.mark.parametrize("kind", ["keys", "pairs", "lengths"])
def test_attention_ignores_what_is_not_allowed(kind, shape, dt):
    """Keys, values, queries and gradients of tokens that take part in nothing hold NaN and infinities."""
    B, Sq, Sk, Hq, Hkv, D = shape
    q, k, v, go = qkvg(*shape, dt)
    g = torch.Generator().manual_seed(8)
    dead = torch.rand(Sk, generator=g) < 0.4
    dead[0] = False
    kw = {}
    empty = torch.zeros(Sq, dtype=torch.bool)
    if kind == "keys":
        kw["mask"] = (~dead)[None, None, None].expand(B, 1, 1, Sk).contiguous().to(DEV)
    elif kind == "pairs":
        m = (torch.rand(Sq, Sk, generator=g) < 0.6) & ~dead
        if Sq > 3:
            empty[[1, Sq - 1]] = True
        m[empty] = False
        kw["mask"] = m.to(DEV)
    else:
        n = Sk - Sk // 3
        dead = torch.arange(Sk) >= n
        kw["lengths"] = torch.full((B,), n, dtype=torch.int32, device=DEV)
    dead, empty = dead.to(DEV), empty.to(DEV)
    bad = torch.tensor(BAD, dtype=dt, device=DEV)
    k[:, dead] = bad[torch.arange(int(dead.sum()), device=DEV) % 3][None, :, None, None]
    v[:, dead] = bad[(torch.arange(int(dead.sum()), device=DEV) + 1) % 3][None, :, None, None]
    if empty.any():
        q[:, empty] = math.nan
        go[:, empty] = math.inf
    check_attention(q, k, v, go, **kw)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_attention_causal_ignores_the_future(D, dt):
    """A value that is not finite shows in the rows that may attend it, in no earlier one; likewise its key."""
    q, k, v, go = qkvg(1, 150, 150, 2, 2, D, dt)
    want = ops.attention(q, k, v, causal=True)
    for t in (v, k):
        for x in BAD:
            w = t.clone()
            w[0, 100, :, 3] = x
            out = ops.attention(q, w if t is k else k, w if t is v else v, causal=True)
            ok = allowed(1, 2, 150, 150, causal=True)
            assert torch.equal(out[:, :100], want[:, :100])
            if t is v:
                # the one channel, and there the value itself (a NaN stays one)
                hit = out[:, 100:, :, 3].float()
                assert (hit.isnan().all() if math.isnan(x) else (hit == x).all())
                rest = [c for c in range(D) if c != 3]
                assert torch.equal(out[..., rest], want[..., rest])
            else:
                assert not torch.isfinite(out[:, 100:]).all()
    # gradients: an infinite gradient of row 40 reaches the keys up to 40 and no later one
    bad = go.clone()
    bad[0, 40, :, 5] = math.inf
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    a = torch.autograd.grad(ops.attention(*ins, causal=True), ins, go)
    b = torch.autograd.grad(ops.attention(*ins, causal=True), ins, bad)
    for n in (1, 2):
        assert torch.equal(a[n][:, 41:], b[n][:, 41:])
    assert (b[2][:, :41, :, 5] == math.inf).all()
    assert torch.equal(a[2][..., :5], b[2][..., :5])
    keep = [i for i in range(150) if i != 40]
    assert torch.equal(a[0][:, keep], b[0][:, keep])


def test_attention_masked_rows_hear_nothing_of_a_bad_value():
    """A dense mask: NaN in one value shows in the rows that attend it only."""
    q, k, v, _ = qkvg(2, 130, 170, 2, 2, 64, BF)
    g = torch.Generator().manual_seed(5)
    mask = torch.rand(130, 170, generator=g) < 0.5
    mask[:, 0] = True
    want = ops.attention(q, k, v, mask=mask.to(DEV))
    v[:, 77] = math.nan
    out = ops.attention(q, k, v, mask=mask.to(DEV))
    hit = mask[:, 77].to(DEV)
    assert out[:, hit].isnan().all()
    assert torch.equal(out[:, ~hit], want[:, ~hit])


def test_attention_infinite_gradient_is_not_lost():
    """Overflow of a scaled loss: an infinite gradient must reach every gradient that depends on it."""
    q, k, v, go = qkvg(1, 70, 90, 2, 2, 64, HF)
    go[0, 30, 1] = math.inf
    for kw in ({}, {"causal": True}, {"mask": torch.ones(70, 90, dtype=torch.bool, device=DEV)}):
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        dq, dk, dv = torch.autograd.grad(ops.attention(*ins, **kw), ins, go)
        assert not torch.isfinite(dq[0, 30, 1]).any()
        assert not torch.isfinite(dv[0, :40, 1]).any()
        assert not torch.isfinite(dk[0, :40, 1]).any()
        assert torch.isfinite(dv[0, :, 0]).all() and torch.isfinite(dk[0, :, 0]).all()


# --------------------------------------------------------------------------------------------- streams, graphs, reuse
def test_ops_run_on_the_current_stream():
    x, w = rnd((4096, 256), BF, 0), rnd((256,), FF, 1)
    q, k, v, go = qkvg(2, 300, 300, 4, 4, 64, BF)
    pos = ops.grid_positions(15, 20, device=DEV)
    mask = (torch.rand(300, 300, generator=torch.Generator().manual_seed(1)) < 0.5).to(DEV)

    def run():
        ins = [t.detach().requires_grad_() for t in (q, k, v, x, w)]
        a = ops.attention(ops.rotary(ins[0], pos, (32, 32)), ops.rotary(ins[1], pos, (32, 32)), ins[2], mask)
        b = ops.layer_norm(ins[3], ins[4])
        return [a.detach(), b.detach(), *torch.autograd.grad([a, b], ins, [go, x])]

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_captured_graphs_replay_in_any_order():
    """Forward and backward captured twice, with splits, masks and the weights' gradient sums: each graph keeps its own
    workspaces, replays follow its inputs, and eager work between the replays changes nothing."""
    def case(seed, Sq, Sk):
        q, k, v, go = qkvg(1, Sq, Sk, 2, 2, 64, BF, seed)
        x, w, gy = rnd((500, 96), BF, seed), rnd((96,), FF, seed + 1), rnd((500, 96), BF, seed + 2)
        mask = (torch.rand(Sk, generator=torch.Generator().manual_seed(seed)) < 0.8)[None, None, None].to(DEV)
        pos = torch.arange(Sq, device=DEV, dtype=torch.int32)[None]
        leaves = [t.requires_grad_() for t in (q, k, v, x, w)]

        def run():
            a = ops.attention(ops.rotary(leaves[0], pos, (64,)), leaves[1], leaves[2], mask)
            b = ops.layer_norm(leaves[3], leaves[4])
            return [a.detach(), b.detach(), *torch.autograd.grad([a, b], leaves, [go, gy])]
        return leaves, run

    made = []
    for seed, Sq, Sk in ((1, 20, 2000), (50, 700, 150)):
        leaves, run = case(seed, Sq, Sk)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        made.append((leaves, run, graph, out))
    for step in range(3):
        for leaves, run, graph, out in made if step % 2 else made[::-1]:
            with torch.no_grad():
                for t in leaves:
                    t.mul_(0.9)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            for a, b in zip(got, run()):
                assert torch.equal(a, b)


def test_attention_long_keys_and_far_offsets():
    """One query over 300,000 keys whose rows span more than 2^31 bytes; the last keys count."""
    S, wide = 300_000, 4096
    kv = torch.zeros(1, S, 1, wide, dtype=BF, device=DEV)
    kv[..., :16] = rnd((1, S, 1, 16), BF, 0)
    kv[..., 16:32] = rnd((1, S, 1, 16), BF, 1)
    k, v = kv[..., :16], kv[..., 16:32]
    assert S * wide * 2 > 2 ** 31
    q = rnd((1, 1, 1, 16), BF, 2)
    check_attention(q, k, v, rnd((1, 1, 1, 16), BF, 3))
    k[0, S - 1] = 8 * q[0, 0]
    v[0, S - 1] = 5.0
    out = ops.attention(q, k, v, scale=2.0)
    assert (out == 5.0).all()


def test_attention_mask_past_the_table_of_tiles():
    """Keys beyond the tiles whose class a block keeps: processed, masked all the same."""
    S = 64 * 2048 + 500
    q, k, v, go = qkvg(1, 3, S, 1, 1, 8, BF)
    mask = (torch.rand(1, 1, 1, S, generator=torch.Generator().manual_seed(2)) < 0.5).to(DEV)
    mask[..., 64 * 2048 + 128:64 * 2048 + 300] = False
    check_attention(q, k, v, go, mask=mask)
    many = 32 * 2048 + 200                                   # as many rows, walked by the keys' blocks
    q, k, v, go = qkvg(1, many, 40, 1, 1, 8, BF)
    mask = (torch.rand(many, 40, generator=torch.Generator().manual_seed(3)) < 0.5).to(DEV)
    check_attention(q, k, v, go, mask=mask)


# ------------------------------------------------------------------------------- walks split over blocks, calls at once
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["lengths", "lengths causal", "mask", "mask causal"])
@pytest.mark.parametrize("shape", [(3, 70, 1500, 2, 1, 64), (3, 900, 900, 2, 2, 96), (3, 1, 4000, 4, 2, 32),
                                   (3, 1400, 90, 3, 1, 128)])
def test_attention_split_walks(shape, kind, dt):
    """Few row or key blocks: several blocks share a walk, some of whose parts are empty. Dead keys hold NaN."""
    B, Sq, Sk = shape[:3]
    q, k, v, go = qkvg(*shape, dt)
    kw = {"causal": "causal" in kind}
    n = [0, Sk // 2, Sk]
    if "lengths" in kind:
        kw["lengths"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    else:
        g = torch.Generator().manual_seed(23)
        m = (torch.rand(B, 1, 1, Sk, generator=g) < 0.7) & (torch.arange(Sk) < torch.tensor(n)[:, None, None, None])
        kw["mask"] = m.to(DEV)
        dead = ~m[:, 0, 0].to(DEV)
        k[dead] = math.nan
        v[dead] = math.inf
    if "lengths" in kind:
        for b in range(B):
            k[b, n[b]:] = math.inf
            v[b, n[b]:] = math.nan
    check_attention(q, k, v, go, **kw)


def test_gradient_of_a_sum_is_that_of_ones():
    """An expanded gradient (strides of 0) is read as what it stands for."""
    q, k, v, _ = qkvg(2, 50, 60, 2, 2, 32, BF)
    x, pos = rnd((2, 50, 2, 32), BF, 4), torch.arange(50, device=DEV)[None]
    w = rnd((32,), FF, 5)
    for f, ins in ((lambda *t: ops.attention(*t), (q, k, v)), (lambda t: ops.rotary(t, pos, (32,)), (x,)),
                   (lambda t, u: ops.layer_norm(t, u), (x, w))):
        ins = [t.detach().requires_grad_() for t in ins]
        a = torch.autograd.grad(f(*ins).sum(), ins)
        out = f(*ins)
        b = torch.autograd.grad(out, ins, torch.ones_like(out))
        for s, t in zip(a, b):
            assert torch.equal(s, t)


def test_calls_at_once_on_two_streams_and_threads():
    """Workspaces are a call's own: two threads on streams of their own get what one gets."""
    import threading
    cases = []
    for seed, shape in ((1, (1, 30, 3000, 2, 2, 64)), (7, (2, 600, 500, 2, 1, 32))):
        q, k, v, go = qkvg(*shape, BF, seed)
        x, w, gy = rnd((3000, 96), BF, seed), rnd((96,), FF, seed), rnd((3000, 96), BF, seed + 1)

        def run(q=q, k=k, v=v, go=go, x=x, w=w, gy=gy):
            ins = [t.detach().requires_grad_() for t in (q, k, v, x, w)]
            out = [ops.attention(*ins[:3], causal=True), ops.layer_norm(*ins[3:])]
            return [t.detach() for t in out] + list(torch.autograd.grad(out, ins, [go, gy]))
        cases.append((run, run()))
    torch.cuda.synchronize()
    bad = []

    def work(run, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = run()
            s.synchronize()
        bad.extend(n for n, (a, b) in enumerate(zip(got, want)) if not torch.equal(a, b))

    ts = [threading.Thread(target=work, args=c) for c in cases]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
        assert not t.is_alive()
    assert not bad


def test_layer_norm_is_the_same_every_time():
    x, w, b, gy = rnd((5000, 200), BF, 0), rnd((200,), FF, 1), rnd((200,), FF, 2), rnd((5000, 200), BF, 3)
    runs = []
    for _ in range(3):
        ins = [t.detach().requires_grad_() for t in (x, w, b)]
        runs.append(torch.autograd.grad(ops.layer_norm(*ins), ins, gy))
    for r in runs[1:]:
        for s, t in zip(r, runs[0]):
            assert torch.equal(s, t)


def test_attention_keeps_its_own_mask():
    """The packed mask is the call's: writing over the tensor before the backward pass changes nothing. A length that was
    written over is refused, as torch refuses any saved tensor that changed."""
    q, k, v, go = qkvg(2, 60, 70, 2, 2, 32, BF)
    mask = (torch.rand(60, 70, generator=torch.Generator().manual_seed(4)) < 0.5).to(DEV)
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    want = torch.autograd.grad(ops.attention(*ins, mask=mask.clone()), ins, go)
    out = ops.attention(*ins, mask=mask)
    mask.fill_(False)
    for a, b in zip(torch.autograd.grad(out, ins, go), want):
        assert torch.equal(a, b)
    lengths = torch.tensor([70, 30], dtype=torch.int32, device=DEV)
    out = ops.attention(*ins, lengths=lengths)
    lengths.fill_(5)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, ins, go)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_groups_do_not_hear_each_other(bad, D, dt):
    """Two images packed into one row of tokens: whatever breaks in one - a query, a key, a value, a gradient - leaves
    the other's output and gradients as they were, bit for bit, and shows in its own."""
    S, cut = 210, 110                                        # the border inside a tile of rows and of keys
    group = torch.arange(S, device=DEV) >= cut
    mask = group[:, None] == group[None]
    base = qkvg(1, S, S, 2, 1, D, dt)

    def run(ts):
        q, k, v, go = ts
        ins = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*ins, mask=mask)
        return [out.detach(), *torch.autograd.grad(out, ins, go)]

    want = run(base)
    for n in range(4):
        ts = [t.clone() for t in base]
        ts[n][0, cut - 3, 0, 1] = bad
        got = run(ts)
        for a, b in zip(got, want):
            assert torch.equal(a[:, cut:], b[:, cut:]), n
        assert not all(torch.isfinite(t[:, :cut]).all() for t in got), n


def test_attention_refuses_more_blocks_than_a_launch_has():
    q = torch.zeros(1 << 24, 1, 1, 8, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="too large for one launch"):
        ops.attention(q, q, q)
    assert not ops.attention(q[1:], q[1:], q[1:]).any()


def test_forward_mode_tangents_are_refused():
    """No forward-mode derivative: the call says so instead of dropping the tangent."""
    import torch.autograd.forward_ad as fwd
    q, k, v, go = qkvg(1, 4, 4, 1, 1, 32, BF)
    pos = torch.arange(4, device=DEV)[None]
    with fwd.dual_level():
        d = fwd.make_dual(q, go)
        for call in (lambda: ops.attention(d, k, v), lambda: ops.layer_norm(d), lambda: ops.rotary(d, pos, (32,))):
            with pytest.raises(RuntimeError):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError):
                call()
