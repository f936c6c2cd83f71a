"""How near attention comes to rounding nothing but its results, whatever the call's size and the magnitude of its
values (marked gpu).

The measure is the 2-norm of an output's error over that of the 64-bit result rounded to the tensors' type. 1 is an
output whose only error is its own rounding, u = finfo.eps / 2 relative. Two 16-bit parts of a weight leave u^2 of it, at
most 2^-8 of u. A score is a sum of D fp32 products: their roundings are independent, so that it is off by about
sqrt(D + 4) 2^-24 of the magnitude of its terms, here below 2^-17, 2^-6 of float16's u; dp and the sums over keys or rows
likewise. Each of these adds to 1 in squares, by less than a hundredth: LIMIT leaves ten. A weight rounded to one part
alone would give sqrt(2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from crack_detection_federatedlearning_grpc_amd import ops  # noqa: E402

DEV = torch.device("cuda")
BF, HF = torch.bfloat16, torch.float16
LIMIT = 1.1


def rnd(shape, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dt).to(DEV)


def definition(q, k, v, go, ok=None):
    """out, dq, dk, dv in 64 bits; ok: pairs that are allowed, (B, 1, Sq, Sk) or fewer axes."""
    B, Sq, Hq, D = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    Q, K, V, g = (t.double().transpose(1, 2).contiguous() for t in (q, k, v, go))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = Q @ K.transpose(2, 3) / math.sqrt(D)
    if ok is not None:
        s = s.masked_fill(~ok, -math.inf)
    p = torch.softmax(s, 3)
    o = p @ V
    ds = p * (g @ V.transpose(2, 3) - (g * o).sum(3, keepdim=True)) / math.sqrt(D)
    dk, dv = (t.unflatten(1, (Hkv, G)).sum(2) for t in (ds.transpose(2, 3) @ Q, p.transpose(2, 3) @ g))
    return [t.transpose(1, 2) for t in (o, ds @ K, dk, dv)]


def excess(q, k, v, go, ok=None, **kw):
    """error over that of rounding the results, of out, dq, dk and dv"""
    want = definition(q, k, v, go, ok)
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*ins, **kw)
    got = [out.detach(), *torch.autograd.grad(out, ins, go)]
    r = []
    for g, w in zip(got, want):
        assert torch.isfinite(w.to(q.dtype)).all()                   # the results themselves are in the type's range
        r.append(float((g.double() - w).norm() / (w.to(q.dtype).double() - w).norm()))
    return dict(zip(("out", "dq", "dk", "dv"), r))


def check(q, k, v, go, ok=None, **kw):
    e = excess(q, k, v, go, ok, **kw)
    assert all(x <= LIMIT for x in e.values()), e


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["plain", "causal", "lengths", "mask"])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
def test_many_pairs_are_as_accurate_as_few(D, kind, dt):
    """More than 2^24 pairs of a query and a key: the weights and dS are as exact as in a small call."""
    B, S, Hq, Hkv = 4, 1100, 4, 2
    assert B * Hq * S * S > 1 << 24
    q, k, v, go = (rnd((B, S, h, D), dt, n) for n, h in enumerate((Hq, Hkv, Hkv, Hq)))
    i = torch.arange(S, device=DEV)
    if kind == "causal":
        check(q, k, v, go, i <= i[:, None], causal=True)
    elif kind == "lengths":
        n = torch.tensor([S, 900, 333, 1], dtype=torch.int32, device=DEV)
        check(q, k, v, go, (i < n[:, None])[:, None, None], lengths=n)
    elif kind == "mask":
        m = (torch.rand(S, S, generator=torch.Generator().manual_seed(9)) < 0.6).to(DEV)
        check(q, k, v, go, m, mask=m)
    else:
        check(q, k, v, go)


@pytest.mark.parametrize("dt", [BF, HF])
def test_an_image_alone_and_in_a_large_batch(dt):
    """The number of images does not decide how exact a row is: an image's results in a batch are those of the image
    alone but for the order of fp32 sums, so that few of them round to another value."""
    B, S, H, D = 48, 640, 2, 64
    q, k, v, go = (rnd((B, S, H, D), dt, n) for n in range(4))

    def run(n):
        ins = [t[:n].detach().requires_grad_() for t in (q, k, v)]
        out = ops.attention(*ins)
        return [t[:1] for t in (out.detach(), *torch.autograd.grad(out, ins, go[:n]))]

    assert H * S * S < 1 << 24 < B * H * S * S
    for name, a, b in zip(("out", "dq", "dk", "dv"), run(1), run(B)):
        # a sum in another order differs by less than a 2^-9th of a half step here: a value in 2^8 rounds elsewhere
        assert float((a != b).double().mean()) <= 2 ** -5, name


# -------------------------------------------------------------------------------- float16: its range is 2^-24 .. 65,504
@pytest.mark.parametrize("Sq,Sk,D", [(64, 65536, 32), (16, 262144, 16), (200, 40000, 128)])
def test_float16_weights_of_long_keys(Sq, Sk, D):
    """Weights of 1 / Sk are below float16's normal range, dv is not."""
    q, k, v, go = (rnd((1, n, 1, D), HF, i) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    e = excess(q, k, v, go * 64)
    assert e["out"] <= LIMIT and e["dv"] <= LIMIT, e


@pytest.mark.parametrize("Sq", [1, 70])
def test_float16_weights_far_below_the_largest(Sq):
    """One key that outweighs all others by 2^20 and has no value: the output is what the others say."""
    D = 32
    q, k, v, go = (rnd((1, n, 1, D), HF, i) for i, n in enumerate((Sq, 65, 65, Sq)))
    q[..., 0], k[..., 0] = 8, 0
    k[:, 0], v[:, 0] = 0, 0
    k[:, 0, :, 0] = 20 * math.log(2) * math.sqrt(D) / 8
    e = excess(q, k, v * 1000, go)
    assert e["out"] <= LIMIT and e["dv"] <= LIMIT, e


@pytest.mark.parametrize("power", [-11, -13, -15])
@pytest.mark.parametrize("Sk", [4, 64, 700])
def test_float16_small_outputs(Sk, power):
    """dp - delta cancels to what the output's rounding took away, and that is below the type's smallest number."""
    q, k, v, go = (rnd((1, n, 2, 64), HF, i) for i, n in enumerate((200, Sk, Sk, 200)))
    check(q, k * 0.3, v * 2.0 ** power, go * 64)


DS = [(1, 1024, 4096, 2, 1, 64), (1, 256, 1024, 2, 2, 32), (1, 2048, 8192, 1, 1, 16), (2, 300, 300, 2, 2, 128),
      (2, 20, 900, 2, 1, 96)]


@pytest.mark.parametrize("kind", ["plain", "causal", "mask"])
@pytest.mark.parametrize("power", [-12, -8, 0, 7])
@pytest.mark.parametrize("shape", DS)
def test_float16_gradients_of_any_magnitude(shape, power, kind):
    """dS is about |go| sqrt(D) / Sk: far below float16's normal range where dq and dk, sums of many, are in it."""
    B, Sq, Sk, Hq, Hkv, D = shape
    q, k, v, go = (rnd((B, n, h, D), HF, i) for i, (n, h) in enumerate(((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq))))
    go = go * 2.0 ** power
    if kind == "causal":
        ok = torch.arange(Sk, device=DEV) <= torch.arange(Sq, device=DEV)[:, None] + Sk - Sq
        check(q, k, v, go, ok, causal=True)
    elif kind == "mask":
        m = (torch.rand(Sq, Sk, generator=torch.Generator().manual_seed(9)) < 0.6).to(DEV)
        check(q, k, v, go, m, mask=m)
    else:
        check(q, k, v, go)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_float16_ds_above_the_largest_number(D):
    """p (dp - delta) passes 65,504, dq and dk do not."""
    q, k, v, go = (rnd((1, n, 2, D), HF, i) for i, n in enumerate((16, 4, 4, 16)))
    q, k, v, go = q * 0.1, k * 0.1, v * 16, go * 2048
    w = go.double().transpose(1, 2) @ v.double().transpose(1, 2).transpose(2, 3)
    assert float((w - w.mean(3, keepdim=True)).abs().max()) / 4 > 65504          # p is about 1 / 4
    check(q, k, v, go)


@pytest.mark.parametrize("kind", ["plain", "causal"])
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
def test_float16_magnitudes_that_change_along_a_walk(D, up, kind):
    """Values and gradients that grow, or fall, by 2^16 from the first token to the last: every query's dq and every
    key's dk and dv is as exact as its own size allows."""
    S = 700
    q, k, v, go = (rnd((1, S, 2, D), HF, i) for i in range(4))
    s = 2.0 ** (torch.linspace(-10, 6, S, device=DEV) * (1 if up else -1) - (0 if up else 4))[:, None, None]
    v, go = (v * s).to(HF), (go * s).to(HF)
    ok = torch.arange(S, device=DEV) <= torch.arange(S, device=DEV)[:, None] if kind == "causal" else None
    want = definition(q, k, v, go, ok)
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.attention(*ins, causal=kind == "causal")
    for name, g, w in zip(("dq", "dk", "dv"), torch.autograd.grad(out, ins, go), want[1:]):
        size = w.abs().amax(3, keepdim=True)                                      # a token's own magnitude
        size = torch.where(size == 0, torch.ones_like(size), size)
        off, least = (g.double() - w) / size, (w.to(HF).double() - w) / size
        assert float(off.norm() / least.norm()) <= LIMIT, (name, float(off.norm() / least.norm()))
