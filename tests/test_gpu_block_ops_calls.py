"""Calls of attention, rotary positions and layer norm that are unusual, not wrong, or that have to be refused (marked
gpu)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

import torch.utils.checkpoint  # noqa: E402
from torch.fx.experimental.proxy_tensor import make_fx  # noqa: E402

from crack_detection_federatedlearning_grpc_amd import ops  # noqa: E402

DEV = torch.device("cuda")
BF, HF, FF = torch.bfloat16, torch.float16, torch.float32


def rnd(shape, dt, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dt).to(DEV)


POS = torch.arange(6, dtype=torch.int32)[None].to(DEV)
CALLS = {
    "attention": (lambda t: ops.attention(t, t, t), (2, 6, 2, 32)),
    "attention_qkv": (lambda t: ops.attention_qkv(t, 2), (2, 6, 6, 32)),
    "layer_norm": (lambda t: ops.layer_norm(t), (6, 32)),
    "rotary": (lambda t: ops.rotary(t, POS, (32,)), (2, 6, 2, 32)),
}


@pytest.fixture(params=list(CALLS))
def call(request):
    f, shape = CALLS[request.param]
    return f, rnd(shape, BF, 0)


def test_a_traced_backward_pass_is_refused(call):
    """The graph was made by an ordinary call; its backward pass writes through pointers like the call itself."""
    f, x = call
    x.requires_grad_()
    y = f(x)
    go = torch.ones_like(y)
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(y, x, g, retain_graph=True))(go)
    with pytest.raises(NotImplementedError, match="zero tensors"):
        torch.autograd.grad(y, x, torch._efficientzerotensor(y.shape, dtype=BF, device=DEV), retain_graph=True)
    (a,), (b,) = (torch.autograd.grad(y, x, go, retain_graph=True) for _ in range(2))
    assert torch.equal(a, b)


def test_a_compiled_function_calls_them_eagerly(call):
    """A compiler that meets the call breaks its graph there: the same result."""
    f, x = call
    g = torch.compile(lambda t: f(t * 2) + 1, backend="eager")
    assert torch.equal(g(x), f(x * 2) + 1)


def test_pending_signs_are_read():
    """The imaginary part of a conjugate is a view of the same memory with its sign pending."""
    z = torch.randn(2, 6, dtype=torch.complex64, generator=torch.Generator().manual_seed(3)).to(DEV)
    pos = z.conj().imag
    assert pos.is_neg()
    x = rnd((1, 6, 2, 32), FF, 1)
    assert torch.equal(ops.rotary(x, pos, (16, 16)), ops.rotary(x, pos.clone(), (16, 16)))
    one = z.view(12, 1).conj().imag                          # rows of one column, read at their stride
    w, b = (t.detach().requires_grad_() for t in (one[0], one[1]))
    assert w.is_neg() and one.is_neg()
    y = ops.layer_norm(one, w, b)
    u, v = (t.detach().clone().requires_grad_() for t in (w, b))
    want = ops.layer_norm(one.clone(), u, v)
    assert torch.equal(y, want)
    for s, t in zip(torch.autograd.grad(y, (w, b), one), torch.autograd.grad(want, (u, v), one.clone())):
        assert torch.equal(s, t)


def test_block_of_an_empty_batch():
    x = torch.zeros(0, 4, 4, 512, dtype=BF, device=DEV, requires_grad=True)
    w = [torch.ones(512, device=DEV), torch.zeros(512, device=DEV), rnd((1, 1, 512, 12 * 128), FF, 0),
         rnd((1, 1, 512, 512), FF, 1)]
    w = [t.requires_grad_() for t in w]
    y = ops.self_attention2d(x, *w, heads=4)
    assert y.shape == x.shape
    for g, t in zip(torch.autograd.grad(y.sum(), [x, *w]), [x, *w]):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 40, 32), (33, 40, 64), (100, 130, 96), (70, 300, 128)])
def test_a_key_of_minus_infinity_gives_its_value_no_gradient(Sq, Sk, D, causal, dt):
    """Its weight is 0 in every row, and the rows that fill up the last tile add nothing."""
    q, k, v, go = (rnd((1, n, 2, D), dt, i) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    q[..., 0] = q[..., 0].abs() + 0.5
    dead = torch.arange(Sk, device=DEV) % 3 == 1
    k[:, dead, :, 0] = -math.inf
    v.requires_grad_()
    (dv,) = torch.autograd.grad(ops.attention(q, k, v, causal=causal), v, go)
    assert (dv[:, dead] == 0).all() and torch.isfinite(dv).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["plain", "lengths", "causal", "mask", "mask causal", "bits"])
@pytest.mark.parametrize("Sq,Sk", [(1, 90), (20, 3000), (150, 150), (300, 70), (200, 2500)])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_rows_whose_every_score_is_minus_infinity(D, Sq, Sk, kind, dt):
    """softmax has no value there: NaN, as any broken row, and not the 0 of a row that may attend nothing. Rows with a
    finite score are what they are without the others."""
    B = 3
    q, k, v, go = (rnd((B, n, 2, D), dt, i) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    q[..., 0] = q[..., 0].abs() + 0.5
    g = torch.Generator().manual_seed(4)
    dead = torch.rand(B, Sk, generator=g) < 0.5
    dead[0] = True                                           # an image without a finite score
    dead[1, :Sk // 2] = True                                 # one whose first half has none
    dead = dead.to(DEV)
    k[..., 0] = torch.where(dead[..., None], torch.full_like(k[..., 0], -math.inf), k[..., 0])
    ok, kw = torch.ones(B, Sq, Sk, dtype=torch.bool, device=DEV), {}
    if "causal" in kind:
        ok = ok & (torch.arange(Sk, device=DEV) <= torch.arange(Sq, device=DEV)[:, None] + Sk - Sq)
        kw["causal"] = True
    if kind == "lengths":
        kw["lengths"] = torch.tensor([Sk - 3, Sk // 2, 0], dtype=torch.int32, device=DEV)
        ok = ok & (torch.arange(Sk, device=DEV) < kw["lengths"][:, None])[:, None]
    if "mask" in kind or kind == "bits":
        m = (torch.rand(B, Sq, Sk, generator=g) < (0.02 if kind == "bits" else 0.6)).to(DEV)
        m[:, Sq // 2] = False
        kw["mask"], ok = m[:, None], ok & m
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    out, lse = ops.attention(*ins, return_lse=True, **kw)
    alive = ok & ~dead[:, None]
    broken = ok.any(2) & ~alive.any(2)                       # (B, Sq)
    empty = ~ok.any(2)
    assert broken.any() or not ok.any()
    assert out[broken].isnan().all() and (out[empty] == 0).all() and torch.isfinite(out[~broken]).all()
    assert (lse.transpose(1, 2)[broken | empty] == -math.inf).all() and torch.isfinite(lse.transpose(1, 2)[~(broken | empty)]).all()
    with torch.no_grad():
        want, wlse = ops.attention(q, k, v, mask=alive[:, None], return_lse=True)
    live = ~(broken | empty)
    # the same pairs count; the tiles that are walked differ, and with them the order of fp32 sums
    assert ((out[live].double() - want[live].double()).abs() <= torch.finfo(dt).eps * (want[live].double().abs() + 2 ** -8)).all()
    assert (lse.transpose(1, 2)[live] - wlse.transpose(1, 2)[live]).abs().max() <= 1e-5 if live.any() else True
    dq, dk, dv = torch.autograd.grad(out, ins, go)
    assert dq[broken].isnan().all() and (dq[empty] == 0).all()
    hit = (ok & broken[..., None]).any(1)                    # keys that a broken row may attend
    assert dv[hit].isnan().all() and torch.isfinite(dv[~hit]).all()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["causal", "mask"])
@pytest.mark.parametrize("Sq", [20, 150])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_a_small_weight_hides_no_infinity(D, Sq, kind, dt):
    """A weight of 2^-43 of the row's largest is none that 16 bits hold, and still not 0."""
    S = 150
    q, k, v, go = (rnd((1, n, 2, D), dt, i) for i, n in enumerate((Sq, S, S, Sq)))
    q[..., 0], k[..., 0] = 8, 0
    j = S - Sq + 5                                           # the rows from 5 on may attend it
    k[:, j] = 0
    k[:, j, :, 0] = -30 * math.sqrt(D) / 8
    tri = torch.arange(S, device=DEV) <= torch.arange(Sq, device=DEV)[:, None] + S - Sq
    kw = {"causal": True} if kind == "causal" else {"mask": tri}
    want = ops.attention(q, k, v, **kw)
    for x in (math.inf, -math.inf, math.nan):
        w = v.clone()
        w[0, j, :, 3] = x
        out = ops.attention(q, k, w, **kw)
        hit = out[0, 5:, :, 3].float()
        assert (hit.isnan().all() if math.isnan(x) else (hit == x).all())
        assert torch.equal(out[0, :5], want[0, :5])
    g = go.clone()
    g[0, Sq - 1, :, 4] = math.inf                            # the row that attends every key
    v.requires_grad_()
    (dv,) = torch.autograd.grad(ops.attention(q, k, v, **kw), v, g)
    assert (dv[..., 4] == math.inf).all() and torch.isfinite(dv[..., :4]).all()


def test_calls_at_once_on_two_streams_and_threads_each_of_them():
    """Two threads on streams of their own: every result of every call is what a call alone gives, and none raises."""
    import threading
    cases = []
    for seed, shape in ((1, (1, 30, 3000, 2, 2, 64)), (7, (2, 600, 500, 2, 1, 32))):
        B, Sq, Sk, Hq, Hkv, D = shape
        q, k, v, go = (rnd((B, n, h, D), BF, seed + i) for i, (n, h) in enumerate(((Sq, Hq), (Sk, Hkv), (Sk, Hkv), (Sq, Hq))))
        x, w, gy = rnd((3000, 96), BF, seed), rnd((96,), FF, seed), rnd((3000, 96), BF, seed + 1)
        mask = (torch.rand(Sk, generator=torch.Generator().manual_seed(seed)) < 0.7)[None, None, None].to(DEV)
        pos = torch.arange(Sq, device=DEV)[None]

        def run(q=q, k=k, v=v, go=go, x=x, w=w, gy=gy, mask=mask, pos=pos, D=D):
            ins = [t.detach().requires_grad_() for t in (q, k, v, x, w)]
            out = [ops.attention(ops.rotary(ins[0], pos, (D,)), ins[1], ins[2], mask), ops.layer_norm(*ins[3:])]
            return [t.detach() for t in out] + list(torch.autograd.grad(out, ins, [go, gy]))
        cases.append((run, run()))
    torch.cuda.synchronize()
    bad, done, together = [], [], threading.Barrier(2, timeout=30)

    def work(n, run, want):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                together.wait()
                got = [run() for _ in range(20)]
                s.synchronize()
            for i, g in enumerate(got):
                bad.extend((n, i, j) for j, (a, b) in enumerate(zip(g, want)) if not torch.equal(a, b))
            done.append(n)
        except Exception as e:  # noqa: BLE001 - a thread's exception would be lost
            bad.append((n, repr(e)))

    ts = [threading.Thread(target=work, args=(n, *c)) for n, c in enumerate(cases)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
        assert not t.is_alive()
    assert not bad and sorted(done) == [0, 1]


def test_inference_mode_and_saved_tensor_hooks(call):
    """What autograd saves may come back from elsewhere, as a copy with other strides; without autograd nothing is."""
    f, x = call
    x.requires_grad_()
    y = f(x)
    go = torch.ones_like(y)
    (want,) = torch.autograd.grad(y, x, go)
    with torch.inference_mode():
        assert torch.equal(f(x.detach().clone()), y)
    with torch.autograd.graph.save_on_cpu():
        z = f(x)
    assert torch.equal(torch.autograd.grad(z, x, go)[0], want)
    z = torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(z, x, go)[0], want)


@pytest.mark.parametrize("causal", [False, True])
def test_saved_slices_come_back_as_copies(causal):
    """q, k and v are slices of one tensor, with a mask and lengths, and what is saved of them returns contiguous."""
    qkv = rnd((2, 70, 8, 64), BF, 0)
    q, k, v = (t.detach().requires_grad_() for t in qkv.split([4, 2, 2], 2))
    assert not q.is_contiguous()
    mask = (torch.rand(2, 1, 70, 70, generator=torch.Generator().manual_seed(1)) < 0.6).to(DEV)
    lengths = torch.tensor([[70, 0], [33, 0]], dtype=torch.int32, device=DEV)[:, 0]
    go = rnd((2, 70, 4, 64), BF, 1)
    want = torch.autograd.grad(ops.attention(q, k, v, mask, lengths, causal), (q, k, v), go)
    with torch.autograd.graph.save_on_cpu():
        out = ops.attention(q, k, v, mask, lengths, causal)
    for a, b in zip(torch.autograd.grad(out, (q, k, v), go), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", [BF, HF, FF])
def test_rotary_of_an_odd_number_of_channels(dt, inter):
    x, pos = rnd((2, 9, 3, 33), dt, 0), torch.arange(18, device=DEV).view(2, 9)
    whole = ops.rotary(x, pos, (16, 16), interleaved=inter)
    assert torch.equal(whole[..., 32:], x[..., 32:])
    assert torch.equal(whole[..., :32], ops.rotary(x[..., :32], pos, (16, 16), interleaved=inter))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("kind", ["plain", "causal", "lengths", "mask"])
@pytest.mark.parametrize("B,Sq,Hq,Hkv,D", [(1, 1, 3, 3, 64), (4, 1, 16, 4, 16), (3, 200, 2, 1, 128)])
def test_one_key_has_no_gradient_through_its_score(B, Sq, Hq, Hkv, D, kind, dt):
    """A softmax over one key is 1: dq and dk are 0, dv the sum of the gradients of the rows that attend it."""
    q, k, v, go = (rnd((B, n, h, D), dt, i) for i, (n, h) in enumerate(((Sq, Hq), (1, Hkv), (1, Hkv), (Sq, Hq))))
    kw = {"causal": {"causal": True}, "mask": {"mask": (torch.arange(Sq, device=DEV) % 3 != 1)[:, None]},
          "lengths": {"lengths": torch.tensor([1, 0, 1, 1][:B], dtype=torch.int32, device=DEV)}}.get(kind, {})
    ins = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(ops.attention(*ins, **kw), ins, go)
    assert not dq.any() and not dk.any()
    on = torch.ones(B, Sq, dtype=torch.bool, device=DEV)
    if kind == "causal":
        on[:, :-1] = False
    elif kind == "lengths":
        on = on & (kw["lengths"] > 0)[:, None]
    elif kind == "mask":
        on = on & kw["mask"].T
    want = (go.double() * on[..., None, None]).unflatten(2, (Hkv, Hq // Hkv)).sum(3).sum(1, keepdim=True)
    mag = (go.double().abs() * on[..., None, None]).unflatten(2, (Hkv, Hq // Hkv)).sum(3).sum(1, keepdim=True)
    # one rounding of the result, and as many of fp32 as there are terms (a weight is 1 within two steps of fp32)
    assert ((dv.double() - want).abs() <= torch.finfo(dt).eps / 2 * want.abs() * 1.001 + (Sq * Hq + 8) * 2.0 ** -24 * mag).all()
