"""What is measured of the attention-block operators (``ops.attention``, ``ops.attention_qkv``, ``ops.rotary``,
``ops.layer_norm``): listed cases, drawn ones of the same ranges, a plain torch form and a definition in 64 bits.

The operators work on feature maps read as tokens (an H x W map is H * W tokens), next to the convolutions of
``ops``. With ``own`` set, ``run`` makes the calls a user makes of the framework; otherwise it computes the same in
elementary torch operations."""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 1 << 28                      # attention scores held at a time by the plain form


# ---------------------------------------------------------------------------------------------------- the cases
def _attn(name, train, dtype, b, sq, sk, hq, hkv, d, causal=False, mask="none", grid=(0, 0), radius=0, packed=False):
    c = {"op": "attention", "train": train, "dtype": dtype, "b": b, "sq": sq, "sk": sk, "hq": hq, "hkv": hkv, "d": d,
         "causal": causal, "mask": mask, "gh": grid[0], "gw": grid[1], "radius": radius, "packed": packed}
    return {"name": name, **c} if name else c


def _norm(name, train, dtype, rows, c, wide=0):
    d = {"op": "layer_norm", "train": train, "dtype": dtype, "rows": rows, "c": c, "wide": wide}
    return {"name": name, **d} if name else d


def _rot(name, train, dtype, b, grid, h, d, dims, joint=False, interleaved=False, start=0, fractional=False):
    c = {"op": "rotary", "train": train, "dtype": dtype, "b": b, "t": grid[0], "gh": grid[1], "gw": grid[2], "h": h,
         "d": d, "dims": "%d,%d,%d" % tuple(dims), "joint": joint, "interleaved": interleaved, "start": start,
         "fractional": fractional}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one learned query a head reads every pixel of 64 x 64 maps (attention pooling; a single token at a time)
        _attn("attn_one_query", False, "bf16", 8, 1, 4096, 8, 8, 32),
        # the 16 x 16 bottleneck of a 256 x 256 image batch, trained: the call that the headline configuration makes
        _attn("attn_bottleneck_train", True, "bf16", 16, 256, 256, 8, 8, 32, packed=True),
        # the 32 x 32 level of 512 x 512 images, trained in fp16
        _attn("attn_level_train", True, "fp16", 16, 1024, 1024, 8, 8, 64, packed=True),
        # images of different sizes padded into one batch: odd lengths, shared key heads, a head width between tiles
        _attn("attn_ragged_train", True, "bf16", 6, 1531, 1531, 8, 2, 80, mask="lengths"),
        # a 40 x 40 map where a pixel attends its neighbourhood only (a dense boolean mask)
        _attn("attn_window_train", True, "bf16", 4, 1600, 1600, 8, 8, 64, mask="window", grid=(40, 40), radius=6),
        # a long sequence of frames, causal, shared key heads: the largest
        _attn("attn_causal_train", True, "bf16", 2, 8192, 8192, 16, 2, 128, causal=True),
        # one 16 x 16 map at inference: the smallest, where latency counts
        _norm("norm_small", False, "bf16", 256, 256),
        # the 128 x 128 x 32 maps of a 256 x 256 batch of 16, trained
        _norm("norm_map_train", True, "bf16", 16 * 128 * 128, 32),
        # half of the channels of a wider fp32 map, an odd width, trained
        _norm("norm_odd_train", True, "fp32", 20011, 333, wide=667),
        # wide token rows, trained
        _norm("norm_wide_train", True, "fp16", 16384, 4096),
        # rows and columns of a 16 x 16 map: latency
        _rot("rotary_small", False, "bf16", 1, (1, 16, 16), 16, 32, (0, 16, 16)),
        # a video's frames, rows and columns far into the stream, query and key heads in one tensor, trained
        _rot("rotary_video_train", True, "bf16", 2, (16, 31, 33), 20, 128, (32, 48, 48), joint=True, start=1 << 20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    op = rng.choice(["attention", "attention", "attention", "layer_norm", "layer_norm", "rotary"])
    train = rng.random() < 0.6
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "fp16"])
        hkv = rng.choice([1, 2, 3, 4, 8])
        hq = hkv * rng.choice([1, 1, 1, 2, 4])
        d = 8 * rng.randint(2, 16)
        b = _log(rng, 1, 24)
        mask = rng.choice(["none", "none", "lengths", "keys", "window"])
        if mask == "window":
            gh, gw = _log(rng, 3, 64), _log(rng, 3, 64)
            return _attn("", train, dtype, b, gh * gw, gh * gw, hq, hkv, d, mask=mask, grid=(gh, gw),
                         radius=rng.randint(1, 12), packed=rng.random() < 0.5)
        shape = rng.choice(["self", "self", "cross", "one"])
        sk = _log(rng, 1, 8192)
        sq = {"self": sk, "cross": _log(rng, 1, 4096), "one": 1}[shape]
        return _attn("", train, dtype, b, sq, sk, hq, hkv, d, causal=rng.random() < 0.3, mask=mask,
                     packed=sq == sk and rng.random() < 0.5)
    if op == "layer_norm":
        c = _log(rng, 1, 8192)
        return _norm("", train, rng.choice(["bf16", "fp16", "fp32"]), _log(rng, 1, 300000), c,
                     wide=c + rng.randint(1, 64) if rng.random() < 0.3 else 0)
    grid = (_log(rng, 1, 32), _log(rng, 1, 48), _log(rng, 1, 48))
    d = 2 * rng.randint(4, 128)
    cut = sorted(rng.randint(0, d // 2) for _ in range(3))
    dims = (2 * cut[0], 2 * (cut[1] - cut[0]), 2 * (cut[2] - cut[1]))
    if sum(dims) == 0:
        dims = (0, 2 * (d // 4), 2 * (d // 4))
    return _rot("", train, rng.choice(["bf16", "fp16", "fp32"]), _log(rng, 1, 16), grid, _log(rng, 1, 32), d, dims,
                joint=rng.random() < 0.5, interleaved=rng.random() < 0.5, start=_log(rng, 1, 1 << 30),
                fractional=rng.random() < 0.3)


def draw(rng: random.Random):
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["op"], [0, 0])
        t[0], t[1] = max(t[0], w["bytes"]), max(t[1], w["flops"])
    while True:
        c = _draw_once(rng)
        w = work(c)
        full = 4 * c["b"] * c["hq"] * c["sq"] * c["sk"] * c["d"] if c["op"] == "attention" else 0
        if w["bytes"] <= top[c["op"]][0] and w["flops"] <= top[c["op"]][1] and full <= 2e12:
            return c


# --------------------------------------------------------------------------------------------------- their inputs
def _lengths(case):
    """Valid keys of each image of a padded batch: the first one full, then shorter; the last of three or more empty."""
    b, sk = case["b"], case["sk"]
    n = [max(1, sk - (sk * i) // (b + 1)) for i in range(b)]
    if b >= 3:
        n[-1] = 0
    return n


def _key_counts(case):
    """Valid pixels of each image where a key mask marks them."""
    return [max(1, (case["sk"] * (8 - i % 6)) // 8) for i in range(case["b"])]


def _window(case):
    gh, gw, r = case["gh"], case["gw"], case["radius"]
    y = torch.arange(gh * gw) // gw
    x = torch.arange(gh * gw) % gw
    return ((y[:, None] - y[None]).abs() <= r) & ((x[:, None] - x[None]).abs() <= r)


def _rand(gen, shape, dtype, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).mul_(scale).add_(shift).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 17)
    host = random.Random(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "attention":
        b, sq, sk, hq, hkv, d = (case[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
        if case["packed"]:
            s["qkv"] = _rand(gen, (b, sq, hq + 2 * hkv, d), dt)
        else:
            s["q"], s["k"], s["v"] = (_rand(gen, (b, n, h, d), dt) for n, h in ((sq, hq), (sk, hkv), (sk, hkv)))
        if case["train"]:
            s["go"] = _rand(gen, (b, sq, hq, d), dt)
        if case["mask"] == "lengths":
            n = _lengths(case)
            host.shuffle(n)
            s["lengths"] = torch.tensor(n, dtype=torch.int32).to(DEV)
        elif case["mask"] == "keys":
            n = _key_counts(case)
            host.shuffle(n)
            order = torch.rand(b, sk, generator=gen, device=DEV).argsort(1).argsort(1)
            s["mask"] = (order < torch.tensor(n, device=DEV)[:, None])[:, None, None, :]
        elif case["mask"] == "window":
            s["mask"] = _window(case).to(DEV)[None, None]
    elif case["op"] == "layer_norm":
        rows, c = case["rows"], case["c"]
        full = _rand(gen, (rows, case["wide"] or c), dt, 1.5, 0.5)
        s["x"] = full[:, :c]
        s["weight"] = _rand(gen, (c,), torch.float32, 0.2, 1.0)
        s["bias"] = _rand(gen, (c,), torch.float32, 0.2)
        if case["train"]:
            s["gy"] = _rand(gen, (rows, c), dt)
    else:
        t, gh, gw = case["t"], case["gh"], case["gw"]
        n = t * gh * gw
        i = torch.arange(n, device=DEV)
        pos = torch.stack([i // (gh * gw) + case["start"], i // gw % gh, i % gw])
        if case["fractional"]:
            s["pos"] = pos.to(torch.float32) * (0.5 + host.random())
        else:
            s["pos"] = (pos + host.randint(0, 7)).to(torch.int32)
        s["x"] = _rand(gen, (case["b"], n, case["h"], case["d"]), dt)
        if case["train"]:
            s["gy"] = _rand(gen, (case["b"], n, case["h"], case["d"]), dt)
    return s


# ------------------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from crack_detection_federatedlearning_grpc_amd import ops
    case = s["case"]
    train = case["train"]

    def leaf(t):
        return t.detach().requires_grad_() if train else t

    if case["op"] == "attention":
        kw = {"mask": s.get("mask"), "lengths": s.get("lengths"), "causal": case["causal"]}
        if case["packed"]:
            ins = (leaf(s["qkv"]),)
            out = ops.attention_qkv(ins[0], case["hq"], case["hkv"], **kw)
        else:
            ins = (leaf(s["q"]), leaf(s["k"]), leaf(s["v"]))
            out = ops.attention(*ins, **kw)
        return [out.detach(), *torch.autograd.grad(out, ins, s["go"])] if train else [out]
    if case["op"] == "layer_norm":
        ins = (leaf(s["x"]), leaf(s["weight"]), leaf(s["bias"]))
        y = ops.layer_norm(*ins)
        return [y.detach(), *torch.autograd.grad(y, ins, s["gy"])] if train else [y]
    x = leaf(s["x"])
    y = ops.rotary(x, s["pos"], _dims(case), joint=case["joint"], interleaved=case["interleaved"])
    return [y.detach(), *torch.autograd.grad(y, x, s["gy"])] if train else [y]


def _dims(case):
    return tuple(int(n) for n in case["dims"].split(","))


# --------------------------------------------------------------------------------------------------- the plain form
def _allowed(s, b0, b1):
    """The pairs (query, key) that images b0..b1 may use, broadcastable to (b1 - b0, 1, 1, sq, sk), or None."""
    case = s["case"]
    sq, sk = case["sq"], case["sk"]
    ok = None
    if "mask" in s:
        m = s["mask"]
        ok = (m if m.shape[0] == 1 else m[b0:b1])[:, None]
    if "lengths" in s:
        a = (torch.arange(sk, device=DEV) < s["lengths"][b0:b1, None])[:, None, None, None, :]
        ok = a if ok is None else ok & a
    if case["causal"]:
        a = torch.arange(sk, device=DEV) <= torch.arange(sq, device=DEV)[:, None] + (sk - sq)
        ok = a if ok is None else ok & a
    return ok


def _plain_attention(s):
    case = s["case"]
    b, sq, sk, hq, hkv, d = (case[n] for n in ("b", "sq", "sk", "hq", "hkv", "d"))
    g = hq // hkv
    if case["packed"]:
        q, k, v = s["qkv"].split([hq, hkv, hkv], 2)
    else:
        q, k, v = s["q"], s["k"], s["v"]
    train, dt = case["train"], q.dtype
    scale = 1 / math.sqrt(d)
    out = torch.empty(b, sq, hq, d, dtype=dt, device=DEV)
    dq, dk, dv = (torch.empty(b, t.shape[1], t.shape[2], d, dtype=dt, device=DEV) for t in (q, k, v)) if train else [None] * 3
    nh = max(1, min(hkv, CHUNK // (g * sq * sk)))
    nb = max(1, min(b, CHUNK // (hkv * g * sq * sk))) if nh == hkv else 1
    for b0 in range(0, b, nb):
        b1 = min(b, b0 + nb)
        ok = _allowed(s, b0, b1)
        for h0 in range(0, hkv, nh):
            h1 = min(hkv, h0 + nh)
            qs = slice(h0 * g, h1 * g)

            def heads(t, n):           # (images, key heads, heads that share one, tokens, d) in 32 bits
                return t.float().unflatten(2, (h1 - h0, n)).permute(0, 2, 3, 1, 4)

            qf = heads(q[b0:b1, :, qs], g)
            kf, vf = heads(k[b0:b1, :, h0:h1], 1), heads(v[b0:b1, :, h0:h1], 1)
            p = (qf @ kf.transpose(-1, -2)) * scale
            if ok is not None:
                p = p.masked_fill(~ok, -math.inf)
            m = p.amax(-1, keepdim=True)
            p = torch.exp(p - torch.where(m == -math.inf, 0.0, m))
            n = p.sum(-1, keepdim=True)
            p = p / torch.where(n == 0, 1.0, n)
            o = p @ vf
            out[b0:b1, :, qs] = o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(dt)
            if train:
                go = heads(s["go"][b0:b1, :, qs], g)
                dv[b0:b1, :, h0:h1] = (p.transpose(-1, -2) @ go).sum(2).transpose(1, 2).to(dt)
                ds = p * (go @ vf.transpose(-1, -2) - (go * o).sum(-1, keepdim=True)) * scale
                dq[b0:b1, :, qs] = (ds @ kf).permute(0, 3, 1, 2, 4).flatten(2, 3).to(dt)
                dk[b0:b1, :, h0:h1] = (ds.transpose(-1, -2) @ qf).sum(2).transpose(1, 2).to(dt)
    if not train:
        return [out]
    return [out, torch.cat([dq, dk, dv], 2)] if case["packed"] else [out, dq, dk, dv]


def _plain_norm(s, eps=1e-3):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = (xh * s["weight"] + s["bias"]).to(s["x"].dtype)
    if not s["case"]["train"]:
        return [y]
    gy = s["gy"].float()
    g = gy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    gy = gy.double()                                            # long sums
    return [y, dx.to(y.dtype), (gy * xh).sum(0).float(), gy.sum(0).float()]


def _angles(case, pos):
    """(tokens, pairs) angles in 64 bits: pair i of an axis turns by position * 10000^(-2 i / dims)."""
    dims, out, i0 = _dims(case), [], 0
    for a, n in enumerate(dims):
        i = torch.arange(n // 2, device=DEV, dtype=torch.float64)
        if case["joint"]:
            e = (i + i0) * 2 / sum(dims)
        else:
            e = i * 2 / max(n, 1)
        out.append(pos[a].double()[:, None] * 10000.0 ** -e)
        i0 += n // 2
    return torch.cat(out, 1)


def _turn(case, x, cos, sin):
    n = sum(_dims(case))
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., n:]], -1)


def _plain_rotary(s):
    case = s["case"]
    ang = _angles(case, s["pos"])
    cos, sin = ang.cos().float()[None, :, None], ang.sin().float()[None, :, None]
    y = _turn(case, s["x"].float(), cos, sin).to(s["x"].dtype)
    if not case["train"]:
        return [y]
    return [y, _turn(case, s["gy"].float(), cos, -sin).to(y.dtype)]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"attention": _plain_attention, "layer_norm": _plain_norm, "rotary": _plain_rotary}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- the definition, 64 bits
def _exact_attention(s):
    case = s["case"]
    hq, hkv, d, train = case["hq"], case["hkv"], case["d"], case["train"]
    if case["packed"]:
        q, k, v = s["qkv"][:, :, :hq], s["qkv"][:, :, hq:hq + hkv], s["qkv"][:, :, hq + hkv:]
    else:
        q, k, v = s["q"], s["k"], s["v"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (q, k, v)) if train else [None] * 3
    keys = torch.arange(case["sk"], device=DEV)
    last = torch.arange(case["sq"], device=DEV)[:, None] + case["sk"] - case["sq"]
    for b in range(case["b"]):
        hide = None
        if "mask" in s:
            hide = ~s["mask"][b if s["mask"].shape[0] > 1 else 0, 0]
        if "lengths" in s:
            hide = keys[None] >= s["lengths"][b]
        if case["causal"]:
            hide = (keys > last) if hide is None else hide | (keys > last)
        for h in range(hq):
            j = h * hkv // hq
            kd, vd = k[b, :, j].double(), v[b, :, j].double()
            z = q[b, :, h].double() @ kd.T / math.sqrt(d)
            if hide is not None:
                z = z.masked_fill(hide, -math.inf)
            p = torch.exp(z - torch.logsumexp(z, 1, True).nan_to_num(neginf=0.0))
            out[b, :, h] = p @ vd
            if train:
                go = s["go"][b, :, h].double()
                dv[b, :, j] += p.T @ go
                dp = go @ vd.T
                dz = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dq[b, :, h] = dz @ kd
                dk[b, :, j] += dz.T @ q[b, :, h].double()
    if not train:
        return [out]
    return [out, torch.cat([dq, dk, dv], 2)] if case["packed"] else [out, dq, dk, dv]


def _exact_norm(s, eps=1e-3):
    x, w, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    c = x.shape[1]
    dev = x - x.sum(1, keepdim=True) / c
    std = torch.sqrt((dev * dev).sum(1, keepdim=True) / c + eps)
    n = dev / std
    y = n * w + bias
    if not s["case"]["train"]:
        return [y]
    gy = s["gy"].double()
    gn = gy * w
    dx = (gn - gn.sum(1, keepdim=True) / c - n * ((gn * n).sum(1, keepdim=True) / c)) / std
    return [y, dx, (gy * n).sum(0), gy.sum(0)]


def _exact_rotary(s):
    case = s["case"]
    dims = _dims(case)
    n = sum(dims)
    pairs = [(a, i) for a, m in enumerate(dims) for i in range(m // 2)]
    axis = torch.tensor([a for a, _ in pairs], device=DEV)
    if case["joint"]:
        rate = [10000.0 ** (-2.0 * i / n) for i in range(n // 2)]
    else:
        rate = [10000.0 ** (-2.0 * i / dims[a]) for a, i in pairs]
    ang = s["pos"].double()[axis].T * torch.tensor(rate, device=DEV, dtype=torch.float64)
    unit = torch.polar(torch.ones_like(ang), ang)[None, :, None]

    def turn(x, by):
        x = x.double()
        if case["interleaved"]:
            z = torch.complex(x[..., 0:n:2], x[..., 1:n:2]) * by
            y = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., :n // 2], x[..., n // 2:n]) * by
            y = torch.cat([z.real, z.imag], -1)
        return torch.cat([y, x[..., n:]], -1)

    y = turn(s["x"], unit)
    return [y, turn(s["gy"], unit.conj())] if case["train"] else [y]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attention": _exact_attention, "layer_norm": _exact_norm, "rotary": _exact_rotary}[case["op"]](s)


# ------------------------------------------------------------------------------------------------------ what it costs
def _pairs(case):
    """(query, key) pairs of one head, over the batch."""
    b, sq, sk = case["b"], case["sq"], case["sk"]
    if case["mask"] == "window":
        def axis(n):
            return sum(min(n, i + case["radius"] + 1) - max(0, i - case["radius"]) for i in range(n))
        return b * axis(case["gh"]) * axis(case["gw"])
    n = _lengths(case) if case["mask"] == "lengths" else [sk] * b
    if not case["causal"]:
        return sq * sum(_key_counts(case) if case["mask"] == "keys" else n)
    part = sum(sum(min(max(i + 1 + sk - sq, 0), m) for i in range(sq)) for m in n)
    if case["mask"] == "keys":
        part = part * sum(_key_counts(case)) // (b * sk)       # the valid keys lie evenly
    return part


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    passes = 2 if case["train"] else 1
    if case["op"] == "attention":
        nq = case["b"] * case["sq"] * case["hq"] * case["d"]
        nk = case["b"] * case["sk"] * case["hkv"] * case["d"]
        m = {"none": 0, "lengths": 4 * case["b"], "keys": case["b"] * case["sk"], "window": case["sq"] * case["sk"]}
        # two products forward; backward the probabilities again and four more
        flops = 2 * (7 if case["train"] else 2) * _pairs(case) * case["hq"] * case["d"]
        return {"bytes": passes * 2 * size * (nq + nk) + m[case["mask"]], "flops": flops}
    if case["op"] == "layer_norm":
        n = case["rows"] * case["c"]
        return {"bytes": passes * (2 * size * n + 8 * case["c"]), "flops": (20 if case["train"] else 8) * n}
    n = case["b"] * case["t"] * case["gh"] * case["gw"]
    return {"bytes": passes * 2 * size * n * case["h"] * case["d"] + 12 * case["t"] * case["gh"] * case["gw"],
            "flops": passes * 3 * n * case["h"] * sum(_dims(case))}
