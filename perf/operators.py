"""What a transformer block runs between its matrix products, as cases that can be timed and compared.

A case is a dict: `kind` names the operator and direction, the other entries are its sizes and options.

kind         what it is
rope         rotary positions on the heads of a projection, forward or (inverse) for its gradient
norm_fwd     out = x + scale * gate * N(y; w_post), h = N(out; w_pre): the norms after and before a block,
             its gate and the residual, one pass
norm_bwd     the gradients of that, from what the forward pass left
attn_fwd     causal attention with a sliding window and first tokens that stay visible (sinks)
attn_step    the same in training: forward, then backward
attn_decode  the same for one new token per sequence over a cache

With `own` false, run() computes an operator in elementary torch operations, in fp32 (angles in fp64), rounded once at the
end; with `own` true it makes the framework's calls.  exact() is the operator's definition in fp64.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # Token-by-token inference: the q and k heads of eight sequences, each far into its context.  All latency.
        dict(name="rope decode 8", kind="rope", dtype="bf16", b=8, t=1, heads=24, of=36, hd=64, rot=64, interleaved=False,
             inverse=False, far=100000, factor=1.0),
        # GPT-2 small in training, 8 x 1024 tokens: q and k rotated inside the packed projection's rows.
        dict(name="rope packed 8192", kind="rope", dtype="bf16", b=8, t=1024, heads=24, of=36, hd=64, rot=64, interleaved=False,
             inverse=False, far=0, factor=1.0),
        # The gradient of a long sequence's rotation: half of each head, neighbouring pairs, scaled to eight times the
        # trained length.
        dict(name="rope long inverse", kind="rope", dtype="bf16", b=1, t=32768, heads=40, of=48, hd=128, rot=64, interleaved=True,
             inverse=True, far=0, factor=8.0),
        # One new token of eight sequences between two blocks.
        dict(name="norm 8 rows", kind="norm_fwd", act="bf16", res="bf16", rows=8, c=768, post=True, gate=True, groups=1),
        # GPT-2-XL-wide rows in training, the residual stream in fp32.
        dict(name="norm fwd 8192", kind="norm_fwd", act="bf16", res="fp32", rows=8192, c=1600, post=True, gate=True, groups=1),
        # A short batch of a width that suits no vector, all fp32, without a post-norm.
        dict(name="norm bwd odd", kind="norm_bwd", act="fp32", res="fp32", rows=1537, c=771, post=False, gate=True, groups=1),
        # The same block's gradients in training, a gate of its own for each of eight sequences.
        dict(name="norm bwd 8192", kind="norm_bwd", act="bf16", res="bf16", rows=8192, c=1600, post=True, gate=True, groups=8),
        # A prompt of uneven length through a layer whose window is shorter than it.
        dict(name="attention prompt 333", kind="attn_fwd", b=4, h=12, hkv=12, tq=333, tk=333, hd=64, window=128, sinks=4),
        # GPT-2 small in training, a window of a quarter of the sequence.
        dict(name="attention step 1024", kind="attn_step", b=8, h=12, hkv=12, tq=1024, tk=1024, hd=64, window=256, sinks=4),
        # A long document in training with grouped heads.
        dict(name="attention step 8192", kind="attn_step", b=1, h=16, hkv=4, tq=8192, tk=8192, hd=128, window=2048, sinks=4),
        # Serving: one token of 32 sequences of uneven length, the window decides what is read.
        dict(name="decode 32", kind="attn_decode", b=32, h=12, hkv=12, cap=1024, hd=64, window=256, sinks=4),
        # Serving: few sequences, a long cache, every token visible, grouped heads.
        dict(name="decode long", kind="attn_decode", b=4, h=32, hkv=8, cap=65536, hd=128, window=0, sinks=0),
    ]


# ------------------------------------------------------------------------------ drawn cases

def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    hkv = rng.choice((1, 2, 3, 4, 8, 12))
    return hkv * rng.choice((1, 1, 2, 3, 4)), hkv


def _window(rng, t):
    """A window and its sinks: off, shorter than the sequence, or longer than it."""
    if rng.random() < 0.25:
        return 0, 0
    return _log(rng, 1, 2 * t + 1), rng.choice((0, 1, 4, 4, 16, 130))


def draw(rng):
    kind = rng.choice(("rope", "norm_fwd", "norm_bwd", "attn_fwd", "attn_step", "attn_decode"))
    if kind == "rope":
        hd = rng.choice((32, 64, 64, 80, 96, 128, 256))
        rot = hd if rng.random() < 0.5 else 2 * rng.randint(1, hd // 2)
        heads = rng.randint(1, 48)
        tokens = min(_log(rng, 1, 40000), 160_000_000 // (heads * hd))
        b = rng.randint(1, min(8, tokens))
        return dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp32")), b=b, t=max(1, tokens // b), heads=heads,
                    of=heads + rng.choice((0, 0, 1, heads)), hd=hd, rot=rot, interleaved=rng.random() < 0.5,
                    inverse=rng.random() < 0.5, far=rng.choice((0, 5, 4000, 1000000)), factor=rng.choice((1.0, 4.0, 8.0)))
    if kind in ("norm_fwd", "norm_bwd"):
        c = _log(rng, 17, 12800)
        step = rng.choice((64, 64, 8, 1))
        c = max(step, c // step * step)
        rows = min(_log(rng, 1, 16384), 13_000_000 // c)
        act, res = rng.choice((("bf16", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")))
        gate = rng.random() < 0.7
        groups = rng.choice([g for g in (1, 1, 2, 3, 5, 8, rows) if rows % g == 0 and g <= 1024]) if gate else 1
        return dict(kind=kind, act=act, res=res, rows=rows, c=c, post=rng.random() < 0.6, gate=gate, groups=groups)
    h, hkv = _heads(rng)
    hd = rng.choice((32, 64, 64, 72, 96, 128, 128))
    if kind == "attn_decode":
        b = _log(rng, 1, 64)
        cap = max(1, min(_log(rng, 1, 65536), 268_435_456 // (b * hkv * hd)))
        window, sinks = _window(rng, cap)
        return dict(kind=kind, b=b, h=h, hkv=hkv, cap=cap, hd=hd, window=window, sinks=sinks)
    # one visible key leaves nothing to differentiate: the gradients of q and k are zero but for their rounding
    tk = _log(rng, 2 if kind == "attn_step" else 1, 8192)
    b = max(1, min(rng.choice((1, 1, 2, 3, 8)), 1_000_000_000 // (h * tk * tk)))
    while h * tk * tk > 1_000_000_000:
        tk //= 2
    tq = tk if kind == "attn_step" or rng.random() < 0.6 else rng.randint(1, tk)
    window, sinks = _window(rng, tk)
    if kind == "attn_step" and window == 1:
        window = 2
    return dict(kind=kind, b=b, h=h, hkv=hkv, tq=tq, tk=tk, hd=hd, window=window, sinks=sinks)


# ------------------------------------------------------------------------------ inputs

def _normal(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _frequencies(case):
    """Radians per token of each pair, fp64: base 10000, slow ones slowed by `factor` for a context of that many times 1024."""
    f = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
    keep = ((1024 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return f * ((1 - keep) / case["factor"] + keep)


def _norm(z, eps=EPS):
    r = torch.rsqrt((z * z).mean(-1, keepdim=True) + eps)
    return z * r, r


def _gate_rows(case, gate):
    """The gate's row of each row of the data."""
    return gate.repeat_interleave(case["rows"] // case["groups"], 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case=case)
    k = case["kind"]
    if k == "rope":
        dt = DTYPES[case["dtype"]]
        rows = _normal(g, case["b"], case["t"], case["of"], case["hd"], dtype=dt)
        s["x"] = rows[:, :, :case["heads"]]
        s["y"] = torch.empty_like(rows)[:, :, :case["heads"]]
        s["freqs"] = _frequencies(case)
        # where each sequence stands: at its start in training, somewhere far in its context when it is served
        start = torch.randint(0, case["far"] + 1, (case["b"], 1), device="cuda", generator=g)
        s["positions"] = (start + torch.arange(case["t"], device="cuda")).to(torch.int32)
        s["scale"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        return s
    if k in ("norm_fwd", "norm_bwd"):
        act, res, rows, c = DTYPES[case["act"]], DTYPES[case["res"]], case["rows"], case["c"]
        x = _normal(g, rows, c, dtype=res, std=2.0)
        y = _normal(g, rows, c, dtype=act)
        s["w_post"] = 1 + _normal(g, c, std=0.1) if case["post"] else None
        s["w_pre"] = 1 + _normal(g, c, std=0.1)
        s["gate"] = _normal(g, case["groups"], c, std=0.3) if case["gate"] else None
        s["scale"] = 0.7
        if k == "norm_fwd":
            s.update(x=x, y=y, out=torch.empty_like(x), h=torch.empty_like(y), rstd_pre=torch.empty(rows, device="cuda"),
                     rstd_post=torch.empty(rows, device="cuda") if case["post"] else None)
            return s
        out, _, rstd_post, rstd_pre = _norm_plain(case, x, y, s["w_post"], s["gate"], s["w_pre"], s["scale"])
        s.update(y=y, out=out, rstd_post=rstd_post, rstd_pre=rstd_pre)
        s["dh"] = _normal(g, rows, c, dtype=act, std=1e-2)
        s["dout"] = _normal(g, rows, c, dtype=res, std=1e-2)
        s["dx"], s["dy"] = torch.empty_like(out), torch.empty_like(y)
        s["dw_post"] = torch.empty(c, device="cuda") if case["post"] else None
        s["dw_pre"] = torch.empty(c, device="cuda")
        s["dgate"] = torch.empty(case["groups"], c, device="cuda") if case["gate"] else None
        return s
    bf = torch.bfloat16
    h, hkv, hd, b = case["h"], case["hkv"], case["hd"], case["b"]
    if k == "attn_decode":
        cap = case["cap"]
        s["q"] = _normal(g, b, h, hd, dtype=bf)
        s["k"] = _normal(g, b, cap, hkv, hd, dtype=bf)
        s["v"] = _normal(g, b, cap, hkv, hd, dtype=bf)
        lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
        s["lengths"] = lengths[torch.randperm(b, device="cuda", generator=g)]
        s["out"] = torch.empty_like(s["q"])
        return s
    tq, tk = case["tq"], case["tk"]
    if tq == tk:   # out of the packed projection's token rows
        qkv = _normal(g, b, tk, h + 2 * hkv, hd, dtype=bf)
        s["q"], s["k"], s["v"] = qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]
    else:          # a later part of a prompt over the cache of the whole
        s["q"] = _normal(g, b, tq, h, hd, dtype=bf)
        s["k"], s["v"] = (_normal(g, b, tk, hkv, hd, dtype=bf) for _ in "kv")
    s["out"] = torch.empty(b, tq, h, hd, device="cuda", dtype=bf)
    s["lse"] = torch.empty(b, h, tq, device="cuda")
    if k == "attn_step":
        s["dout"] = _normal(g, b, tq, h, hd, dtype=bf, std=1e-2)
        dqkv = torch.empty(b, tk, h + 2 * hkv, hd, device="cuda", dtype=bf)
        s["dq"], s["dk"], s["dv"] = dqkv[:, :, :h], dqkv[:, :, h:h + hkv], dqkv[:, :, h + hkv:]
    return s


def _lengths(case):
    """The sequences' lengths, from a few tokens to a full cache; prepare() deals them out."""
    b, cap = case["b"], case["cap"]
    return [cap - (cap - 1) * i * 7 // (8 * b) for i in range(b)]


# ------------------------------------------------------------------------------ one pass

def run(s):
    return (_run_own if own else _run_plain)(s["case"]["kind"], s)


def _run_own(k, s):
    import llmt_b200 as L
    case = s["case"]
    if k == "rope":
        L.rope(s["y"], s["x"], s["freqs"], positions=s["positions"], interleaved=case["interleaved"], inverse=case["inverse"],
               scale=s["scale"])
        return s["y"]
    if k == "norm_fwd":
        L.norm_residual_fwd(s["out"], s["h"], s["x"], s["y"], w_post=s["w_post"], gate=s["gate"], w_pre=s["w_pre"],
                            rstd_post=s["rstd_post"], rstd_pre=s["rstd_pre"], scale=s["scale"], eps=EPS)
        return [s["out"], s["h"], s["rstd_post"], s["rstd_pre"]]
    if k == "norm_bwd":
        L.norm_residual_bwd(s["dx"], s["dy"], s["dout"], s["dh"], s["out"], s["y"], w_post=s["w_post"], gate=s["gate"],
                            w_pre=s["w_pre"], rstd_post=s["rstd_post"], rstd_pre=s["rstd_pre"], dw_post=s["dw_post"],
                            dgate=s["dgate"], dw_pre=s["dw_pre"], scale=s["scale"])
        return [s["dx"], s["dy"], s["dw_post"], s["dgate"], s["dw_pre"]]
    w = dict(window=case["window"], sinks=case["sinks"])
    if k == "attn_decode":
        L.attention_window_decode(s["out"], s["q"], s["k"], s["v"], lengths=s["lengths"], **w)
        return s["out"]
    L.attention_window_fwd(s["out"], s["lse"], s["q"], s["k"], s["v"], **w)
    if k == "attn_fwd":
        return [s["out"], s["lse"]]
    L.attention_window_bwd(s["dq"], s["dk"], s["dv"], s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], **w)
    return [s["out"], s["lse"], s["dq"], s["dk"], s["dv"]]


def _run_plain(k, s):
    case = s["case"]
    if k == "rope":
        return _rope_plain(case, s["x"], s["freqs"], s["positions"], s["scale"])
    if k == "norm_fwd":
        return list(_norm_plain(case, s["x"], s["y"], s["w_post"], s["gate"], s["w_pre"], s["scale"]))
    if k == "norm_bwd":
        return _norm_bwd_plain(case, s)
    q, kk, v = s["q"].float(), s["k"].float(), s["v"].float()
    if k == "attn_decode":
        n = s["lengths"][:, None]
        j = torch.arange(case["cap"], device="cuda")[None]
        seen = _visible(j, n - 1, case)[:, None, None, None]
        return _attend(q[:, None], kk, v, seen)[0][:, 0].to(torch.bfloat16)
    i = torch.arange(case["tq"], device="cuda")[:, None] + case["tk"] - case["tq"]
    seen = _visible(torch.arange(case["tk"], device="cuda")[None], i, case)
    o, lse, p = _attend(q, kk, v, seen)
    if k == "attn_fwd":
        return [o.to(torch.bfloat16), lse]
    return [o.to(torch.bfloat16), lse] + _attend_bwd(s["dout"].float(), q, kk, v, o, p)


def _rope_plain(case, x, freqs, positions, scale):
    a = positions.double()[..., None, None] * freqs
    c, n = (a.cos() * scale).float(), (a.sin() * scale).float()
    if case["inverse"]:
        n = -n
    x = x.float()
    r = case["rot"]
    if case["interleaved"]:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((u * c - w * n, u * n + w * c), -1).flatten(-2)
    else:
        u, w = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((u * c - w * n, u * n + w * c), -1)
    return torch.cat((turned, x[..., r:]), -1).to(DTYPES[case["dtype"]])


def _norm_plain(case, x, y, w_post, gate, w_pre, scale):
    n, rstd_post = y.float(), None
    if w_post is not None:
        n, rstd_post = _norm(n)
        n = n * w_post
    if gate is not None:
        n = n * _gate_rows(case, gate)
    out = x.float() + scale * n
    h, rstd_pre = _norm(out)
    return (out.to(x.dtype), (h * w_pre).to(y.dtype), None if rstd_post is None else rstd_post[:, 0], rstd_pre[:, 0])


def _norm_bwd_plain(case, s):
    out, y, dh, dout = (s[n].float() for n in ("out", "y", "dh", "dout"))
    r = s["rstd_pre"][:, None]
    hat, a = out * r, dh * s["w_pre"]
    dx = dout + r * (a - hat * (a * hat).mean(-1, keepdim=True))
    dw_pre = (dh * hat).sum(0)
    dn = dx * s["scale"]
    u, dw_post, dgate = y, None, None
    if s["w_post"] is not None:
        r = s["rstd_post"][:, None]
        hat = y * r
        u = hat * s["w_post"]
    if s["gate"] is not None:
        dgate = (dn * u).view(case["groups"], -1, case["c"]).sum(1)
        dn = dn * _gate_rows(case, s["gate"])
    dy = dn
    if s["w_post"] is not None:
        dw_post = (dn * hat).sum(0)
        a = dn * s["w_post"]
        dy = r * (a - hat * (a * hat).mean(-1, keepdim=True))
    return [dx.to(s["dx"].dtype), dy.to(s["dy"].dtype), dw_post, dgate, dw_pre]


def _visible(j, p, case):
    """Whether the query at position p sees key j."""
    seen = j <= p
    if case["window"] > 0:
        seen = seen & ((j > p - case["window"]) | (j < case["sinks"]))
    return seen


def _by_group(x, hkv):
    """[B, T, H, hd] as [B, Hkv, heads of the group, T, hd]."""
    b, t, h, hd = x.shape
    return x.view(b, t, hkv, h // hkv, hd).permute(0, 2, 3, 1, 4)


def _by_token(x):
    b, hkv, g, t, hd = x.shape
    return x.permute(0, 3, 1, 2, 4).reshape(b, t, hkv * g, hd)


def _attend(q, k, v, seen):
    hkv, scale = k.shape[2], 1 / math.sqrt(q.shape[-1])
    q, k, v = _by_group(q.contiguous(), hkv), _by_group(k.contiguous(), hkv), _by_group(v.contiguous(), hkv)
    p = (q @ k.transpose(-1, -2)).mul_(scale)
    p.masked_fill_(~seen, -math.inf)
    m = p.amax(-1, keepdim=True)
    m.masked_fill_(m == -math.inf, 0)
    p.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(total.clamp(min=1e-30))
    return _by_token(p @ v), (m + total.log())[..., 0].flatten(1, 2), p


def _attend_bwd(do, q, k, v, o, p):
    hkv, scale = k.shape[2], 1 / math.sqrt(q.shape[-1])
    d = _by_group((do * o).sum(-1, keepdim=True), hkv)
    do, q, k, v = (_by_group(x.contiguous(), hkv) for x in (do, q, k, v))
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    ds = (do @ v.transpose(-1, -2)).sub_(d).mul_(p).mul_(scale)
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return [_by_token(x).to(torch.bfloat16) for x in (ds @ k, dk, dv)]


# ------------------------------------------------------------------------------ what a pass cannot do without

def _pairs(case):
    """Visible (query, key) pairs of one head."""
    w = case["window"] if case["window"] > 0 else case["tk"] + 1
    n = 0
    for p in range(case["tk"] - case["tq"], case["tk"]):
        recent = max(0, p - w + 1)
        n += p + 1 - recent + min(case["sinks"], recent)
    return n


def work(case):
    k = case["kind"]
    if k == "rope":
        n = case["b"] * case["t"] * case["heads"]
        size = DTYPES[case["dtype"]].itemsize
        return dict(bytes=2 * n * case["hd"] * size + 4 * case["b"] * case["t"] + 4 * case["rot"], flops=3 * n * case["rot"])
    if k in ("norm_fwd", "norm_bwd"):
        n, c = case["rows"] * case["c"], case["c"]
        a, r = DTYPES[case["act"]].itemsize, DTYPES[case["res"]].itemsize
        vectors = 4 * c * (1 + case["post"] + (case["groups"] if case["gate"] else 0))
        stats = 4 * case["rows"] * (1 + case["post"])
        if k == "norm_fwd":
            return dict(bytes=n * 2 * (a + r) + vectors + stats, flops=12 * n)
        return dict(bytes=n * 3 * (a + r) + 2 * vectors + stats, flops=24 * n)
    h, hkv, hd, b = case["h"], case["hkv"], case["hd"], case["b"]
    if k == "attn_decode":
        w = case["window"]
        seen = [n if w <= 0 else min(n, w) + min(case["sinks"], max(0, n - w)) for n in _lengths(case)]
        return dict(bytes=2 * (2 * sum(seen) * hkv * hd + 2 * b * h * hd) + 4 * b, flops=4 * sum(seen) * h * hd)
    nq, nk, pairs = b * case["tq"] * h * hd, b * case["tk"] * hkv * hd, b * h * _pairs(case)
    if k == "attn_fwd":
        return dict(bytes=2 * (2 * nq + 2 * nk) + 4 * nq // hd, flops=4 * hd * pairs)
    return dict(bytes=2 * (4 * nq + 4 * nk) + 4 * nq // hd, flops=14 * hd * pairs)


# ------------------------------------------------------------------------------ the definitions in fp64

def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k == "rope":
        x, r = s["x"].double(), case["rot"]
        angle = s["positions"].double()[:, :, None, None] * s["freqs"] * (-1 if case["inverse"] else 1)
        unit = torch.complex(angle.cos(), angle.sin()) * s["scale"]
        if case["interleaved"]:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * unit
            x[..., 0:r:2], x[..., 1:r:2] = z.real, z.imag
        else:
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * unit
            x[..., :r // 2], x[..., r // 2:r] = z.real, z.imag
        return x
    if k in ("norm_fwd", "norm_bwd"):
        return _norm_exact(case, s)
    if k == "attn_decode":
        return _decode_exact(case, s)
    return _attention_exact(case, s)


def _norm_exact(case, s):
    c, per = case["c"], case["rows"] // case["groups"]
    d = {n: None if s.get(n) is None else s[n].double() for n in ("x", "y", "out", "dh", "dout", "w_post", "w_pre", "gate",
                                                                   "rstd_post", "rstd_pre")}
    gate = torch.ones(case["groups"], c, device="cuda", dtype=torch.float64) if d["gate"] is None else d["gate"]
    which = torch.arange(case["rows"], device="cuda") // per
    if case["kind"] == "norm_fwd":
        u, rp = d["y"], None
        if case["post"]:
            rp = (u.square().sum(-1) / c + EPS).pow(-0.5)
            u = u * rp[:, None] * d["w_post"]
        out = d["x"] + s["scale"] * gate[which] * u
        rs = (out.square().sum(-1) / c + EPS).pow(-0.5)
        return [out, out * rs[:, None] * d["w_pre"], rp, rs]

    def back(z, rstd, w, grad):   # of z * rstd(z) * w
        return rstd[:, None] * w * grad - z * (rstd.pow(3) * (grad * w * z).sum(-1) / c)[:, None]

    dx = d["dout"] + back(d["out"], d["rstd_pre"], d["w_pre"], d["dh"])
    dw_pre = (d["rstd_pre"][:, None] * d["out"] * d["dh"]).sum(0)
    du = s["scale"] * gate[which] * dx
    if case["post"]:
        u = d["y"] * d["rstd_post"][:, None]
        dw_post, dy = (du * u).sum(0), back(d["y"], d["rstd_post"], d["w_post"], du)
        u = u * d["w_post"]
    else:
        u, dw_post, dy = d["y"], None, du
    dgate = None
    if case["gate"]:
        dgate = torch.zeros_like(gate).index_add_(0, which, s["scale"] * dx * u)
    return [dx, dy, dw_post, dgate, dw_pre]


def _decode_exact(case, s):
    g = case["h"] // case["hkv"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    for i, n in enumerate(s["lengths"].tolist()):
        at = torch.arange(n, device="cuda")
        if case["window"] > 0:
            at = at[(at >= n - case["window"]) | (at < case["sinks"])]
        for h in range(case["h"]):
            kk, v = s["k"][i, at, h // g].double(), s["v"][i, at, h // g].double()
            out[i, h] = torch.softmax(kk @ s["q"][i, h].double() / math.sqrt(case["hd"]), 0) @ v
    return out


def _attention_exact(case, s):
    b, h, hkv, tq, tk, hd = (case[n] for n in ("b", "h", "hkv", "tq", "tk", "hd"))
    at = torch.arange(tk, device="cuda")
    p = torch.arange(tk - tq, tk, device="cuda")[:, None]
    hidden = at > p
    if case["window"] > 0:
        hidden |= (at <= p - case["window"]) & (at >= case["sinks"])
    new = lambda n, t: torch.zeros(b, t, n, hd, device="cuda", dtype=torch.float64)  # noqa: E731
    out, lse = new(h, tq), torch.zeros(b, h, tq, device="cuda", dtype=torch.float64)
    step = case["kind"] == "attn_step"
    dq, dk, dv = (new(h, tq), new(hkv, tk), new(hkv, tk)) if step else (None, None, None)
    for i in range(b):
        for n in range(h):
            q, k, v = s["q"][i, :, n].double(), s["k"][i, :, n * hkv // h].double(), s["v"][i, :, n * hkv // h].double()
            a = (q @ k.T / math.sqrt(hd)).masked_fill_(hidden, -math.inf)
            lse[i, n] = torch.logsumexp(a, -1)
            a = torch.exp(a - lse[i, n, :, None])
            out[i, :, n] = a @ v
            if step:
                do = s["dout"][i, :, n].double()
                dv[i, :, n * hkv // h] += a.T @ do
                da = do @ v.T
                da = a * (da - (da * a).sum(-1, keepdim=True)) / math.sqrt(hd)
                dq[i, :, n] = da @ k
                dk[i, :, n * hkv // h] += da.T @ q
    return [out, lse, dq, dk, dv] if step else [out, lse]
