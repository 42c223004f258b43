"""The norms around a block with its gate and residual, against the formulas in 64 bits and against differences."""
import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5
TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)]


def _inputs(rows, cols, res, act, groups, post, gate, pre, seed=0):
    g = torch.Generator(device=DEV).manual_seed(rows * 7919 + cols + seed)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)
    return dict(x=n(rows, cols).to(res), y=n(rows, cols).to(act), w_post=1 + 0.1 * n(cols) if post else None,
                gate=0.5 * n(groups, cols) if gate else None, w_pre=1 + 0.1 * n(cols) if pre else None,
                dout=n(rows, cols).to(res), dh=n(rows, cols).to(act) if pre else None)


def _forward(d, scale, rows, groups):
    """out, h, rstd_post, rstd_pre in fp64, differentiable in what requires it."""
    u, rp, rs, h = d["y"], None, None, None
    if d["w_post"] is not None:
        rp = (u.square().mean(-1) + EPS).rsqrt()
        u = u * rp[:, None] * d["w_post"]
    if d["gate"] is not None:
        u = u * d["gate"].repeat_interleave(rows // groups, 0)
    out = d["x"] + scale * u
    if d["w_pre"] is not None:
        rs = (out.square().mean(-1) + EPS).rsqrt()
        h = out * rs[:, None] * d["w_pre"]
    return out, h, rp, rs


def _close(got, want, slack, size, what):
    """Half a step of the result's type, and `slack` fp32 roundings of terms of the given size."""
    bound = want.abs() * torch.finfo(got.dtype).eps / 2 + slack * 2.0 ** -24 * size
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off / bound).max()):.2f} of the bound"


SHAPES = [(1, 1, 1), (3, 5, 3), (7, 64, 1), (33, 771, 1), (20, 256, 4), (16, 768, 2), (9, 1600, 3), (5, 2049, 1), (6, 4096, 2), (4, 4104, 2),
          (3, 9001, 1), (2, 16384, 1)]


@pytest.mark.parametrize("res,act", TYPES)
@pytest.mark.parametrize("rows,cols,groups", SHAPES)
@pytest.mark.parametrize("post,gate,pre", [(True, True, True), (False, True, True), (True, False, False), (False, False, True)])
def test_forward_and_backward(rows, cols, groups, res, act, post, gate, pre):
    scale = 0.7
    d = _inputs(rows, cols, res, act, groups, post, gate, pre)
    wide = {k: None if v is None else v.double() for k, v in d.items()}
    groups = groups if gate else 1
    ref = _forward(wide, scale, rows, groups)
    out = torch.full_like(d["x"], 3.0)
    h = torch.full_like(d["y"], 3.0) if pre else None
    rp, rs = (torch.empty(rows, device=DEV) if on else None for on in (post, pre))
    w = dict(w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"], rstd_post=rp, rstd_pre=rs, scale=scale)
    L.norm_residual_fwd(out, h, d["x"], d["y"], eps=EPS, **w)
    # a row's sum of squares: cols products added in a tree of depth 13 over runs of up to 32: 45 roundings at most,
    # all of one sign, halved by the square root; then a handful of products
    _close(out, ref[0], 32, wide["x"].abs() + (ref[0] - wide["x"]).abs(), "out")
    if post:
        _close(rp, ref[2], 32, ref[2], "rstd_post")
    if pre:
        _close(rs, ref[3], 64, ref[3] * (1 + (wide["x"].abs() + (ref[0] - wide["x"]).abs()).square().mean(-1) * ref[3].square()), "rstd_pre")
        _close(h, ref[1], 128, ref[1].abs() + (wide["x"].abs() + (ref[0] - wide["x"]).abs()) * ref[3][:, None] * wide["w_pre"].abs(), "h")
    where = d["x"].clone()
    L.norm_residual_fwd(where, h.clone() if pre else None, where, d["y"], eps=EPS, **w)
    assert torch.equal(where, out), "in place"

    # backward, from what the forward pass stored
    dx, dy = torch.full_like(out, 3.0), torch.full_like(d["y"], 3.0)
    dw = dict(dw_post=torch.full((cols,), 2.0, device=DEV) if post else None, dgate=torch.full((groups, cols), 2.0, device=DEV) if gate else None,
              dw_pre=torch.full((cols,), 2.0, device=DEV) if pre else None)
    L.norm_residual_bwd(dx, dy, d["dout"], d["dh"], out, d["y"], beta=0.5, **w, **dw)
    o, y, dout = out.double(), wide["y"], wide["dout"]
    gt = torch.ones(rows, cols, device=DEV, dtype=torch.float64) if not gate else wide["gate"].repeat_interleave(rows // groups, 0)
    gdx, size = dout, dout.abs()
    if pre:
        r, a = rs.double()[:, None], wide["dh"] * wide["w_pre"]
        b = o * r
        gdx = dout + r * (a - b * (a * b).mean(-1, keepdim=True))
        size = dout.abs() + r * (a.abs() + b.abs() * (a * b).abs().mean(-1, keepdim=True))
    _close(dx, gdx, 64, size, "dx")
    k = scale * gt * (wide["w_post"] if post else 1)
    if post:
        r = rp.double()[:, None]
        c = y * r
        gdy = r * (k * gdx - c * (k * gdx * c).mean(-1, keepdim=True))
        # the sums over a row are of the terms of gdx, each to be counted by itself
        sdy = r * (k.abs() * size + c.abs() * (k.abs() * size * c.abs()).mean(-1, keepdim=True))
    else:
        c, gdy, sdy = y, k * gdx, k.abs() * size
    _close(dy, gdy, 160, sdy, "dy")
    # sums over rows: each term carries its own roundings, then a chain of fewer than 64 + 32 additions here
    if pre:
        t = wide["dh"] * o * rs.double()[:, None]
        _close(dw["dw_pre"], 1.0 + t.sum(0), 100, 1 + t.abs().sum(0), "dw_pre")
    if post:
        _close(dw["dw_post"], 1.0 + (scale * gt * gdx * c).sum(0), 200, 1 + (gt.abs() * size * c.abs()).sum(0), "dw_post")
    if gate:
        t = scale * gdx * c * (wide["w_post"] if post else 1)
        s = size * c.abs() * (wide["w_post"].abs() if post else 1)
        _close(dw["dgate"], 1.0 + t.view(groups, -1, cols).sum(1), 200, 1 + s.view(groups, -1, cols).sum(1), "dgate")
    again = {n: None if v is None else torch.full_like(v, 2.0) for n, v in dw.items()}
    dx2, dy2 = d["dout"].clone(), torch.empty_like(dy)
    L.norm_residual_bwd(dx2, dy2, dx2, d["dh"], out, d["y"], beta=0.5, **w, **again)
    assert torch.equal(dx2, dx) and torch.equal(dy2, dy), "dx may be dout"
    assert all(v is None or torch.equal(v, dw[n]) for n, v in again.items()), "the same bits on every run"


@pytest.mark.parametrize("rows,cols,groups", [(600, 96, 3), (4000, 40, 1), (1000, 33, 1000)])
def test_many_rows_share_the_weight_gradients(rows, cols, groups):
    d = _inputs(rows, cols, torch.float32, torch.float32, groups, True, True, True)
    out, h = torch.empty_like(d["x"]), torch.empty_like(d["y"])
    rp, rs = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    w = dict(w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"], rstd_post=rp, rstd_pre=rs)
    L.norm_residual_fwd(out, h, d["x"], d["y"], eps=EPS, **w)
    leaves = {k: v.double().requires_grad_() for k, v in d.items() if k not in ("dout", "dh")}
    o, hh, _, _ = _forward(dict(leaves, dout=None, dh=None), 1.0, rows, groups)
    ((o * d["dout"].double()).sum() + (hh * d["dh"].double()).sum()).backward()
    dx, dy = torch.empty_like(out), torch.empty_like(h)
    dw = {n: torch.full_like(d[n], float("nan")) for n in ("w_post", "gate", "w_pre")}
    L.norm_residual_bwd(dx, dy, d["dout"], d["dh"], out, d["y"], dw_post=dw["w_post"], dgate=dw["gate"], dw_pre=dw["w_pre"], **w)
    for n, got in (("x", dx), ("y", dy), *dw.items()):
        want = leaves[n].grad
        # against the whole chain, out and the statistics rounded to fp32 in between: 256 roundings relative to the norm
        assert float((got.double() - want).norm() / want.norm()) <= 256 * 2.0 ** -24, n


def test_gradients_match_differences():
    rows, cols = 4, 24
    d = _inputs(rows, cols, torch.float32, torch.float32, 2, True, True, True)

    def loss(**other):
        e = {**d, **other}
        out, h = torch.empty_like(d["x"]), torch.empty_like(d["y"])
        L.norm_residual_fwd(out, h, e["x"], e["y"], w_post=e["w_post"], gate=e["gate"], w_pre=e["w_pre"], scale=0.8)
        return float((out.double() * d["dout"].double()).sum() + (h.double() * d["dh"].double()).sum())

    out, h, rp, rs = torch.empty_like(d["x"]), torch.empty_like(d["y"]), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    w = dict(w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"], rstd_post=rp, rstd_pre=rs, scale=0.8)
    L.norm_residual_fwd(out, h, d["x"], d["y"], **w)
    g = dict(x=torch.empty_like(out), y=torch.empty_like(h), w_post=torch.empty(cols, device=DEV), gate=torch.empty(2, cols, device=DEV),
             w_pre=torch.empty(cols, device=DEV))
    L.norm_residual_bwd(g["x"], g["y"], d["dout"], d["dh"], out, d["y"], dw_post=g["w_post"], dgate=g["gate"], dw_pre=g["w_pre"], **w)
    for name, grad in g.items():
        way = torch.randn(d[name].shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
        e = 2.0 ** -7
        slope = (loss(**{name: d[name] + e * way}) - loss(**{name: d[name] - e * way})) / (2 * e)
        # third derivatives of order 1 times e^2 / 6, and roundings of 200 terms of order 1 over 2 e: 1e-5 + 2e-3 at most
        assert abs(slope - float((grad.double() * way.double()).sum())) <= 3e-3 * float(grad.norm() * way.norm() + 1)


def test_without_a_block_and_without_a_residual_gradient():
    rows, cols = 6, 100
    d = _inputs(rows, cols, torch.float32, torch.bfloat16, 1, False, False, True)
    h, rs = torch.empty_like(d["y"]), torch.empty(rows, device=DEV)
    L.norm_residual_fwd(None, h, d["x"], w_pre=d["w_pre"], rstd_pre=rs)
    x = d["x"].double()
    r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    _close(h, x * r * d["w_pre"].double(), 64, (x * r).abs(), "h")
    dx, dw = torch.empty_like(d["x"]), torch.empty(cols, device=DEV)
    L.norm_residual_bwd(dx, None, None, d["dh"], d["x"], w_pre=d["w_pre"], rstd_pre=rs, dw_pre=dw)
    a, b = d["dh"].double() * d["w_pre"].double(), x * r
    want = r * (a - b * (a * b).mean(-1, keepdim=True))
    _close(dx, want, 64, r * (a.abs() + b.abs() * (a * b).abs().mean(-1, keepdim=True)), "dx")
    t = d["dh"].double() * b
    _close(dw, t.sum(0), 64, t.abs().sum(0), "dw_pre")


def test_a_row_of_zeros_and_rows_that_are_not_finite_stay_their_own():
    rows, cols = 40, 96
    d = _inputs(rows, cols, torch.float32, torch.float32, 1, True, True, True)
    d["x"][3] = 0
    d["y"][3] = 0
    d["x"][5, 7] = float("nan")
    d["y"][9, 0] = float("inf")
    out, h, rp, rs = torch.empty_like(d["x"]), torch.empty_like(d["y"]), torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    L.norm_residual_fwd(out, h, d["x"], d["y"], w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"], rstd_post=rp, rstd_pre=rs)
    assert bool((out[3] == 0).all()) and bool((h[3] == 0).all()) and bool(torch.isfinite(rs[3]))
    others = [r for r in range(rows) if r not in (5, 9)]
    assert bool(torch.isfinite(h[others]).all()) and bool(torch.isnan(h[5]).all()) and bool(torch.isnan(h[9]).any())
    dx, dy = torch.empty_like(out), torch.empty_like(h)
    L.norm_residual_bwd(dx, dy, d["dout"], d["dh"], out, d["y"], w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"], rstd_post=rp, rstd_pre=rs)
    assert bool(torch.isfinite(dx[others]).all()) and bool(torch.isfinite(dy[others]).all())


def test_pitches_other_streams_and_a_captured_call():
    rows, cols = 37, 72
    wide = torch.randn(4, rows, 100, device=DEV)
    d = _inputs(rows, cols, torch.float32, torch.float32, 1, True, True, True)
    x, y, out, h = (wide[i, :, 13:13 + cols] for i in range(4))
    x.copy_(d["x"]); y.copy_(d["y"])
    guard = wide.clone()
    w = dict(w_post=d["w_post"], gate=d["gate"], w_pre=d["w_pre"])
    o, hh = torch.empty_like(d["x"]), torch.empty_like(d["y"])
    L.norm_residual_fwd(o, hh, d["x"], d["y"], **w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    L.norm_residual_fwd(out, h, x, y, stream=side, **w)
    side.synchronize()
    half = 4 * 2.0 ** -24   # the two layouts add a row's squares in another order
    assert torch.allclose(out, o, rtol=half, atol=1e-6) and torch.allclose(h, hh, rtol=1e-5, atol=1e-6)
    wide[2:, :, 13:13 + cols] = guard[2:, :, 13:13 + cols]
    assert torch.equal(wide, guard), "nothing outside the rows is written"
    rp, rs = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    dx, dy, dw = torch.empty_like(o), torch.empty_like(o), torch.zeros(cols, device=DEV)
    ws = torch.empty(L.norm_residual_workspace_bytes(rows, cols), dtype=torch.uint8, device=DEV)

    def step():
        L.norm_residual_fwd(o, hh, d["x"], d["y"], rstd_post=rp, rstd_pre=rs, **w)
        L.norm_residual_bwd(dx, dy, d["dout"], d["dh"], o, d["y"], rstd_post=rp, rstd_pre=rs, dw_pre=dw, beta=1.0, workspace=ws, **w)
    step()
    torch.cuda.synchronize()
    once, first = dw.clone(), dx.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    dx.zero_()
    graph.replay()
    assert torch.equal(dx, first) and torch.allclose(dw, 2 * once, rtol=2.0 ** -22)
    del graph


def test_no_rows():
    e = torch.empty(0, 8, device=DEV)
    w = torch.ones(8, device=DEV)
    L.norm_residual_fwd(e, e.clone(), e.clone(), e.clone(), w_post=w, w_pre=w)
    dw = torch.full((8,), 5.0, device=DEV)
    s = torch.empty(0, device=DEV)
    L.norm_residual_bwd(e, e.clone(), e.clone(), e.clone(), e.clone(), e.clone(), w_pre=w, rstd_pre=s, dw_pre=dw)
    assert bool((dw == 0).all())
