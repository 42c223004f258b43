"""The block operators in the order in which a transformer block has them, with the products between them: norm -> QKV
product -> rotary positions inside the packed rows -> windowed attention -> output product -> norm, gate and residual, forward
and backward, against the same block in 64 bits with automatic differentiation; captured into a graph; two blocks at once on
two streams; then one token at a time over a cache against the same block over all tokens."""
import pytest
import torch

import llmt_b200 as L

pytestmark = pytest.mark.gpu

B, T, C, H, HKV, HD, ROT, WINDOW, SINKS = 2, 160, 256, 4, 2, 64, 32, 70, 3
W = (H + 2 * HKV) * HD
EPS, SCALE = 1e-5, 0.5


class Block:
    """One attention block with buffers of its own; x fp32, everything inside bf16."""

    def __init__(self, seed, batch=B, tokens=T):
        g = torch.Generator(device="cuda").manual_seed(seed)
        bf = lambda *s, k=1.0: (k * torch.randn(*s, device="cuda", generator=g)).to(torch.bfloat16)
        f32 = lambda *s, base=0.0, k=0.3: base + k * torch.randn(*s, device="cuda", generator=g)
        self.wqkv, self.wo = bf(W, C, k=C ** -0.5), bf(C, H * HD, k=(H * HD) ** -0.5)
        self.w_in, self.w_post, self.gate, self.w_pre = f32(C, base=1.0), f32(C, base=1.0), f32(batch, C, base=1.0), f32(C, base=1.0)
        self.x, self.dout, self.dh = f32(batch, tokens, C, k=1.0), f32(batch, tokens, C, k=1.0), bf(batch, tokens, C)
        self.freqs = L.rope_frequencies(ROT)
        n = batch * tokens
        e16 = lambda *s: torch.full(s, float("nan"), device="cuda", dtype=torch.bfloat16)
        e32 = lambda *s: torch.full(s, float("nan"), device="cuda")
        self.hin, self.qkv, self.att, self.y, self.h = e16(batch, tokens, C), e16(batch, tokens, W), e16(batch, tokens, H * HD), e16(batch, tokens, C), e16(batch, tokens, C)
        self.out, self.lse, self.r_in, self.r_post, self.r_pre = e32(batch, tokens, C), e32(batch, H, tokens), e32(n), e32(n), e32(n)
        self.dx, self.dy, self.datt, self.dqkv, self.dhin = e32(batch, tokens, C), e16(batch, tokens, C), e16(batch, tokens, H * HD), e16(batch, tokens, W), e16(batch, tokens, C)
        self.dw_in, self.dw_post, self.dgate, self.dw_pre = e32(C), e32(C), e32(batch, C), e32(C)
        self.dwqkv, self.dwo = e32(W, C), e32(C, H * HD)

    def split(self, t):
        heads = t.view(t.shape[0], t.shape[1], H + 2 * HKV, HD)
        return heads[:, :, :H], heads[:, :, H:H + HKV], heads[:, :, H + HKV:]

    def forward(self, stream=None):
        two = lambda t: t.view(-1, t.shape[-1])
        L.norm_residual_fwd(None, self.hin, self.x, w_pre=self.w_in, rstd_pre=self.r_in, eps=EPS, stream=stream)
        L.gemm(two(self.qkv), two(self.hin), self.wqkv, trans_b=True, stream=stream)
        turn = self.qkv.view(*self.qkv.shape[:2], H + 2 * HKV, HD)[:, :, :H + HKV]
        L.rope(turn, turn, self.freqs, stream=stream)
        q, k, v = self.split(self.qkv)
        L.attention_window_fwd(self.att.view(*q.shape), self.lse, q, k, v, window=WINDOW, sinks=SINKS, stream=stream)
        L.gemm(two(self.y), two(self.att), self.wo, trans_b=True, stream=stream)
        L.norm_residual_fwd(self.out, self.h, self.x, self.y, w_post=self.w_post, gate=self.gate, w_pre=self.w_pre, rstd_post=self.r_post,
                            rstd_pre=self.r_pre, scale=SCALE, eps=EPS, stream=stream)

    def backward(self, stream=None):
        two = lambda t: t.view(-1, t.shape[-1])
        L.norm_residual_bwd(self.dx, self.dy, self.dout, self.dh, self.out, self.y, w_post=self.w_post, gate=self.gate, w_pre=self.w_pre,
                            rstd_post=self.r_post, rstd_pre=self.r_pre, dw_post=self.dw_post, dgate=self.dgate, dw_pre=self.dw_pre, scale=SCALE,
                            stream=stream)
        L.gemm(two(self.datt), two(self.dy), self.wo, stream=stream)
        L.gemm(self.dwo, two(self.dy), two(self.att), trans_a=True, stream=stream)
        q, k, v = self.split(self.qkv)
        dq, dk, dv = self.split(self.dqkv)
        L.attention_window_bwd(dq, dk, dv, self.datt.view(*q.shape), q, k, v, self.att.view(*q.shape), self.lse, window=WINDOW, sinks=SINKS, stream=stream)
        turn = self.dqkv.view(*self.dqkv.shape[:2], H + 2 * HKV, HD)[:, :, :H + HKV]
        L.rope(turn, turn, self.freqs, inverse=True, stream=stream)
        L.gemm(two(self.dhin), two(self.dqkv), self.wqkv, stream=stream)
        L.gemm(self.dwqkv, two(self.dqkv), two(self.hin), trans_a=True, stream=stream)
        L.norm_residual_bwd(self.dx, None, self.dx, self.dhin, self.x, w_pre=self.w_in, rstd_pre=self.r_in, dw_pre=self.dw_in, stream=stream)

    def results(self):
        return {n: getattr(self, n) for n in ("out", "h", "dx", "dw_in", "dw_post", "dgate", "dw_pre", "dwqkv", "dwo")}


def plain(blk):
    """The block and its gradients in 64 bits."""
    d = lambda t: t.double().requires_grad_()
    x, w_in, w_post, gate, w_pre, wqkv, wo = (d(t) for t in (blk.x, blk.w_in, blk.w_post, blk.gate, blk.w_pre, blk.wqkv, blk.wo))
    b, t = x.shape[:2]
    norm = lambda z, w: z * (z.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w
    qkv = (norm(x, w_in) @ wqkv.t()).view(b, t, H + 2 * HKV, HD)
    angle = torch.arange(t, device="cuda", dtype=torch.float64)[:, None] * blk.freqs
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    u, w = qkv[:, :, :H + HKV, :ROT // 2], qkv[:, :, :H + HKV, ROT // 2:ROT]
    qk = torch.cat((u * c - w * s, u * s + w * c, qkv[:, :, :H + HKV, ROT:]), -1)
    q, k, v = qk[:, :, :H], qk[:, :, H:].repeat_interleave(H // HKV, 2), qkv[:, :, H + HKV:].repeat_interleave(H // HKV, 2)
    i, j = torch.arange(t, device="cuda")[:, None], torch.arange(t, device="cuda")
    seen = (j <= i) & ((j > i - WINDOW) | (j < SINKS))
    p = (torch.einsum("bihd,bjhd->bhij", q, k) * HD ** -0.5).masked_fill(~seen, float("-inf")).softmax(-1)
    att = torch.einsum("bhij,bjhd->bihd", p, v).reshape(b, t, H * HD)
    out = x + SCALE * gate[:, None] * norm(att @ wo.t(), w_post)
    h = norm(out, w_pre)
    leaves = dict(dx=x, dw_in=w_in, dw_post=w_post, dgate=gate, dw_pre=w_pre, dwqkv=wqkv, dwo=wo)
    grads = torch.autograd.grad((out * blk.dout.double()).sum() + (h * blk.dh.double()).sum(), list(leaves.values()))
    return dict(out=out.detach(), h=h.detach(), **dict(zip(leaves, grads)))


def test_the_block_and_its_gradients():
    """A result is behind at most 14 roundings to bf16 (forward hin, qkv, turned qkv, P, att, y, h; backward dy, datt, dS, dq
    or dk, turned dqkv, dhin, and the rounding of out's copy in D), each off by at most 2^-8 of its value, and the products
    between them (random matrices of row norm 1) and norms pass a relative error on at its size: 14 * 2^-8 = 5.5 % of a
    result's norm.  `out` has x, which is not rounded, beside what is."""
    blk = Block(1)
    blk.forward()
    blk.backward()
    want = plain(blk)
    for name, got in blk.results().items():
        err = (got.double() - want[name]).norm() / want[name].norm()
        assert err <= 14 * 2.0 ** -8, (name, float(err))
        assert bool(torch.isfinite(got).all()), name


def test_the_block_in_a_graph_and_on_two_streams():
    """A replay, and two blocks under way at once on two streams, give the eager results to the bit, with inputs changed in
    between."""
    one, two = Block(2), Block(3)
    fresh = torch.randn_like(one.x)
    eager = {}
    for blk, key in ((one, "one"), (two, "two")):
        blk.forward()
        blk.backward()
        eager[key] = {n: t.clone() for n, t in blk.results().items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one.forward()
        one.backward()
    x = one.x.clone()
    one.x.copy_(fresh)
    graph.replay()
    assert not torch.equal(one.out, eager["one"]["out"])
    one.x.copy_(x)
    graph.replay()
    for n, t in one.results().items():
        assert torch.equal(t, eager["one"][n]), n
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for blk in (one, two):
        for t in blk.results().values():
            t.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(3):
        for blk, s in zip((one, two), streams):
            blk.forward(stream=s)
            blk.backward(stream=s)
    torch.cuda.synchronize()
    for blk, key in ((one, "one"), (two, "two")):
        for n, t in blk.results().items():
            assert torch.equal(t, eager[key][n]), (key, n)
    del graph


def test_token_by_token_over_a_cache():
    """Each new token through the operators, its k and v into a cache, gives the rows that the whole sequence gives: both
    are off from the exact block by at most 7 forward roundings (above), so from one another by twice that."""
    blk = Block(4)
    blk.forward()
    places = T + 5
    kc = torch.full((B, places, HKV, HD), float("nan"), device="cuda", dtype=torch.bfloat16)
    vc = kc.clone()
    step = Block(4, tokens=1)
    for n in ("wqkv", "wo", "w_in", "w_post", "gate", "w_pre"):
        setattr(step, n, getattr(blk, n))
    ws = torch.empty(max(16, L.attention_window_decode_workspace_bytes(step.qkv[:, 0, :H * HD].view(B, H, HD), kc, WINDOW, SINKS)), dtype=torch.uint8, device="cuda")
    for t in range(T):
        step.x.copy_(blk.x[:, t:t + 1])
        two = lambda z: z.view(-1, z.shape[-1])
        L.norm_residual_fwd(None, step.hin, step.x, w_pre=step.w_in, rstd_pre=step.r_in, eps=EPS)
        L.gemm(two(step.qkv), two(step.hin), step.wqkv, trans_b=True)
        turn = step.qkv.view(B, 1, H + 2 * HKV, HD)[:, :, :H + HKV]
        L.rope(turn, turn, step.freqs, offset=t)
        q, k, v = step.split(step.qkv)
        kc[:, t], vc[:, t] = k[:, 0], v[:, 0]
        lengths = torch.full((B,), t + 1, dtype=torch.int32, device="cuda")
        L.attention_window_decode(step.att.view(B, H, HD), q[:, 0], kc, vc, lengths=lengths, window=WINDOW, sinks=SINKS, workspace=ws)
        L.gemm(two(step.y), two(step.att), step.wo, trans_b=True)
        L.norm_residual_fwd(step.out, step.h, step.x, step.y, w_post=step.w_post, gate=step.gate, w_pre=step.w_pre, scale=SCALE, eps=EPS)
        for n in ("out", "h"):
            got, want = getattr(step, n)[:, 0].double(), getattr(blk, n)[:, t].double()
            assert (got - want).norm() <= 14 * 2.0 ** -8 * want.norm(), (t, n)
