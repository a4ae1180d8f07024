"""The norms before and after a block with gate and residual scale, and their gradient, against plain 64-bit arithmetic.

Tolerances, with u = 2^-24: a sum of positive terms over a row passes each through at most 8 + 5 + 5 + 8 additions (a thread's
values, lanes, warps, a cluster's CTAs), so 1 / sqrt(mean + eps) is off by 26 / 2 + 4 roundings at most, and what is computed
from it in a few more steps by C = 40 u of the sum of the sizes of its terms (64 u where two norms lie one behind the other).
Sums over rows pass T more additions. A result is then rounded by half a step of its type."""
import ctypes as C

import numpy as np
import pytest
import torch

import pelica_b200 as pb
from tests.test_gpu_rows import DT, U, half_step, inside, tiny, untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx():
    c = pb.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


class Case:
    def __init__(self, ctx, T, d, dtype="f32", wtype="f32", post=True, pre=True, gate="channel", alpha=0.75, beta=1.5, offset=0.0, pitch=0,
                 shift=0, weights=True, eps=1e-6, seed=1):
        self.g = torch.Generator().manual_seed(seed + T + 7 * d)
        self.T, self.d, self.dtype, self.pitch, self.shift = T, d, dtype, pitch, shift
        self.post, self.pre, self.gate, self.alpha, self.beta, self.offset, self.eps = post, pre, gate, alpha, beta, offset, eps
        self.op = pb.BlockNorm(ctx, d, dtype=dtype, wtype=wtype, post=post, pre=pre, gate=gate, alpha=alpha, beta=beta, eps_post=eps,
                               eps_pre=eps, offset_post=offset, offset_pre=offset, stride=d + pitch)

        def vector(n):
            return (torch.randn(n, generator=self.g) * 0.5 + 1.0 - offset).to(DT[wtype]).cuda()

        self.w_post = vector(d) if post and weights else None
        self.w_pre = vector(d) if pre and weights else None
        self.gates = None if gate == "none" else vector(d if gate == "channel" else T)
        self.x, self.f = self.stream()[0], self.stream()[0]

    def stream(self, fill=True):
        buf = torch.full((self.T * (self.d + self.pitch) + self.shift,), 55.0, dtype=DT[self.dtype], device="cuda")
        v = buf[self.shift:].view(self.T, self.d + self.pitch)[:, :self.d]
        if fill:
            v.copy_(torch.randn(self.T, self.d, generator=self.g))
        return v, buf

    def weight(self, w):
        return 1.0 if w is None else w.cpu().double() + self.offset

    def gate64(self):
        if self.gates is None:
            return torch.ones((), dtype=torch.float64)
        g = self.gates.cpu().double()
        return g if self.gate == "channel" else g[:, None]

    def inv(self, v):
        return 1.0 / (v.pow(2).mean(1, keepdim=True) + self.eps).sqrt()

    def formula(self, x, f):
        """(r, n, the sizes of r's terms)"""
        p = f * self.inv(f) * self.weight(self.w_post) if self.post else f
        a, b = self.alpha * x, self.beta * self.gate64() * p
        r = a + b
        return r, r * self.inv(r) * self.weight(self.w_pre) if self.pre else None, a.abs() + b.abs()


def at(t):
    return None if t is None else t.data_ptr()


def rounding(dtype, want):
    return half_step(dtype) * want.abs() * (1 + 2.0 ** -8) + tiny(dtype)


def normed(c, r, size):
    """What n is off by before its rounding: what r is off by (its terms may cancel: by their sizes, not by its own), in its own
    element and, at most the row's largest, through the norm."""
    s = c.inv(r)
    return 64 * U * (size + size.pow(2).mean(1, keepdim=True).sqrt() * (r.abs() * s)) * s * abs(c.weight(c.w_pre))


def run_forward(c):
    r, r_buf = c.stream(False)
    n, n_buf = c.stream(False)
    c.op.forward(c.T, at(c.x), at(c.f), at(r), at(n) if c.pre else None, w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
    c.op.ctx.sync()
    want_r, want_n, size = c.formula(c.x.cpu().double(), c.f.cpu().double())
    inside(r, want_r, 40 * U * size + rounding(c.dtype, want_r), "r")
    untouched(r, r_buf, c.d)
    if c.pre:
        inside(n, want_n, normed(c, want_r, size) + rounding(c.dtype, want_n), "n")
        untouched(n, n_buf, c.d)
    else:
        assert bool((n_buf == 55.0).all())


def gradients(c, r, f, dr, dn):
    """The formula's gradients in 64 bits: {name: (value, sizes of the terms)}."""
    out, T = {}, c.T
    D, D_abs = dr, dr.abs()
    if c.pre:
        s, u = c.inv(r), dn * c.weight(c.w_pre)
        D = D + s * (u - r * s * s * (u * r).mean(1, keepdim=True))
        D_abs = D_abs + s * (u.abs() + r.abs() * s * s * (u * r).abs().mean(1, keepdim=True))
        out["dw_pre"] = ((dn * r * s).sum(0), (dn * r * s).abs().sum(0))
    out["dx"] = (c.alpha * D, abs(c.alpha) * D_abs)
    s = c.inv(f) if c.post else 1.0
    w = c.weight(c.w_post)
    q, q_abs = c.beta * D, abs(c.beta) * D_abs
    if c.gates is not None:
        over = 0 if c.gate == "channel" else 1
        out["dgate"] = ((q * f * s * w).sum(over), (q_abs * (f * s * w).abs()).sum(over))
        q, q_abs = q * c.gate64(), q_abs * c.gate64().abs()
    if c.post:
        out["dw_post"] = ((q * f * s).sum(0), (q_abs * (f * s).abs()).sum(0))
        v, v_abs = q * w, q_abs * abs(w)
        q = s * (v - f * s * s * (v * f).mean(1, keepdim=True))
        q_abs = s * (v_abs + f.abs() * s * s * (v_abs * f.abs()).mean(1, keepdim=True))
    out["df"] = (q, q_abs)
    return out


def run_grad(c, want_all=True):
    r, dr = c.x, c.stream()[0]
    dn = c.stream()[0] if c.pre else None
    dx, dx_buf = c.stream(False)
    df, df_buf = c.stream(False)
    new = lambda n: torch.full((n,), 55.0, device="cuda")  # noqa: E731
    got = dict(dx=dx, df=df)
    if want_all:
        if c.pre:
            got["dw_pre"] = new(c.d)
        if c.post:
            got["dw_post"] = new(c.d)
        if c.gates is not None:
            got["dgate"] = new(c.gates.numel())
    scratch = torch.empty(c.op.scratch_bytes(c.T), dtype=torch.uint8, device="cuda")
    c.op.grad(c.T, at(r), at(c.f), at(dr), at(dn), at(dx), at(df), w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre),
              dw_post=at(got.get("dw_post")), dgate=at(got.get("dgate")), dw_pre=at(got.get("dw_pre")), scratch=at(scratch),
              scratch_bytes=scratch.numel())
    c.op.ctx.sync()
    want = gradients(c, *(None if t is None else t.cpu().double() for t in (r, c.f, dr, dn)))
    for k, v in got.items():
        value, size = want[k]
        if k in ("dx", "df"):
            inside(v, value, 64 * U * size + rounding(c.dtype, value), k)
        else:
            inside(v, value, (64 + c.T) * U * size + rounding("f32", value), k)
    untouched(dx, dx_buf, c.d)
    untouched(df, df_buf, c.d)


SHAPES = [
    dict(T=1, d=64), dict(T=1, d=1, gate="token"), dict(T=3, d=7, pitch=3, gate="none"), dict(T=5, d=33, shift=1), dict(T=17, d=256),
    dict(T=40, d=264, gate="token"), dict(T=9, d=1000, pitch=8), dict(T=700, d=320, gate="token", alpha=1.0, beta=0.22), dict(T=330, d=2048),
    dict(T=6, d=2880, offset=1.0), dict(T=200, d=4100, gate="token"), dict(T=3, d=8192), dict(T=5, d=8200, gate="none"), dict(T=160, d=16384),
    dict(T=2, d=49152, gate="token"), dict(T=3, d=40001), dict(T=4, d=24, weights=False),
]


@pytest.mark.parametrize("dtype, wtype", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("shape", SHAPES, ids=["_".join(f"{k}{v}" for k, v in s.items()) for s in SHAPES])
def test_both_norms(tctx, shape, dtype, wtype):
    c = Case(tctx, dtype=dtype, wtype=wtype, **shape)
    run_forward(c)
    run_grad(c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("post, pre", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("T, d", [(1, 96), (65, 520), (4, 9000)])
def test_one_norm_or_none(tctx, T, d, post, pre, gate, dtype):
    c = Case(tctx, T=T, d=d, dtype=dtype, post=post, pre=pre, gate=gate)
    run_forward(c)
    run_grad(c)
    run_grad(c, want_all=False)


def test_the_stream_alone_and_the_block_alone(tctx):
    """f null: the first norm of a model; x null: a norm behind a block without a residual stream; r null: only n."""
    c = Case(tctx, T=11, d=200, post=False, gate="none", alpha=1.0)
    r, n = c.stream()[0], c.stream()[0]
    x = c.x.cpu().double()
    c.op.forward(11, at(c.x), None, None, at(n), w_pre=at(c.w_pre))
    tctx.sync()
    want = x * c.inv(x) * c.weight(c.w_pre)
    inside(n, want, 64 * U * want.abs(), "n")
    c = Case(tctx, T=11, d=200, pre=False, gate="none", beta=1.0)
    c.op.forward(11, None, at(c.f), at(r), w_post=at(c.w_post))
    tctx.sync()
    f = c.f.cpu().double()
    want = f * c.inv(f) * c.weight(c.w_post)
    inside(r, want, 64 * U * want.abs(), "r")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T, d", [(33, 200), (5, 9000)])
def test_in_place(tctx, T, d, dtype):
    """r over x, n over f; dx over dr, df over f and over dn: the same bits as in buffers of their own."""
    c = Case(tctx, T=T, d=d, dtype=dtype)
    r, n = c.stream()[0], c.stream()[0]
    kw = dict(w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
    c.op.forward(T, at(c.x), at(c.f), at(r), at(n), **kw)
    x, f = c.x.clone(), c.f.clone()
    c.op.forward(T, at(x), at(f), at(x), at(f), **kw)
    tctx.sync()
    assert torch.equal(x, r) and torch.equal(f, n)
    dr, dn, dx, df = (c.stream()[0] for _ in range(4))
    c.op.grad(T, at(r), at(c.f), at(dr), at(dn), at(dx), at(df), **kw)
    a, b = dr.clone(), dn.clone()
    c.op.grad(T, at(r), at(c.f), at(a), at(b), at(a), at(b), **kw)
    tctx.sync()
    assert torch.equal(a, dx) and torch.equal(b, df)
    f = c.f.clone()
    c.op.grad(T, at(r), at(f), at(dr), at(dn), at(dx), at(f), **kw)
    tctx.sync()
    assert torch.equal(f, df)


def test_no_rows(tctx):
    c = Case(tctx, T=0, d=40)
    c.op.forward(0, None, None, None)
    out = [torch.full((40,), 55.0, device="cuda") for _ in range(3)]
    c.op.grad(0, None, None, None, None, None, None, dw_post=at(out[0]), dgate=at(out[1]), dw_pre=at(out[2]), scratch=None, scratch_bytes=0)
    tctx.sync()
    assert not any(t.any() for t in out)


def test_rows_of_zeros_and_of_large_values(tctx):
    """A zero row stays zero (eps), values of 2^60 whose squares still fit are normed, an infinity makes its own row only NaN."""
    c = Case(tctx, T=4, d=136, gate="none", alpha=1.0, beta=1.0)
    c.x[0], c.f[0] = 0.0, 0.0
    c.x[1], c.f[1] = 2.0 ** 60, -(2.0 ** 60)
    c.f[2, 5] = float("inf")
    r, n = c.stream()[0], c.stream()[0]
    c.op.forward(4, at(c.x), at(c.f), at(r), at(n), w_post=at(c.w_post), w_pre=at(c.w_pre))
    tctx.sync()
    assert not r[0].any() and not n[0].any()
    want_r, want_n, size = c.formula(c.x.cpu().double(), c.f.cpu().double())
    ok = torch.tensor([1, 3])
    inside(r[ok], want_r[ok], (40 * U * size + rounding("f32", want_r))[ok], "r")
    inside(n[ok], want_n[ok], (normed(c, want_r, size) + rounding("f32", want_n))[ok], "n")
    assert bool(torch.isnan(n[2]).all())


def test_gradient_against_differences(tctx):
    """Derivatives of <r, a> + <n, b> along a random direction, by central differences of the formula in 64 bits."""
    for gate in ("channel", "token"):
        c = Case(tctx, T=6, d=48, gate=gate)
        a, b = torch.randn(6, 48, generator=c.g).double(), torch.randn(6, 48, generator=c.g).double()
        x, f = c.x.cpu().double(), c.f.cpu().double()
        kept = dict(w_post=c.w_post, w_pre=c.w_pre, gates=c.gates)
        at0 = dict(x=x, f=f, **{k: v.cpu().double() for k, v in kept.items()})

        def loss(v):
            c.w_post, c.w_pre, c.gates = v["w_post"], v["w_pre"], v["gates"]
            r, n, _ = c.formula(v["x"], v["f"])
            return float((r * a).sum() + (n * b).sum())

        r = c.formula(x, f)[0].float().cuda()
        dx, df = torch.empty(6, 48, device="cuda"), torch.empty(6, 48, device="cuda")
        dwp, dwn, dg = (torch.empty_like(kept[k]) for k in ("w_post", "w_pre", "gates"))
        scratch = torch.empty(c.op.scratch_bytes(6), dtype=torch.uint8, device="cuda")
        ad, bd = a.float().cuda(), b.float().cuda()
        c.op.grad(6, at(r), at(c.f), at(ad), at(bd), at(dx), at(df), w_post=at(kept["w_post"]), gate=at(kept["gates"]), w_pre=at(kept["w_pre"]),
                  dw_post=at(dwp), dgate=at(dg), dw_pre=at(dwn), scratch=at(scratch), scratch_bytes=scratch.numel())
        tctx.sync()
        for name, g in dict(x=dx, f=df, w_post=dwp, w_pre=dwn, gates=dg).items():
            way = torch.randn(at0[name].shape, generator=c.g).double()
            h = 1e-5
            diff = (loss({**at0, name: at0[name] + h * way}) - loss({**at0, name: at0[name] - h * way})) / (2 * h)
            mine = float((g.cpu().double() * way).sum())
            # third derivatives times h^2 and 64-bit rounding over h are below 1e-6 of the terms' sizes; f32 sums add 1e-5 of them
            assert abs(mine - diff) <= 2e-5 * float((g.cpu().double() * way).abs().sum()) + 1e-5, (gate, name)


def test_refusals(tctx):
    c = Case(tctx, T=4, d=32)
    r, n = c.stream()[0], c.stream()[0]
    host = np.zeros(4096, np.float32)
    kw = dict(w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
    scratch = torch.empty(c.op.scratch_bytes(4), dtype=torch.uint8, device="cuda")
    dw = torch.empty(32, device="cuda")
    plain = Case(tctx, T=4, d=32, post=False, pre=False, gate="none")
    calls = [
        (lambda: c.op.forward(4, None, None, at(r), at(n), **kw), "neither"),
        (lambda: c.op.forward(4, at(c.x), None, at(r), at(n), **kw), "without f"),
        (lambda: c.op.forward(4, at(c.x), at(c.f), at(r), None, **kw), "n is null"),
        (lambda: c.op.forward(4, at(c.x), at(c.f), at(r), at(n), w_post=at(c.w_post), w_pre=at(c.w_pre)), "gate is null"),
        (lambda: c.op.forward(4, host.ctypes.data, at(c.f), at(r), at(n), **kw), "x must be"),
        (lambda: c.op.forward(4, at(c.x) + 2, at(c.f), at(r), at(n), **kw), "aligned"),
        (lambda: plain.op.forward(4, at(c.x), at(c.f), None), "r is null"),
        (lambda: c.op.grad(4, None, at(c.f), None, at(n), at(r), None, **kw), "r is null"),
        (lambda: c.op.grad(4, at(r), at(c.f), None, None, at(r), None, **kw), "dn is null"),
        (lambda: c.op.grad(4, at(r), at(c.f), None, at(n), at(r), None, dw_pre=at(dw), scratch=at(scratch), scratch_bytes=16, **kw), "scratch of 16"),
        (lambda: c.op.grad(4, at(r), at(c.f), None, at(n), at(r), None, dw_pre=at(dw), scratch=at(scratch) + 4, scratch_bytes=1 << 30, **kw), "aligned"),
        (lambda: plain.op.grad(4, None, at(c.f), at(r), None, at(n), None, dw_pre=at(dw)), "dw_pre without"),
        (lambda: plain.op.grad(4, None, at(c.f), at(r), None, at(n), None, dw_post=at(dw)), "dw_post without"),
        (lambda: plain.op.grad(4, None, at(c.f), at(r), None, at(n), None, dgate=at(dw)), "dgate without"),
        (lambda: plain.op.grad(4, None, None, at(r), None, at(n), at(r)), "df without f"),
    ]
    for call, word in calls:
        with pytest.raises(pb.PelicaError, match=word):
            call()
    with pytest.raises(pb.PelicaError):
        pb.BlockNorm(tctx, 0)
    tctx.sync()


def test_recorded_and_replayed(tctx):
    """Forward and gradient from a recorded graph, other sizes in between: the same bits."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx2 = pb.Context(0, stream=side.cuda_stream)
        c = Case(ctx2, T=200, d=264, dtype="bf16")
        r, n, dr, dn, dx, df = (c.stream()[0] for _ in range(6))
        dw = [torch.empty(c.d, device="cuda") for _ in range(3)]
        scratch = torch.empty(c.op.scratch_bytes(c.T), dtype=torch.uint8, device="cuda")

        def step():
            kw = dict(w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
            c.op.forward(c.T, at(c.x), at(c.f), at(r), at(n), **kw)
            c.op.grad(c.T, at(r), at(c.f), at(dr), at(dn), at(dx), at(df), dw_post=at(dw[0]), dgate=at(dw[1]), dw_pre=at(dw[2]), scratch=at(scratch),
                      scratch_bytes=scratch.numel(), **kw)

        step()
        side.synchronize()
        first = [t.clone() for t in (r, n, dx, df, *dw)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for t in (r, n, dx, df, *dw):
            t.zero_()
        graph.replay()
        run_grad(Case(ctx2, T=900, d=520))
        graph.replay()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, (r, n, dx, df, *dw)))
        ctx2.sync()
        ctx2.close()
