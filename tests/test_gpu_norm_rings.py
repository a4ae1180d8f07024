"""The norms' kernels of prompts and training batches: more rows than the GPU holds at once, so that a group of threads works
through several rows, its ring of rows ahead comes round, and several groups share a CTA and several CTAs an SM. Every group has
four rows or more on 148 SMs, in numbers that the groups do not divide.

Against the formulas in 64 bits. Tolerances as for the few rows, but for the sums over rows: a value passes at most the rows of its
group (16 here), the groups of its CTA (8), a warp's share of the CTAs' sums (19) and the warps (32): 80 additions of U = 2^-24 each
beside the 64 of its terms - less than the share of one row of 16,384, so that a lost row shows."""
import pytest
import torch

import pelica_b200 as pb
from tests.test_gpu_block_norm import Case, at, gradients, normed, rounding
from tests.test_gpu_rows import DT, U, untouched

pytestmark = pytest.mark.gpu
SUM = 64 + 80


@pytest.fixture(scope="module")
def tctx():
    c = pb.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


class OnGpu(Case):
    """The same, the 64-bit side and the streams' values made on the GPU."""

    def stream(self, fill=True):
        buf = torch.full((self.T * (self.d + self.pitch) + self.shift,), 55.0, dtype=DT[self.dtype], device="cuda")
        v = buf[self.shift:].view(self.T, self.d + self.pitch)[:, :self.d]
        if fill:
            v.copy_(torch.randn(self.T, self.d, generator=torch.Generator("cuda").manual_seed(int(torch.randint(1 << 30, (1,), generator=self.g))),
                                device="cuda"))
        return v, buf

    def weight(self, w):
        return 1.0 if w is None else w.double() + self.offset

    def gate64(self):
        if self.gates is None:
            return torch.ones((), dtype=torch.float64, device="cuda")
        return self.gates.double() if self.gate == "channel" else self.gates.double()[:, None]


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (what, float((off - bound).max()), int((~(off <= bound)).sum()))


def forward(c):
    (r, r_buf), (n, n_buf) = c.stream(False), c.stream(False)
    c.op.forward(c.T, at(c.x), at(c.f), at(r), at(n) if c.pre else None, w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
    c.op.ctx.sync()
    want_r, want_n, size = c.formula(c.x.double(), c.f.double())
    within(r, want_r, 40 * U * size + rounding(c.dtype, want_r), "r")
    untouched(r, r_buf, c.d)
    if c.pre:
        within(n, want_n, normed(c, want_r, size) + rounding(c.dtype, want_n), "n")
        untouched(n, n_buf, c.d)


def backward(c, with_dr=True):
    r, dr = c.x, c.stream()[0]
    dn = c.stream()[0] if c.pre else None
    (dx, dx_buf), (df, df_buf) = c.stream(False), c.stream(False)
    got = dict(dx=dx, df=df)
    for k, n in dict(dw_pre=c.d if c.pre else 0, dw_post=c.d if c.post else 0, dgate=0 if c.gates is None else c.gates.numel()).items():
        if n:
            got[k] = torch.full((n,), 55.0, device="cuda")
    scratch = torch.empty(c.op.scratch_bytes(c.T), dtype=torch.uint8, device="cuda")
    c.op.grad(c.T, at(r), at(c.f), at(dr) if with_dr else None, at(dn), at(dx), at(df), w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre),
              dw_post=at(got.get("dw_post")), dgate=at(got.get("dgate")), dw_pre=at(got.get("dw_pre")), scratch=at(scratch),
              scratch_bytes=scratch.numel())
    c.op.ctx.sync()
    want = gradients(c, r.double(), c.f.double(), dr.double() * float(with_dr), None if dn is None else dn.double())
    for k, v in got.items():
        value, size = want[k]
        terms = 64 if k in ("dx", "df") or (k == "dgate" and c.gate == "token") else SUM
        within(v, value, terms * U * size + rounding(c.dtype if k in ("dx", "df") else "f32", value), k)
    untouched(dx, dx_buf, c.d)
    untouched(df, df_buf, c.d)


# (rows, width): 8, 4, 2 groups a CTA and one, in 16 bits and in f32; CTAs of 896 and 1,024 threads; clusters; rows value by value
SHAPES = [(16383, 320), (8191, 520), (4001, 2048), (1301, 7168), (701, 8200), (333, 24576), (2503, 2045)]


@pytest.mark.parametrize("dtype, wtype", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("form", [dict(gate="channel"), dict(gate="token", offset=1.0), dict(post=False, gate="none"), dict(pre=False, gate="none"),
                                  dict(post=False, gate="token")],
                         ids=["both_channel", "both_token", "pre", "post", "pre_token"])
@pytest.mark.parametrize("T, d", SHAPES)
def test_many_rows(tctx, T, d, form, dtype, wtype):
    c = OnGpu(tctx, T=T, d=d, dtype=dtype, wtype=wtype, **form)
    forward(c)
    backward(c)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T, d", [(8191, 520), (1301, 7168), (333, 24576)])
def test_many_rows_without_a_stream(tctx, T, d, dtype):
    """No gradient from later blocks; rows in wider rows; the first norm of a model, where there is no block yet; n alone."""
    c = OnGpu(tctx, T=T, d=d, dtype=dtype, pitch=8)
    backward(c, with_dr=False)
    c = OnGpu(tctx, T=T, d=d, dtype=dtype, post=False, gate="none", alpha=1.0, pitch=8)
    n, buf = c.stream(False)
    c.op.forward(T, at(c.x), None, None, at(n), w_pre=at(c.w_pre))
    tctx.sync()
    x = c.x.double()
    want = x * c.inv(x) * c.weight(c.w_pre)
    within(n, want, 64 * U * want.abs() + rounding(dtype, want), "n")
    untouched(n, buf, d)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T, d", [(16383, 320), (1301, 7168), (333, 24576)])
def test_many_rows_in_place_and_again(tctx, T, d, dtype):
    """The rows ahead are read before the rows in front of them are written: in place the same bits, and the same every time."""
    c = OnGpu(tctx, T=T, d=d, dtype=dtype)
    kw = dict(w_post=at(c.w_post), gate=at(c.gates), w_pre=at(c.w_pre))
    r, n, dr, dn, dx, df = (c.stream()[0] for _ in range(6))
    dw = [[torch.empty(d, device="cuda") for _ in range(3)] for _ in range(2)]
    scratch = torch.empty(c.op.scratch_bytes(T), dtype=torch.uint8, device="cuda")
    c.op.forward(T, at(c.x), at(c.f), at(r), at(n), **kw)
    x, f = c.x.clone(), c.f.clone()
    c.op.forward(T, at(x), at(f), at(x), at(f), **kw)
    tctx.sync()
    assert torch.equal(x, r) and torch.equal(f, n)
    a, b = dr.clone(), dn.clone()
    for out, (p, q, u, v) in zip(dw, ((dr, dn, dx, df), (a, b, a, b))):
        c.op.grad(T, at(r), at(c.f), at(p), at(q), at(u), at(v), dw_post=at(out[0]), dgate=at(out[1]), dw_pre=at(out[2]), scratch=at(scratch),
                  scratch_bytes=scratch.numel(), **kw)
    tctx.sync()
    assert torch.equal(a, dx) and torch.equal(b, df)
    assert all(torch.equal(p, q) for p, q in zip(*dw))
