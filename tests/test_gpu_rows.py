"""Tokens sorted by expert and back, and the gradients, against plain 64-bit arithmetic on the CPU.

Tolerances: with u = 2^-24, a sum in which a term passes through n additions is off by at most (n + 1) u times the sum of
the terms' sizes (products are exact or one rounding more); a result is then rounded by half a step of its type. A sum over
top_k has n <= top_k + 1, a dot product over d values at most d / 32 + 16 (a lane's own terms, 16 bytes at a time, then
lanes and warps)."""
import math

import numpy as np
import pytest
import torch

import pelica_b200 as pb

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def tctx():
    """A context ordered on torch's stream."""
    c = pb.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def half_step(dtype):
    return torch.finfo(DT[dtype]).eps / 2


class Case:
    """Inputs and buffers of one set of calls; streams with `pitch` more values a row, filled with what must not change."""

    def __init__(self, ctx, T, d, K, E, dtype="f32", first=0, local=0, align=1, none=0.0, pitch=0, shift=0, seed=0, skew=True, ids=None):
        g = torch.Generator().manual_seed(seed)
        self.T, self.d, self.K, self.E, self.dtype, self.first, self.align = T, d, K, E, dtype, first, align
        self.local = local or E
        self.op = pb.Rows(ctx, d, K, E, dtype=dtype, first_expert=first, n_local=local, align=align, x_stride=d + pitch, rows_stride=d + pitch)
        self.pitch, self.shift, self.g = pitch, shift, g
        if ids is None:
            p = torch.arange(1, E + 1).double() ** (-1.2 if skew else 0.0)
            ids = torch.multinomial(p.expand(max(T, 1), E), K, generator=g)[:T] if K <= E else torch.randint(0, E, (T, K), generator=g)
            ids = ids.long()
            ids[torch.rand(T, K, generator=g) < none] = -1
        self.ids = ids
        self.w = torch.rand(T, K, generator=g) - 0.2
        self.max_rows = self.op.bound(T)
        self.offset = torch.full((self.local + 1,), 77, dtype=torch.int32, device="cuda")
        self.count = torch.full((self.local,), 77, dtype=torch.int32, device="cuda")
        self.pos = torch.full((T, K), 77, dtype=torch.int32, device="cuda")
        one = lambda t: torch.full((self.max_rows,), 77, dtype=t, device="cuda")  # noqa: E731
        self.row_pair, self.row_expert, self.row_weight = one(torch.int32), one(torch.int32), one(torch.float32)
        self.plan = self.op.plan(self.max_rows, *(t.data_ptr() for t in (self.offset, self.count, self.pos, self.row_pair, self.row_expert,
                                                                        self.row_weight)))
        self.ids_d, self.w_d = ids.int().cuda(), self.w.cuda()
        self.want_plan()

    def stream(self, rows, fill=None):
        """[rows][d] in a buffer of wider rows that starts `shift` values behind an aligned address: (the view, all of it)."""
        buf = torch.full((rows * (self.d + self.pitch) + self.shift,), 55.0, dtype=DT[self.dtype], device="cuda")
        v = buf[self.shift:].view(rows, self.d + self.pitch)[:, :self.d]
        if fill is None:
            v.copy_(torch.randn(rows, self.d, generator=self.g))
        return v, buf

    def want_plan(self):
        groups = [[] for _ in range(self.local)]
        for p, e in enumerate(self.ids.reshape(-1).tolist()):
            if self.first <= e < self.first + self.local and e < self.E and e >= 0:
                groups[e - self.first].append(p)
        self.want = dict(offset=[0], count=[len(q) for q in groups], pos=[-1] * (self.T * self.K), row_pair=[77] * self.max_rows,
                         row_expert=[77] * self.max_rows, row_weight=[77.0] * self.max_rows)
        w, at = self.w.reshape(-1).tolist(), 0
        for i, q in enumerate(groups):
            n = math.ceil(len(q) / self.align) * self.align
            for j in range(n):
                self.want["row_pair"][at + j] = q[j] if j < len(q) else -1
                self.want["row_expert"][at + j] = i + self.first
                self.want["row_weight"][at + j] = w[q[j]] if j < len(q) else 0.0
                if j < len(q):
                    self.want["pos"][q[j]] = at + j
            at += n
            self.want["offset"].append(at)
        self.total = at

    def check_plan(self):
        for k, v in self.want.items():
            got = getattr(self, k).reshape(-1).cpu().numpy()
            assert np.array_equal(got, np.array(v, got.dtype)), k

    def use_plan(self):
        """Plan buffers as the definition has them, for calls that are tested alone."""
        for k in ("offset", "count", "pos"):
            t = getattr(self, k)
            t.copy_(torch.tensor(self.want[k], dtype=torch.int32).reshape(t.shape))

    def has(self):
        return torch.tensor(self.want["pos"]).reshape(self.T, self.K) >= 0

    def gathered(self, rows):
        """[T][K][d] f64: the pairs' rows, zeros where a pair has none."""
        p = torch.tensor(self.want["pos"], dtype=torch.long).reshape(self.T, self.K)
        return rows.cpu().double()[p.clamp(min=0)] * (p >= 0)[..., None]


def inside(got, want, bound, what):
    got, want = got.cpu().double(), want.double()
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {float(over.max()):.3g} over the bound, at {np.unravel_index(int(over.argmax()), over.shape)}"


def untouched(view, buf, d):
    """The columns behind the rows, and what lies in front of the first, hold what they held."""
    keep = torch.ones_like(buf, dtype=torch.bool)
    keep[buf.numel() - view.shape[0] * view.stride(0):].view(view.shape[0], view.stride(0))[:, :d] = False
    assert bool((buf[keep] == 55.0).all())


def run_dispatch(c, scale):
    x, _ = c.stream(c.T)
    rows, buf = c.stream(c.max_rows, fill=False)
    c.op.dispatch(c.T, c.ids_d.data_ptr(), c.plan, x.data_ptr(), rows.data_ptr(), w=c.w_d.data_ptr(), scale=scale)
    c.op.ctx.sync()
    c.check_plan()
    untouched(rows, buf, c.d)
    pair = torch.tensor(c.want["row_pair"][:c.total], dtype=torch.long)
    want = x.cpu()[pair.clamp(min=0) // c.K]
    if scale:  # one rounding of an exact product to f32, one to the type
        want = (want.float() * c.w.reshape(-1)[pair.clamp(min=0)][:, None]).to(DT[c.dtype])
    want[pair < 0] = 0
    got = rows.cpu()
    assert torch.equal(got[:c.total], want)
    assert bool((got[c.total:] == 55.0).all())


def run_collect(c, add, weighted=True, in_place=False):
    c.use_plan()
    rows, _ = c.stream(c.max_rows)
    a = c.stream(c.T)[0] if add else None
    y, buf = c.stream(c.T, fill=False)
    terms = c.gathered(rows) * (c.w.double()[..., None] if weighted else 1.0)
    base = a.cpu().double() if add else torch.zeros(c.T, c.d, dtype=torch.float64)
    if in_place:
        y.copy_(a)
        a = y
    c.op.collect(c.T, c.plan, rows.data_ptr(), y.data_ptr(), w=c.w_d.data_ptr() if weighted else None, add=a.data_ptr() if add else None)
    c.op.ctx.sync()
    want = base + terms.sum(1)
    inside(y, want, (c.K + 2) * U * (base.abs() + terms.abs().sum(1)) + half_step(c.dtype) * want.abs() * (1 + 2.0 ** -8) + tiny(c.dtype), "y")
    untouched(y, buf, c.d)


def tiny(dtype):
    """Half of the smallest step of the type (values below its normal range)."""
    f = torch.finfo(DT[dtype])
    return f.tiny * f.eps / 2


def dots(c, rows, x):
    p = c.gathered(rows)
    q = x.cpu().double()[:, None]
    return (p * q).sum(-1), (c.d / 32 + 17) * U * (p * q).abs().sum(-1)


def run_dispatch_grad(c, weighted, dw):
    c.use_plan()
    rows, _ = c.stream(c.max_rows)
    x, _ = c.stream(c.T)
    dx, buf = c.stream(c.T, fill=False)
    d_w = torch.full((c.T, c.K), 55.0, device="cuda")
    c.op.dispatch_grad(c.T, c.plan, rows.data_ptr(), dx.data_ptr(), w=c.w_d.data_ptr() if weighted else None,
                       x=x.data_ptr() if dw else None, dw=d_w.data_ptr() if dw else None)
    c.op.ctx.sync()
    terms = c.gathered(rows) * (c.w.double()[..., None] if weighted else 1.0)
    want = terms.sum(1)
    inside(dx, want, (c.K + 1) * U * terms.abs().sum(1) + half_step(c.dtype) * want.abs() * (1 + 2.0 ** -8) + tiny(c.dtype), "dx")
    untouched(dx, buf, c.d)
    if dw:
        inside(d_w, *dots(c, rows, x), "dw")
        assert bool((d_w.cpu()[~c.has()] == 0).all())


def run_collect_grad(c, weighted, dw):
    c.use_plan()
    rows, _ = c.stream(c.max_rows)
    dy, _ = c.stream(c.T)
    drows, buf = c.stream(c.max_rows, fill=False)
    d_w = torch.full((c.T, c.K), 55.0, device="cuda")
    c.op.collect_grad(c.T, c.plan, dy.data_ptr(), drows.data_ptr(), w=c.w_d.data_ptr() if weighted else None,
                      rows=rows.data_ptr() if dw else None, dw=d_w.data_ptr() if dw else None)
    c.op.ctx.sync()
    pair = torch.tensor(c.want["row_pair"][:c.total], dtype=torch.long)
    want = dy.cpu()[pair.clamp(min=0) // c.K].float()
    if weighted:
        want = want * c.w.reshape(-1)[pair.clamp(min=0)][:, None]
    want[pair < 0] = 0
    assert torch.equal(drows.cpu()[:c.total], want.to(DT[c.dtype]))
    assert bool((drows.cpu()[c.total:] == 55.0).all())
    untouched(drows, buf, c.d)
    if dw:
        inside(d_w, *dots(c, rows, dy), "dw")
        assert bool((d_w.cpu()[~c.has()] == 0).all())


# tokens, d, top_k, experts, and what else is unusual
SHAPES = [
    dict(T=1, d=64, K=8, E=64),                                    # a decode step
    dict(T=1, d=1, K=1, E=1),                                      # one value
    dict(T=7, d=33, K=3, E=5, none=0.3),                           # nothing that a vector divides
    dict(T=16, d=2048, K=8, E=128, align=16),                      # every group padded
    dict(T=128, d=72, K=8, E=256, align=256, none=0.1),            # padding far beyond the rows; 1,024 pairs: the last small sort
    dict(T=129, d=72, K=8, E=512, align=3),                        # 1,032: the first large one
    dict(T=300, d=136, K=5, E=40, pitch=8, align=128),             # rows in a wider buffer, still whole words
    dict(T=65, d=136, K=16, E=16, pitch=3),                        # ... that start anywhere
    dict(T=200, d=200, K=2, E=64, shift=1),                        # the buffer itself starts anywhere
    dict(T=500, d=24, K=4, E=32, first=8, local=8, none=0.2),      # a shard
    dict(T=400, d=40, K=4, E=33, first=32, local=1, align=16),     # a shard of one expert
    dict(T=3, d=520, K=2, E=6, align=256),                         # a few pairs, nearly all rows are padding
    dict(T=700, d=64, K=2, E=3, align=200),                        # ... of a few large groups
    dict(T=100, d=49152, K=1, E=2),                                # the widest rows
    dict(T=2500, d=16, K=6, E=512, none=0.05),                     # more experts than most have pairs
]
IDS = ["_".join(f"{k}{v}" for k, v in s.items()) for s in SHAPES]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_all_calls(tctx, shape, dtype):
    c = Case(tctx, dtype=dtype, seed=int(10 * sum(shape.values())), **shape)
    run_dispatch(c, scale=False)
    run_dispatch(c, scale=True)
    run_collect(c, add=True)
    run_collect(c, add=False, weighted=False)
    run_collect(c, add=True, in_place=True)
    run_dispatch_grad(c, weighted=True, dw=True)
    run_dispatch_grad(c, weighted=False, dw=False)
    run_collect_grad(c, weighted=True, dw=True)
    run_collect_grad(c, weighted=False, dw=False)
    run_collect_grad(c, weighted=False, dw=True)


@pytest.mark.parametrize("T, K, E, align", [(16384, 16, 512, 1), (16384, 8, 3, 16), (4097, 7, 200, 5), (16384, 1, 512, 256),
                                            (1024, 4, 64, 1), (4100, 1, 9, 4), (8192, 1, 77, 1), (8193, 1, 77, 2), (8193, 8, 300, 1)])
def test_large_sorts(tctx, T, K, E, align):
    c = Case(tctx, T=T, d=8, K=K, E=E, align=align, none=0.02, seed=T + K)
    run_dispatch(c, scale=False)


@pytest.mark.parametrize("T", [3, 400])
@pytest.mark.parametrize("kind", ["one expert", "nobody", "twice", "elsewhere"])
def test_unusual_routing(tctx, kind, T):
    """Every pair at one expert; no pair with a row; the same expert twice in a token; all experts on other GPUs."""
    K, E = 4, 16
    ids = dict(zip(["one expert", "nobody", "twice", "elsewhere"],
                   [torch.full((T, K), 9), torch.full((T, K), -1), torch.arange(T * K).reshape(T, K) // 2 % E, torch.full((T, K), 2)]))[kind]
    c = Case(tctx, T=T, d=48, K=K, E=E, first=8 if kind == "elsewhere" else 0, local=8 if kind == "elsewhere" else 0, align=8, ids=ids, dtype="bf16")
    run_dispatch(c, scale=False)
    run_collect(c, add=True)
    run_collect(c, add=False)
    run_dispatch_grad(c, weighted=True, dw=True)
    run_collect_grad(c, weighted=True, dw=True)


def test_no_tokens(tctx):
    c = Case(tctx, T=0, d=48, K=4, E=16, align=8)
    x = torch.zeros(8, 48, device="cuda")
    c.op.dispatch(0, None, c.plan, x.data_ptr(), x.data_ptr())
    c.op.collect(0, c.plan, None, None)
    c.op.collect_grad(0, c.plan, None, None)
    c.op.dispatch_grad(0, c.plan, None, None)
    tctx.sync()
    assert not c.offset.any() and not c.count.any()


@pytest.mark.parametrize("T", [5, 700])
def test_plan_alone(tctx, T):
    c = Case(tctx, T=T, d=4096, K=3, E=10, align=4)
    c.op.dispatch(T, c.ids_d.data_ptr(), c.plan, w=c.w_d.data_ptr())
    tctx.sync()
    c.check_plan()


def test_rows_without_values_stay_out_of_sums(tctx):
    """Infinities and NaN in rows that no pair names, and in tokens without pairs, reach nothing; where a weight is 0 they
    count, as in the formula."""
    c = Case(tctx, T=6, d=40, K=2, E=4, align=8, ids=torch.tensor([[0, 1], [-1, -1], [2, -1], [0, 0], [-1, 3], [1, 2]]))
    c.use_plan()
    rows, _ = c.stream(c.max_rows)
    used = torch.zeros(c.max_rows, dtype=torch.bool)
    used[[p for p in c.want["pos"] if p >= 0]] = True
    rows[~used.cuda()] = float("nan")
    y, _ = c.stream(c.T, fill=False)
    c.op.collect(c.T, c.plan, rows.data_ptr(), y.data_ptr(), w=c.w_d.data_ptr())
    tctx.sync()
    assert bool(torch.isfinite(y).all()) and not y[1].any()
    w = c.w.clone()
    w[0, 0] = 0.0
    rows[c.want["pos"][0]] = float("inf")
    c.op.collect(c.T, c.plan, rows.data_ptr(), y.data_ptr(), w=w.cuda().data_ptr())
    tctx.sync()
    assert bool(torch.isnan(y[0]).all()) and bool(torch.isfinite(y[2:]).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d, pitch", [(40, 0), (40, 3), (2048, 0)])
def test_padded_tokens_may_hold_anything(tctx, d, pitch, dtype):
    """Routing weights that are NaN and values that are infinite in tokens without pairs stay where they are: sums over no row
    are zeros (or add), the weights' gradients of pairs without a row are 0."""
    c = Case(tctx, T=5, d=d, K=3, E=4, dtype=dtype, pitch=pitch, ids=torch.tensor([[0, 1, 2], [-1, -1, -1], [3, -1, 0], [-1, -1, -1], [2, 1, 3]]))
    c.use_plan()
    c.w[~c.has()] = float("nan")
    c.w_d = c.w.cuda()
    x, _ = c.stream(5)
    x[1], x[3] = float("inf"), float("nan")
    rows, _ = c.stream(c.max_rows)
    y, _ = c.stream(5)
    add, _ = c.stream(5)
    dw = torch.full((5, 3), 55.0, device="cuda")
    kw = dict(w=c.w_d.data_ptr())
    c.op.collect(5, c.plan, rows.data_ptr(), y.data_ptr(), **kw)
    tctx.sync()
    assert bool(torch.isfinite(y).all()) and not y[1].any() and not y[3].any()
    c.op.collect(5, c.plan, rows.data_ptr(), y.data_ptr(), add=add.data_ptr(), **kw)
    tctx.sync()
    assert torch.equal(y[1], add[1]) and torch.equal(y[3], add[3])
    c.op.dispatch_grad(5, c.plan, rows.data_ptr(), y.data_ptr(), x=x.data_ptr(), dw=dw.data_ptr(), **kw)
    tctx.sync()
    assert bool(torch.isfinite(y).all()) and not y[1].any() and bool(torch.isfinite(dw).all()) and bool((dw.cpu()[~c.has()] == 0).all())
    dw.fill_(55.0)
    drows, _ = c.stream(c.max_rows, fill=False)
    c.op.collect_grad(5, c.plan, x.data_ptr(), drows.data_ptr(), rows=rows.data_ptr(), dw=dw.data_ptr(), **kw)
    tctx.sync()
    assert bool(torch.isfinite(dw).all()) and bool((dw.cpu()[~c.has()] == 0).all()) and bool(torch.isfinite(drows[:c.total]).all())


@pytest.mark.parametrize("T", [5, 600])
def test_ids_that_no_expert_has_are_left_out_and_reported(tctx, T):
    c = Case(tctx, T=T, d=32, K=3, E=7, align=4)
    bad = c.ids.clone()
    bad[T // 2, 1], bad[0, 0] = 7, 2 ** 31 - 1
    left = c.ids.clone()
    left[T // 2, 1] = left[0, 0] = -1
    c.ids = left
    c.want_plan()
    x, _ = c.stream(T)
    rows, _ = c.stream(c.max_rows, fill=False)
    ids = bad.int().cuda()
    c.op.dispatch(T, ids.data_ptr(), c.plan, x.data_ptr(), rows.data_ptr(), w=c.w_d.data_ptr(), scale=False)
    with pytest.raises(pb.PelicaError, match="expert id"):
        tctx.sync()
    c.check_plan()
    tctx.sync()


def test_positions_outside_the_rows_are_left_out_and_reported(tctx):
    c = Case(tctx, T=9, d=32, K=3, E=7)
    c.use_plan()
    c.pos[4, 1], c.pos[5, 2] = c.max_rows, 2 ** 31 - 1
    c.want["pos"][4 * 3 + 1] = c.want["pos"][5 * 3 + 2] = -1
    rows, _ = c.stream(c.max_rows)
    x, _ = c.stream(c.T)
    out, _ = c.stream(c.T)
    d_w = torch.full((c.T, c.K), 55.0, device="cuda")
    grad, _ = c.stream(c.max_rows, fill=False)
    for call in (lambda: c.op.collect(c.T, c.plan, rows.data_ptr(), out.data_ptr()),
                 lambda: c.op.dispatch_grad(c.T, c.plan, rows.data_ptr(), out.data_ptr(), w=c.w_d.data_ptr(), x=x.data_ptr(), dw=d_w.data_ptr()),
                 lambda: c.op.collect_grad(c.T, c.plan, x.data_ptr(), grad.data_ptr()),
                 lambda: c.op.collect_grad(c.T, c.plan, x.data_ptr(), grad.data_ptr(), rows=rows.data_ptr(), dw=d_w.data_ptr())):
        call()
        with pytest.raises(pb.PelicaError, match="row position"):
            tctx.sync()
        tctx.sync()
    inside(d_w, *dots(c, rows, x), "dw")


def test_refusals(tctx):
    c = Case(tctx, T=4, d=32, K=2, E=4, align=2)
    x, _ = c.stream(8)
    rows, _ = c.stream(c.max_rows)
    host = np.zeros(4096, np.float32)
    pinned = torch.zeros(4096).pin_memory()
    ids, p = c.ids_d.data_ptr(), rows.data_ptr()
    small = c.op.plan(c.max_rows - 1, c.offset.data_ptr(), c.count.data_ptr(), c.pos.data_ptr())
    bare = c.op.plan(c.max_rows, None, None, c.pos.data_ptr())
    calls = [
        (lambda: c.op.dispatch(4, ids, small, x.data_ptr(), p), "max_rows"),
        (lambda: c.op.dispatch(4, ids, bare, x.data_ptr(), p), "offset"),
        (lambda: c.op.dispatch(4, None, c.plan, x.data_ptr(), p), "ids"),
        (lambda: c.op.dispatch(4, ids, c.plan, x.data_ptr(), None), "rows"),
        (lambda: c.op.dispatch(4, ids, c.plan, host.ctypes.data, p), "x must be a device pointer"),
        (lambda: c.op.dispatch(4, ids, c.plan, pinned.data_ptr(), p), "x must be a device pointer"),
        (lambda: c.op.dispatch(4, ids, c.plan, x.data_ptr() + 2, p), "aligned"),
        (lambda: c.op.collect(4, c.plan, p, None), "y"),
        (lambda: c.op.collect(4, c.plan, p, x.data_ptr(), w=host.ctypes.data), "w must be"),
        (lambda: c.op.dispatch_grad(4, c.plan, p, x.data_ptr(), w=c.w_d.data_ptr(), dw=c.w_d.data_ptr()), "x is null"),
        (lambda: c.op.dispatch_grad(4, c.plan, p, x.data_ptr(), x=x.data_ptr(), dw=c.w_d.data_ptr()), "w is null"),
        (lambda: c.op.collect_grad(4, c.plan, x.data_ptr(), p, dw=c.w_d.data_ptr()), "rows is null"),
        (lambda: c.op.collect_grad(4, bare, x.data_ptr(), p), "offset"),
    ]
    for call, word in calls:
        with pytest.raises(pb.PelicaError, match=word):
            call()
    lib, flags = c.op.lib, 2
    import ctypes as C
    assert lib.pm_dispatch_rows(tctx.h, C.byref(c.op.desc), 4, ids, None, C.byref(c.plan), x.data_ptr(), p, flags) == -1
    assert lib.pm_dispatch_rows(tctx.h, C.byref(c.op.desc), 4, ids, None, C.byref(c.plan), x.data_ptr(), p, 1) == -1  # scale without w
    tctx.sync()


def test_gradients_are_those_of_the_operators(tctx):
    """<dispatch(x), g> differentiated by x and by w, <collect(rows), h> by rows and by w: against differences of the calls
    themselves (both are linear in each, so a difference over a step of 1 is exact but for rounding)."""
    c = Case(tctx, T=13, d=40, K=3, E=6, none=0.2)
    c.use_plan()
    x, _ = c.stream(c.T)
    rows, _ = c.stream(c.max_rows)
    gen = torch.Generator().manual_seed(5)
    h = torch.randn(c.T, c.d, generator=gen).cuda()
    y0, y1 = c.stream(c.T)[0], c.stream(c.T)[0]
    drows, _ = c.stream(c.max_rows, fill=False)
    drows.zero_()
    dw = torch.zeros(c.T, c.K, device="cuda")
    hh, _ = c.stream(c.T)
    hh.copy_(h)
    c.op.collect_grad(c.T, c.plan, hh.data_ptr(), drows.data_ptr(), w=c.w_d.data_ptr(), rows=rows.data_ptr(), dw=dw.data_ptr())
    step = torch.randn(c.max_rows, c.d, generator=gen).cuda()
    moved, _ = c.stream(c.max_rows)
    moved.copy_(rows + step)
    w2 = c.w_d + 1.0
    def loss(r, w, y):
        c.op.collect(c.T, c.plan, r.data_ptr(), y.data_ptr(), w=w.data_ptr())
        return (y.double() * hh.double()).sum()
    a, b, e = loss(rows, c.w_d, y0), loss(moved, c.w_d, y1), loss(rows, w2, y1)
    tctx.sync()
    size = float((y0.double() * hh.double()).abs().sum()) * 4 + 1
    assert abs(float(b - a - (drows.double() * (moved - rows).double()).sum())) <= 64 * U * size * 4
    assert abs(float(e - a - dw.double().sum())) <= 64 * U * size * 4


def test_one_run_as_another(tctx):
    """The same bits twice, also from a recorded graph replayed between other calls, and on a context of another stream."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ctx2 = pb.Context(0, stream=side.cuda_stream)
        for T in (6, 300):
            c = Case(ctx2, T=T, d=72, K=4, E=12, align=4, dtype="bf16")
            x, _ = c.stream(T)
            rows, _ = c.stream(c.max_rows, fill=False)
            y, _ = c.stream(T)
            drows, _ = c.stream(c.max_rows, fill=False)
            dw = torch.zeros(T, 4, device="cuda")

            def step():
                c.op.dispatch(T, c.ids_d.data_ptr(), c.plan, x.data_ptr(), rows.data_ptr(), w=c.w_d.data_ptr(), scale=False)
                c.op.collect(T, c.plan, rows.data_ptr(), y.data_ptr(), w=c.w_d.data_ptr(), add=x.data_ptr())
                c.op.collect_grad(T, c.plan, x.data_ptr(), drows.data_ptr(), w=c.w_d.data_ptr(), rows=rows.data_ptr(), dw=dw.data_ptr())

            step()
            side.synchronize()
            first = [t.clone() for t in (c.pos, rows, y, drows, dw)]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            for t in (c.pos, y, dw):
                t.zero_()
            graph.replay()
            big = Case(ctx2, T=900, d=72, K=4, E=12, align=4, dtype="bf16")  # another size between the replays
            run_dispatch(big, scale=False)
            graph.replay()
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(first, (c.pos, rows, y, drows, dw)))
            c.check_plan()
        ctx2.sync()
        ctx2.close()


def test_rows_beyond_32_bit_offsets(tctx):
    """Positions whose values lie more than 2^32 elements behind the start."""
    T, K, E, d = 16384, 2, 512, 49152
    ids = torch.stack([torch.arange(T) % 2, 510 + torch.arange(T) % 2], 1)
    op = pb.Rows(tctx, d, K, E, dtype="bf16", align=256, rows_stride=3 * d)
    c = Case(tctx, T=T, d=8, K=K, E=E, align=256, ids=ids, dtype="bf16")
    x = torch.randn(T, 1, dtype=torch.bfloat16, device="cuda").expand(T, d).contiguous()
    n = 2 * T
    rows = torch.empty(n, 3 * d, dtype=torch.bfloat16, device="cuda")
    op.dispatch(T, c.ids_d.data_ptr(), c.plan, x.data_ptr(), rows.data_ptr())
    tctx.sync()
    pair = torch.tensor(c.want["row_pair"][:n])
    assert torch.equal(rows[:, d - 1].cpu(), x[:, 0].cpu()[pair // K]) and torch.equal(rows[:, 0].cpu(), x[:, 0].cpu()[pair // K])
    y = torch.empty_like(x)
    op.collect(T, c.plan, rows.data_ptr(), y.data_ptr())
    tctx.sync()
    assert torch.equal(y, x + x)
