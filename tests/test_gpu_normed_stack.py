"""A model's own norms in the layer loop, and the operators run together as a host with products of its own uses them."""
import ctypes as C

import numpy as np
import pytest
import torch

import pelica_b200 as pb
from pelica_b200 import synth
from tests.helpers import SMALL, bits_equal, tol_ok

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx():
    c = pb.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


class Buf:
    """A torch tensor as a device buffer of the library's calls."""

    def __init__(self, t):
        self.t, self.ptr, self.nbytes = t, t.data_ptr(), t.numel() * t.element_size()


def layers_of(ctx, cfg, n):
    return [pb.MoeLayer(ctx, cfg).load(synth.make_weights(cfg, 30 + i)) for i in range(n)]


NORMS = [dict(pre=True, post=True, alpha=0.5, beta=1.25, offset_pre=1.0, offset_post=1.0, gated=True), dict(pre=True, eps_pre=1e-5, alpha=1.0),
         dict(pre=False, post=True, eps_post=1e-5)]


def norm_weights(d, seed):
    rng = np.random.default_rng(seed)
    return [rng.normal(0.2, 0.3, d).astype(np.float32) for _ in range(3)]


def by_hand(ctx, layers, d, x):
    """The loop from the layers and the block norm."""
    T = x.shape[0]
    x = torch.from_numpy(x).cuda()
    for i, layer in enumerate(layers):
        k = dict(NORMS[i])
        gated = k.pop("gated", False)
        w = [torch.from_numpy(a).cuda() for a in norm_weights(d, i)]
        xn, f = x.clone(), torch.zeros_like(x)
        if k.get("pre"):
            pb.BlockNorm(ctx, d, pre=True, eps_pre=k.get("eps_pre", 1e-6), offset_pre=k.get("offset_pre", 0.0)).forward(
                T, x.data_ptr(), None, None, xn.data_ptr(), w_pre=w[0].data_ptr())
        layer.forward_dev(Buf(xn), T, Buf(f))
        out = torch.empty_like(x)
        pb.BlockNorm(ctx, d, pre=False, post=k.get("post", False), gate="channel" if gated else "none", alpha=k.get("alpha", 1.0),
                     beta=k.get("beta", 1.0), eps_post=k.get("eps_post", 1e-6), offset_post=k.get("offset_post", 0.0)).forward(
            T, x.data_ptr(), f.data_ptr(), out.data_ptr(), w_post=w[1].data_ptr(), gate=w[2].data_ptr() if gated else None)
        x = out
    ctx.sync()
    return x.cpu().numpy()


@pytest.mark.parametrize("name", ["c2", "c3", "c4"])
def test_norms_of_a_stack(tctx, name):
    cfg = SMALL[name]
    layers = layers_of(tctx, cfg, 3)
    st = pb.Stack(tctx, layers)
    had = st.decode_kernel
    xs = {T: synth.make_activations(T, cfg.d, 50 + T) for T in (1, 5, 40)}
    plain = {T: st.forward(x).copy() for T, x in xs.items()}
    for i, k in enumerate(NORMS):
        k = dict(k)
        w = norm_weights(cfg.d, i)
        gate = w[2] if k.pop("gated", False) else None
        st.set_norm(i, w[0], w[1], gate, **k)
    assert not st.decode_kernel
    for T, x in xs.items():
        want = by_hand(tctx, layers, cfg.d, x)
        for _ in range(3):  # the loop, its recording, a replay
            assert bits_equal(st.forward(x), want), T
    st.clear_norm(1)
    st.set_norm(0)  # unit weights: the plain form by the other kernel
    st.clear_norm(2)
    for T, x in xs.items():
        if name == "c3":  # (int8 layers: a value may round the other way)
            assert tol_ok(st.forward(x), plain[T])
    st.clear_norm(0)
    assert st.decode_kernel == had
    for T, x in xs.items():
        assert bits_equal(st.forward(x), plain[T])
    st.close()
    for layer in layers:
        layer.close()


def test_refusals_of_stack_norms(tctx):
    cfg = SMALL["c3"]
    layers = layers_of(tctx, cfg, 1)
    st = pb.Stack(tctx, layers)
    good = dict(dtype=synth.F32, wtype=synth.F32, d=cfg.d, flags=3, gate=0, eps_pre=1e-6, eps_post=1e-6, alpha=1.0, beta=1.0)
    x = synth.make_activations(4, cfg.d, 9)
    before = st.forward(x).copy()

    def call(layer=0, **change):
        return st.lib.pm_stack_set_norm(st.h, layer, C.byref(pb.NormDesc(**{**good, **change})), None, None, None)

    for got in (call(1), call(-1), call(d=cfg.d + 32), call(gate=1), call(x_stride=cfg.d), call(eps_pre=-1.0), call(flags=8)):
        assert got == -1
    for got in (call(dtype=synth.BF16), call(gate=2)):
        assert got == -2
    assert st.lib.pm_stack_set_norm(None, 0, None, None, None, None) == -1
    st.clear_norm(0)
    assert bits_equal(st.forward(x), before)
    st.close()
    layers[0].close()


@pytest.mark.parametrize("name", ["c2", "c3", "c4"])
def test_device_buffers_at_any_start(tctx, name):
    """x and x_out on the device, in place, one and two values behind 16 bytes: the bits of aligned buffers, also where a layer
    without a norm in front takes the stream for its input."""
    cfg = SMALL[name]
    d = cfg.d
    layers = layers_of(tctx, cfg, 2)
    for norms in ([dict(pre=False, post=True)] * 2, [dict(pre=True), dict(pre=False, beta=0.5)], [dict(pre=True, post=True)] * 2):
        st = pb.Stack(tctx, layers)
        for i, k in enumerate(norms):
            st.set_norm(i, *norm_weights(d, i)[:2], **k)
        for T in (1, 5, 40):
            x = synth.make_activations(T, d, 60 + T)
            want = st.forward(x).copy()
            for shift in (0, 1, 2):
                src, out = (torch.full((T * d + 8,), 55.0, device="cuda") for _ in range(2))
                src[shift:shift + T * d] = torch.from_numpy(x).cuda().view(-1)
                st.set_norm(0, *norm_weights(d, 0)[:2], **norms[0])  # (nothing is recorded any more: the loop runs first)
                for buf in (out, out, src):  # into another buffer, from a recording where there are few tokens, in place
                    st.forward_dev(Buf(src[shift:shift + T * d]), T, Buf(buf[shift:shift + T * d]))
                    tctx.sync()
                    assert bits_equal(buf[shift:shift + T * d].view(T, d).cpu().numpy(), want), (T, shift)
                    assert bool((buf[:shift] == 55.0).all()) and bool((buf[shift + T * d:] == 55.0).all())
        st.close()
    for layer in layers:
        layer.close()


@pytest.mark.parametrize("name, T", [("c2", 1), ("c2", 37), ("c3", 20), ("c4", 200)])
def test_the_operators_together(tctx, name, T):
    """norm -> route -> dispatch -> experts on the rows -> collect beside the shared expert -> norm: the layer's own output."""
    cfg = SMALL[name]
    layer = pb.MoeLayer(tctx, cfg).load(synth.make_weights(cfg, 3))
    d, K, E = cfg.d, cfg.top_k, cfg.n_exp
    x = torch.from_numpy(synth.make_activations(T, d, 11)).cuda()
    new = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    norm = pb.BlockNorm(tctx, d, post=True, pre=True, alpha=0.75)
    xn, out, nxt = new(T, d), new(T, d), new(T, d)
    pb.BlockNorm(tctx, d).forward(T, x.data_ptr(), None, None, xn.data_ptr())
    tctx.sync()
    ids, w = layer.route(xn.cpu().numpy())
    ids_d, w_d = torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(w).cuda()
    rows_op = pb.Rows(tctx, d, K, E)
    R = rows_op.bound(T)
    rows, outs = new(R, d), new(R, d)
    offset, count, pos = new(E + 1, t=torch.int32), new(E, t=torch.int32), new(T, K, t=torch.int32)
    expert, weight = new(R, t=torch.int32), new(R)
    plan = rows_op.plan(R, offset.data_ptr(), count.data_ptr(), pos.data_ptr(), row_expert=expert.data_ptr(), row_weight=weight.data_ptr())
    rows_op.dispatch(T, ids_d.data_ptr(), plan, xn.data_ptr(), rows.data_ptr(), w=w_d.data_ptr(), scale=False)
    pb._check(layer.lib.pm_experts_rows(layer.h, rows.data_ptr(), R, expert.data_ptr(), weight.data_ptr(), outs.data_ptr()))
    shared = torch.from_numpy(layer.shared(xn.cpu().numpy())).cuda() if cfg.shared else None
    folded = cfg.weight_fold == synth.FOLD_BEFORE_DOWN  # the experts have applied the weights already
    y = new(T, d)
    rows_op.collect(T, plan, outs.data_ptr(), y.data_ptr(), w=None if folded else w_d.data_ptr(), add=None if shared is None else shared.data_ptr())
    norm.forward(T, x.data_ptr(), y.data_ptr(), out.data_ptr(), nxt.data_ptr())
    tctx.sync()
    want = layer.forward(xn.cpu().numpy())
    assert tol_ok(y.cpu().numpy(), want)  # (the order of the shared expert's addition differs)
    f, x64 = y.cpu().double(), x.cpu().double()
    r = 0.75 * x64 + f / (f.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    size = float(r.abs().max()) + float(x64.abs().max())  # of the terms; 64 roundings of 2^-24 for each of the two norms
    assert float((out.cpu().double() - r).abs().max()) <= 64 * 2.0 ** -24 * 2 * size
    s = (r.pow(2).mean(1, keepdim=True) + 1e-6).sqrt()
    assert float(((nxt.cpu().double() - r / s) * s).abs().max()) <= 128 * 2.0 ** -24 * 2 * size
    layer.close()


@pytest.mark.parametrize("name", ["c2", "c3", "c4"])
def test_one_layer_against_the_formula(tctx, name):
    """x <- alpha x + beta gate post(moe(pre(x))) in 64 bits around the layer's own call. Rows of +-2^k without eps have the norm 2^k
    exactly, so that the layer's input is +-(offset + weight) to the bit and no int8 value of it may round another way; behind the
    layer the result is off by 40 roundings of 2^-24 of its terms (as the norms alone), and its own."""
    cfg = SMALL[name]
    d = cfg.d
    layers = layers_of(tctx, cfg, 1)
    st = pb.Stack(tctx, layers)
    w_pre, w_post, gate = norm_weights(d, 4)
    for T in (1, 6, 40):
        rng = np.random.default_rng(T)
        x = (rng.choice([-1.0, 1.0], (T, d)) * 2.0 ** (np.arange(T) % 5 - 2)[:, None]).astype(np.float32)
        for pre, post, gated in ((True, True, True), (True, False, False), (False, True, True), (False, False, True)):
            xn = np.sign(x) * (np.float32(1.0) + w_pre) if pre else x
            st.set_norm(0, w_pre, w_post, gate if gated else None, pre=pre, post=post, alpha=0.75, beta=1.5, eps_pre=0.0, eps_post=1e-5,
                        offset_pre=1.0, offset_post=0.5)
            f = layers[0].forward(xn).astype(np.float64)
            p = f / np.sqrt((f * f).mean(1, keepdims=True) + 1e-5) * (0.5 + w_post.astype(np.float64)) if post else f
            a, b = 0.75 * x.astype(np.float64), 1.5 * (gate.astype(np.float64) if gated else 1.0) * p
            bound = 40 * 2.0 ** -24 * (np.abs(a) + np.abs(b)) + 2.0 ** -24 * np.abs(a + b)
            buf = torch.from_numpy(x).cuda()
            for got in (st.forward(x), st.forward(x), st.forward(x)):  # the loop, its recording, a replay
                assert bool((np.abs(got - (a + b)) <= bound).all()), (T, pre, post, gated)
            st.forward_dev(Buf(buf), T, Buf(buf))  # in place on the device
            tctx.sync()
            assert bits_equal(buf.cpu().numpy(), got)
    st.close()
    layers[0].close()


@pytest.mark.parametrize("name, T, align", [("c2", 3, 1), ("c2", 70, 16), ("c3", 45, 1), ("c3", 9, 8), ("c4", 150, 4)])
def test_shards_and_padded_tokens(tctx, name, T, align):
    """Experts on two ranks and a batch with padded tokens: how many rows a rank has is in offset[n_local], which the host reads;
    those rows go through pm_experts_rows, and the ranks' shares add up to the layer's pairs. Padded tokens add nothing."""
    cfg = SMALL[name]
    W = synth.make_weights(cfg, 3)
    layer = pb.MoeLayer(tctx, cfg).load(W)
    d, K, E = cfg.d, cfg.top_k, cfg.n_exp
    x = synth.make_activations(T, d, 12)
    ids, w = layer.route(x)
    pairs = layer.experts_rows(np.repeat(x, K, 0), ids.reshape(-1), w.reshape(-1)).reshape(T, K, d).astype(np.float64)
    folded = cfg.weight_fold == synth.FOLD_BEFORE_DOWN
    padded = np.arange(T) % 3 == 1
    want = (pairs * (1.0 if folded else w.astype(np.float64)[:, :, None])).sum(1)
    want[padded] = 0.0
    ids, w = ids.astype(np.uint32), w.copy()
    ids[padded], w[padded], x[padded] = pb.ROWS_NONE, np.nan, np.inf
    new = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    x_d, ids_d, w_d, y = torch.from_numpy(x).cuda(), torch.from_numpy(ids.view(np.int32)).cuda(), torch.from_numpy(w).cuda(), new(T, d)
    for first, n in ((0, E // 2 - 1), (E // 2 - 1, E - E // 2 + 1)):
        shard = pb.MoeLayer(tctx, cfg.scaled(first_local_expert=first, n_exp_local=n)).load(W)
        op = pb.Rows(tctx, d, K, E, first_expert=first, n_local=n, align=align)
        bound = op.bound(T)
        rows, outs = new(bound, d), new(bound, d)
        offset, count, pos, expert = (new(*s, t=torch.int32) for s in ((n + 1,), (n,), (T, K), (bound,)))
        weight = new(bound)
        plan = op.plan(bound, offset.data_ptr(), count.data_ptr(), pos.data_ptr(), row_expert=expert.data_ptr(), row_weight=weight.data_ptr())
        op.dispatch(T, ids_d.data_ptr(), plan, x_d.data_ptr(), rows.data_ptr(), w=w_d.data_ptr(), scale=False)
        tctx.sync()
        R = int(offset[n])
        assert 0 < R < bound
        pb._check(shard.lib.pm_experts_rows(shard.h, rows.data_ptr(), R, expert.data_ptr(), weight.data_ptr(), outs.data_ptr()))
        op.collect(T, plan, outs.data_ptr(), y.data_ptr(), w=None if folded else w_d.data_ptr(), add=y.data_ptr())
        tctx.sync()  # (an expert that the shard does not have would be reported here)
        shard.close()
    assert tol_ok(y.cpu().numpy(), want) and not y[torch.from_numpy(padded).cuda()].any()
    layer.close()
