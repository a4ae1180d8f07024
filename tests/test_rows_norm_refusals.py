"""What the row and norm operators refuse before they look at a GPU: descriptors, token counts, a missing context."""
import ctypes as C
import gc
import types
import weakref

import pytest

import pelica_b200 as pb
from pelica_b200 import synth

LIB = pb.load_library()
ROWS = dict(dtype=synth.BF16, d=64, top_k=2, n_exp=8, first_expert=0, n_local=0, align=1)
NORM = dict(dtype=synth.F16, wtype=synth.F32, d=64, flags=3, gate=1, eps_post=1e-6, eps_pre=1e-6, alpha=1.0, beta=1.0)


def rows_calls(desc, T):
    plan = pb.RowsPlan(None, None, None, None, None, None, 1 << 20)
    d, p = C.byref(desc), C.byref(plan)
    return [LIB.pm_rows_bound(d, T), LIB.pm_dispatch_rows(None, d, T, None, None, p, None, None, 0),
            LIB.pm_dispatch_rows_grad(None, d, T, p, None, None, None, None, None),
            LIB.pm_collect_rows(None, d, T, p, None, None, None, None),
            LIB.pm_collect_rows_grad(None, d, T, p, None, None, None, None, None)]


def norm_calls(desc, T):
    d = C.byref(desc)
    return [LIB.pm_block_norm(None, d, T, *[None] * 7), LIB.pm_block_norm_grad(None, d, T, *[None] * 13, 0)]


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=synth.Q8_0), -2, "type"), (dict(dtype=-1), -2, "type"), (dict(d=0), -7, "d=0"), (dict(d=49153), -7, "d=49153"),
    (dict(top_k=0), -7, "top_k"), (dict(top_k=17), -7, "top_k"), (dict(n_exp=0), -7, "n_exp"), (dict(n_exp=513), -7, "n_exp"),
    (dict(first_expert=-1, n_local=2), -1, "experts"), (dict(first_expert=7, n_local=2), -1, "experts"),
    (dict(first_expert=3, n_local=0), -1, "experts"), (dict(n_local=-1), -1, "experts"), (dict(first_expert=2**31 - 1, n_local=2), -1, "experts"),
    (dict(align=0), -7, "align"), (dict(align=257), -7, "align"), (dict(reserved=1), -1, "reserved"),
    (dict(x_stride=63), -1, "stride"), (dict(rows_stride=-64), -1, "stride")])
def test_row_descriptors(change, code, word):
    desc = pb.RowsDesc(**{**ROWS, **change})
    for got in rows_calls(desc, 4):
        assert got == code
        assert word in LIB.pm_last_error().decode()


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=synth.Q4_K), -2, "type"), (dict(wtype=synth.BF16), -2, "weight type"), (dict(d=0), -7, "d=0"), (dict(d=49153), -7, "d="),
    (dict(flags=4), -1, "flags"), (dict(gate=3), -1, "gate"), (dict(gate=-1), -1, "gate"), (dict(eps_pre=-1.0), -1, "eps"),
    (dict(eps_post=float("nan")), -1, "eps"), (dict(reserved=2), -1, "reserved"), (dict(f_stride=8), -1, "stride")])
def test_norm_descriptors(change, code, word):
    desc = pb.NormDesc(**{**NORM, **change})
    for got in norm_calls(desc, 4):
        assert got == code
        assert word in LIB.pm_last_error().decode()


@pytest.mark.parametrize("T", [-1, 16385])
def test_token_counts(T):
    for got in rows_calls(pb.RowsDesc(**ROWS), T) + norm_calls(pb.NormDesc(**NORM), T):
        assert got == -7


def test_a_context_and_a_descriptor_are_needed():
    assert rows_calls(pb.RowsDesc(**ROWS), 4)[1:] == [-1] * 4 and norm_calls(pb.NormDesc(**NORM), 4) == [-1] * 2
    assert "null context" in LIB.pm_last_error().decode()
    assert LIB.pm_rows_bound(None, 4) == -1 and LIB.pm_block_norm_scratch(None, C.byref(pb.NormDesc(**NORM)), 4) == 0


@pytest.mark.parametrize("T, top_k, n_exp, n_local, align, want", [
    (0, 2, 8, 0, 16, 0), (1, 2, 8, 0, 1, 2), (1, 2, 8, 0, 16, 2 + 2 * 15), (100, 2, 8, 0, 16, 200 + 8 * 15), (100, 2, 8, 3, 16, 200 + 3 * 15),
    (16384, 16, 512, 0, 256, 262144 + 512 * 255)])
def test_bound_of_rows(T, top_k, n_exp, n_local, align, want):
    assert LIB.pm_rows_bound(C.byref(pb.RowsDesc(synth.F32, 64, top_k, n_exp, 0, n_local, align)), T) == want


def test_a_plan_keeps_its_buffers():
    """A plan holds addresses for the library: the buffers that it was given live as long as it does."""
    class Buffer:
        ptr = 256

    rows = pb.Rows(types.SimpleNamespace(lib=LIB, h=None), 64, 2, 8)
    buffers = [Buffer() for _ in range(6)]
    seen = [weakref.ref(b) for b in buffers]
    plan = rows.plan(64, *buffers)
    del buffers
    gc.collect()
    assert all(r() is not None for r in seen) and plan.pos == 256 and plan.max_rows == 64
    del plan
    gc.collect()
    assert not any(r() is not None for r in seen)
    assert rows.plan(64, 1, 2, 3).row_pair is None  # (addresses, and none)
