"""What the layers around the training losses refuse, before any GPU call."""

import ctypes

import pytest
import torch

import fuselse_amd
from fuselse_amd import ExpertOrder, _lib, ext

VP = ctypes.c_void_p(4096)
BIG = 1 << 50


def order(tokens=2, top=2, experts=4):
    return ExpertOrder(torch.zeros(tokens, top, dtype=torch.int32), torch.zeros(experts, dtype=torch.int64),
                       torch.zeros(experts + 1, dtype=torch.int32))


def test_public_entries_refuse_cpu_tensors():
    x, i = torch.zeros(2, 4), torch.zeros(2, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="weight must be CUDA"):
        fuselse_amd.embedding(i, x)
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        fuselse_amd.layer_norm(x)
    with pytest.raises(RuntimeError, match="index must be CUDA"):
        fuselse_amd.expert_order(i, 4)
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        fuselse_amd.expert_dispatch(x, order())
    with pytest.raises(RuntimeError, match="rows must be CUDA"):
        fuselse_amd.expert_combine(torch.zeros(4, 3), torch.zeros(2, 2), order())
    for name, args in [("embedding", (x, i[0])), ("embedding_backward", (x, i[0], 3)), ("layer_norm", (x,)),
                       ("layer_norm_backward", (x, x, None, None, x)), ("expert_order", (i, 3)),
                       ("expert_dispatch", (x, order().position)),
                       ("expert_combine", (x, None, order().position)),
                       ("expert_combine_backward", (x, x, x, order().position))]:
        with pytest.raises(RuntimeError, match="must be CUDA"):
            getattr(ext, name)(*args)


def test_public_entries_refuse_shapes_and_types():
    x, i = torch.zeros(2, 4), torch.zeros(2, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="index must be an integer tensor"):
        fuselse_amd.embedding(torch.zeros(2), x)
    with pytest.raises(RuntimeError, match="index must be an integer tensor"):
        fuselse_amd.expert_order(torch.zeros(2, 2), 4)
    with pytest.raises(RuntimeError, match="mask must have the shape"):
        fuselse_amd.expert_order(i, 4, mask=torch.ones(3, dtype=torch.bool))
    with pytest.raises(RuntimeError, match=r"index must be \(..., top\)"):
        fuselse_amd.expert_order(torch.zeros((), dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="tokens of order"):
        fuselse_amd.expert_dispatch(torch.zeros(3, 4), order())
    with pytest.raises(RuntimeError, match="shape of order's index"):
        fuselse_amd.expert_combine(x, torch.zeros(2, 3), order())
    with pytest.raises(RuntimeError, match="last dimension"):
        fuselse_amd.layer_norm(torch.zeros(()))


def refused(lib, rc, code, message):
    assert rc == code, (rc, lib.fl_last_error())
    assert message in lib.fl_last_error().decode()


@pytest.mark.parametrize("change,code,message", [
    (dict(n=-1), 1, "bad shape"), (dict(v=0), 1, "bad shape"), (dict(d=0), 1, "bad shape"), (dict(dt=3), 1, "dtype"),
    (dict(n=(1 << 30) + 1), 3, "2^30"), (dict(v=(1 << 30) + 1), 3, "2^30"), (dict(d=(1 << 20) + 1, ld=BIG), 3, "2^20"),
    (dict(ld=7), 1, "overlap"), (dict(a=None), 1, "NULL"), (dict(index=None), 1, "NULL"), (dict(out=None), 1, "NULL"),
    (dict(a=ctypes.c_void_p(4097)), 1, "element-aligned"),
])
def test_embedding_entry_refusals(change, code, message):
    lib = _lib.load()
    p = dict(a=VP, ld=8, v=16, d=8, dt=0, index=VP, n=4, out=VP)
    p.update(change)
    refused(lib, lib.fl_embedding_fwd(p["a"], p["ld"], p["v"], p["d"], p["dt"], p["index"], p["n"], 1.0, p["out"],
                                      None), code, message)
    refused(lib, lib.fl_embedding_bwd(p["a"], p["ld"], p["index"], p["n"], p["v"], p["d"], p["dt"], 1.0, -1, p["out"],
                                      VP, BIG, None), code, message)


def test_embedding_workspace_refusals():
    lib = _lib.load()
    args = (VP, 8, VP, 4, 16, 8, 0, 1.0, -1, VP)
    refused(lib, lib.fl_embedding_bwd(*args, VP, 8, None), 1, "needed")
    refused(lib, lib.fl_embedding_bwd(*args, None, BIG, None), 1, "256-byte")
    refused(lib, lib.fl_embedding_bwd(*args, ctypes.c_void_p(4104), BIG, None), 1, "256-byte")
    assert lib.fl_embedding_fwd(VP, 8, 16, 8, 0, None, 0, 1.0, None, None) == 0
    for n, v, d in [(-1, 1, 1), (1, 0, 1), (1, 1, 0), (1 << 31, 1, 1), (1, 1 << 31, 1), (1, 1, 1 << 21)]:
        assert lib.fl_embedding_bwd_workspace_bytes(n, v, d) == 0
    assert lib.fl_embedding_bwd_workspace_bytes(1 << 30, 1 << 30, 1) > 1 << 33


@pytest.mark.parametrize("change,code,message", [
    (dict(n=-1), 1, "bad shape"), (dict(d=0), 1, "bad shape"), (dict(dt=3), 1, "dtype"), (dict(ld=7), 1, "overlap"),
    (dict(n=1 << 31), 3, "2^31"), (dict(d=(1 << 24) + 1, ld=BIG), 3, "2^24"), (dict(pdt=2), 1, "parameters"),
    (dict(x=None), 1, "NULL"), (dict(x=ctypes.c_void_p(4098)), 1, "aligned"),
    (dict(w=ctypes.c_void_p(4098)), 1, "aligned"), (dict(stats=ctypes.c_void_p(4104)), 1, "16-byte"),
])
def test_layer_norm_entry_refusals(change, code, message):
    lib = _lib.load()
    p = dict(x=VP, ld=8, n=4, d=8, dt=0, w=VP, pdt=0, stats=VP)
    p.update(change)
    refused(lib, lib.fl_layer_norm_fwd(p["x"], p["ld"], p["n"], p["d"], p["dt"], p["w"], VP, p["pdt"], 1e-5, VP,
                                       p["stats"], None), code, message)
    refused(lib, lib.fl_layer_norm_bwd(VP, max(p["ld"], 8), p["x"], p["ld"], p["n"], p["d"], p["dt"], p["w"],
                                       p["pdt"], p["stats"], VP, VP, VP, VP, BIG, None), code, message)


def test_layer_norm_other_refusals():
    lib = _lib.load()
    for eps in (-1e-5, float("nan")):
        refused(lib, lib.fl_layer_norm_fwd(VP, 8, 4, 8, 0, None, None, 0, eps, VP, None, None), 1, "eps")
        with pytest.raises(RuntimeError, match="eps"):
            ext._norm_fwd(torch.zeros(2, 4), None, None, eps, False)
    refused(lib, lib.fl_layer_norm_fwd(VP, 8, 4, 8, 0, None, None, 0, 1e-5, None, None, None), 1, "NULL")
    bwd = (VP, 8, VP, 8, 4, 8, 0, VP, 0)
    refused(lib, lib.fl_layer_norm_bwd(*bwd, None, VP, VP, VP, VP, BIG, None), 1, "NULL")
    refused(lib, lib.fl_layer_norm_bwd(*bwd, VP, VP, VP, None, VP, 4, None), 1, "needed")
    refused(lib, lib.fl_layer_norm_bwd(*bwd, VP, VP, None, VP, None, BIG, None), 1, "4-byte")
    refused(lib, lib.fl_layer_norm_bwd(VP, 7, *bwd[2:], VP, VP, VP, VP, VP, BIG, None), 1, "overlap")
    # nothing wanted, nothing to do
    assert lib.fl_layer_norm_bwd(*bwd, VP, None, None, None, None, 0, None) == 0
    assert lib.fl_layer_norm_fwd(None, 8, 0, 8, 0, None, None, 0, 1e-5, None, None, None) == 0
    for n, d, dt in [(-1, 4, 0), (4, 0, 0), (4, (1 << 24) + 1, 0), (4, 4, 3)]:
        assert lib.fl_layer_norm_bwd_workspace_bytes(n, d, dt) == 0


@pytest.mark.parametrize("change,code,message", [
    (dict(t=-1), 1, "bad shape"), (dict(k=0), 1, "bad shape"), (dict(e=0), 1, "bad shape"),
    (dict(e=1025), 3, "1024 experts"), (dict(k=1025), 3, "1024 choices"), (dict(t=(1 << 30) + 1), 3, "2^30"),
    (dict(t=1 << 30, k=2), 3, "2^31"), (dict(index=None), 1, "NULL"), (dict(position=None), 1, "NULL"),
    (dict(counts=None), 1, "NULL"), (dict(offsets=None), 1, "NULL"), (dict(t=4096, nbytes=8), 1, "needed"),
    (dict(t=4096, ws=None), 1, "4-byte"), (dict(t=4096, ws=ctypes.c_void_p(4098)), 1, "4-byte"),
])
def test_expert_order_entry_refusals(change, code, message):
    lib = _lib.load()
    p = dict(index=VP, t=4, k=2, e=8, position=VP, counts=VP, offsets=VP, ws=VP, nbytes=BIG)
    p.update(change)
    refused(lib, lib.fl_expert_order(p["index"], p["t"], p["k"], p["e"], None, p["position"], p["counts"],
                                     p["offsets"], p["ws"], p["nbytes"], None), code, message)


def test_expert_row_entry_refusals():
    lib = _lib.load()

    def dispatch(x=VP, ld=8, t=4, d=8, dt=0, pos=VP, k=2, rows=VP):
        return lib.fl_expert_dispatch(x, ld, t, d, dt, pos, k, rows, None)

    def combine(rows=VP, ld=8, t=4, d=8, dt=0, pos=VP, k=2, w=VP, wdt=0, out=VP):
        return lib.fl_expert_combine(rows, ld, t, d, dt, pos, k, w, wdt, out, None)

    def bwd(g=VP, ldg=8, rows=VP, ld=8, t=4, d=8, dt=0, pos=VP, k=2, w=VP, wdt=0, dr=VP, dw=VP):
        return lib.fl_expert_combine_bwd(g, ldg, rows, ld, t, d, dt, pos, k, w, wdt, dr, dw, None)

    for f in (dispatch, combine, bwd):
        for change, code, message in [
                (dict(t=-1), 1, "bad shape"), (dict(k=0), 1, "bad shape"), (dict(d=0), 1, "D=0"),
                (dict(dt=3), 1, "dtype"), (dict(ld=7), 1, "overlap"), (dict(k=1025), 3, "1024 choices"),
                (dict(t=1 << 30, k=2), 3, "2^31"), (dict(d=(1 << 24) + 1, ld=BIG), 3, "2^24"),
                (dict(pos=None), 1, "NULL"), (dict(rows=None), 1, "NULL"), (dict(t=0, pos=None), 0, "")]:
            refused(lib, f(**change), code, message)
    refused(lib, dispatch(x=None), 1, "NULL")
    refused(lib, dispatch(x=ctypes.c_void_p(4098)), 1, "element-aligned")
    refused(lib, combine(wdt=2), 1, "weights' dtype")
    refused(lib, combine(out=None), 1, "NULL")
    refused(lib, bwd(ldg=7), 1, "overlap")
    refused(lib, bwd(w=None), 1, "NULL")
    refused(lib, bwd(wdt=1), 1, "weights' dtype")
    assert bwd(dr=None, dw=None) == 0
    assert lib.fl_expert_order_workspace_bytes(4, 2, 2000) == 0
    assert lib.fl_expert_order_workspace_bytes(4, 2, 8) == 0
    assert lib.fl_expert_order_workspace_bytes(4097, 1, 8) > 0


def test_positions_are_checked():
    x = torch.zeros(2, 4)
    for bad in (torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32),
                torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="position must be"):
            ext._check_position(x, "x", bad)
