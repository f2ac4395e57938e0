"""What the training losses refuse, before any GPU call."""

import ctypes

import pytest
import torch

import fuselse_amd
from fuselse_amd import _lib, ext


def test_public_entries_refuse_cpu_tensors():
    x, w, t = torch.zeros(2, 4), torch.zeros(5, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="x must be CUDA"):
        fuselse_amd.linear_cross_entropy(x, w, t)
    with pytest.raises(RuntimeError, match="logits must be CUDA"):
        fuselse_amd.topk_distillation(x, x[:, :2], torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="logits must be CUDA"):
        fuselse_amd.router_balance(x, torch.zeros(2, 2, dtype=torch.int64))


def test_public_entries_refuse_shapes_and_types():
    x, w = torch.zeros(2, 4), torch.zeros(5, 4)
    with pytest.raises(RuntimeError, match="target must have input's shape"):
        fuselse_amd.linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="target must be an integer tensor"):
        fuselse_amd.linear_cross_entropy(x, w, torch.zeros(2))
    with pytest.raises(RuntimeError, match="teacher_logits and teacher_index"):
        fuselse_amd.topk_distillation(x, torch.zeros(2, 3), torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="teacher_index must be an integer"):
        fuselse_amd.topk_distillation(x, torch.zeros(2, 3), torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="index must be"):
        fuselse_amd.router_balance(x, torch.zeros(3, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="mask must have the shape"):
        fuselse_amd.router_balance(x, torch.zeros(2, 2, dtype=torch.int64), mask=torch.ones(3, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="reduction must be"):
        ext._reduction("average")


VP = ctypes.c_void_p(4096)


def _message(lib):
    return lib.fl_last_error().decode()


def linear_args(lib, **k):
    a = dict(x=VP, ldx=8, w=VP, ldw=8, t=VP, n=4, v=16, d=8, dt=0, ignore=-100, z=0.0, red=2, loss=VP, lse=VP, ws=VP,
             nbytes=1 << 40)
    a.update(k)
    return lib.fl_linear_ce_fwd(a["x"], a["ldx"], a["w"], a["ldw"], a["t"], a["n"], a["v"], a["d"], a["dt"], a["ignore"],
                                a["z"], a["red"], a["loss"], a["lse"], a["ws"], a["nbytes"], None)


@pytest.mark.parametrize("change,code,message", [
    (dict(n=-1), 1, "bad shape"), (dict(v=0), 1, "bad shape"), (dict(d=0), 1, "bad shape"), (dict(dt=3), 1, "dtype"),
    (dict(red=3), 1, "reduction"), (dict(ldx=7), 1, "overlap"), (dict(ldw=7), 1, "overlap"),
    (dict(n=(1 << 23) + 1), 3, "2^23 rows"), (dict(v=(1 << 28) + 1), 3, "2^23 rows"), (dict(x=None), 1, "NULL"),
    (dict(t=None), 1, "NULL"), (dict(x=ctypes.c_void_p(4097)), 1, "element-aligned"), (dict(nbytes=8), 1, "needed"),
    (dict(ws=ctypes.c_void_p(4100)), 1, "256-byte"), (dict(loss=None), 1, "NULL"),
    (dict(lse=None, nbytes=8), 1, "needed"), (dict(n=0, x=None), 0, ""),
])
def test_linear_entry_refusals(change, code, message):
    lib = _lib.load()
    assert linear_args(lib, **change) == code
    assert message in _message(lib)


def test_backward_and_other_entry_refusals():
    lib = _lib.load()
    big = 1 << 40
    assert lib.fl_linear_ce_bwd(None, VP, 8, VP, 8, VP, VP, 4, 16, 8, 0, -100, 0.0, 2, VP, VP, VP, big, None) == 1
    assert "NULL" in _message(lib)
    assert lib.fl_linear_ce_bwd(VP, VP, 8, VP, 8, VP, VP, 4, 16, 8, 0, -100, 0.0, 2, None, None, VP, big, None) == 0
    assert lib.fl_linear_ce_workspace_bytes(0, 4, 4, 0, 0, VP, 4) == 0
    assert lib.fl_linear_ce_workspace_bytes(4, 4, 4, 5, 0, VP, 4) == 0

    def distill(rows=2, n1=2, v=8, dt=0, t=VP, tdt=0, k=2, temp=1.0, red=0, loss=VP, norm=None, ws=VP, nbytes=big):
        return lib.fl_distill_fwd(VP, rows, n1, 8, 8, v, dt, t, tdt, VP, k, temp, red, loss, VP, VP, norm, ws, nbytes,
                                  None)

    for change, code, message in [
            (dict(rows=-1), 1, "bad shape"), (dict(v=0), 1, "bad shape"), (dict(n1=0), 1, "bad shape"),
            (dict(dt=4), 1, "dtype"), (dict(tdt=-1), 1, "dtype"), (dict(temp=0.0), 1, "temperature"),
            (dict(temp=float("nan")), 1, "temperature"), (dict(temp=float("inf")), 1, "temperature"),
            (dict(k=1025), 3, "1024"), (dict(rows=(1 << 22) + 1), 3, "2^22"), (dict(red=5), 1, "reduction"),
            (dict(t=None), 1, "NULL"), (dict(red=2), 1, "NULL"), (dict(nbytes=1), 1, "needed"),
            (dict(ws=ctypes.c_void_p(4)), 1, "8-byte"), (dict(rows=0), 0, "")]:
        assert distill(**change) == code, change
        assert message in _message(lib), change
    assert lib.fl_distill_bwd(VP, 2, None, VP, 2, 2, 8, 8, 8, 0, VP, 0, VP, 2, 1.0, VP, VP, VP, None) == 1
    assert "grad_stride" in _message(lib)
    assert lib.fl_distill_bwd(VP, 1, None, VP, 2, 2, 8, 8, 8, 0, VP, 0, VP, 2, 1.0, VP, VP, None, None) == 1
    assert "NULL" in _message(lib)

    def router(ld=8, tokens=4, experts=8, dt=0, index=VP, top=2, balance=VP, ws=VP, nbytes=big):
        return lib.fl_router_balance_fwd(VP, ld, tokens, experts, dt, index, top, None, balance, VP, VP, VP, VP, ws,
                                         nbytes, None)

    for change, code, message in [
            (dict(tokens=-1), 1, "bad shape"), (dict(experts=0), 1, "bad shape"), (dict(top=-1), 1, "bad shape"),
            (dict(dt=9), 1, "dtype"), (dict(ld=7), 1, "overlap"), (dict(experts=1025, ld=2000), 3, "1024 experts"),
            (dict(tokens=1 << 30, top=2), 3, "2^31"), (dict(index=None), 1, "NULL"), (dict(balance=None), 1, "NULL"),
            (dict(nbytes=4), 1, "needed"), (dict(ws=ctypes.c_void_p(4)), 1, "8-byte")]:
        assert router(**change) == code, change
        assert message in _message(lib), change
    assert lib.fl_router_balance_bwd(None, None, None, 8, 4, 8, 0, None, VP, VP, VP, None) == 1
    assert "NULL" in _message(lib)
    assert lib.fl_router_workspace_bytes(4, 2000, 0) == 0
