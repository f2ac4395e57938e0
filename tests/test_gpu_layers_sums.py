"""Sums over many tokens and rows against whole numbers, which they hold exactly in
whatever order they are made: what is lost, doubled or put elsewhere shows at any
length, where a bound on rounding grows with it."""

import numpy as np
import pytest
import torch

import fuselse_amd
from test_gpu_layers import randint
from test_gpu_losses import DTYPES

pytestmark = pytest.mark.gpu


def whole(cuda, most, *shape, seed=0):
    """Whole numbers of [-most, most]."""
    return (randint(cuda, 2 * most + 1, *shape, seed=seed) - most).float()


def check_embedding(index, v, d, dtype, scale=1.0, padding=None):
    cuda, n = index.device, index.numel()
    table = torch.zeros(v, d, dtype=dtype, device=cuda, requires_grad=True)
    g = whole(cuda, 8, n, d, seed=n + d)
    (dw,) = torch.autograd.grad(fuselse_amd.embedding(index, table, scale=scale, padding_idx=padding), table,
                                g.to(dtype))
    keep = torch.ones_like(index, dtype=torch.bool) if padding is None else index != padding
    want = torch.zeros(v, d, dtype=torch.float64, device=cuda)
    ids = index[keep].unique()
    if ids.numel() <= 16:  # many additions to one row take long
        for i in ids.tolist():
            want[i] = g[index == i].sum(0, dtype=torch.float64)
    else:
        want.index_add_(0, index[keep], g[keep].double())
    assert float(want.abs().max()) < 2 ** 24
    assert torch.equal(dw, (want * scale).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 5, 64, 520])
@pytest.mark.parametrize("n", [2, 15, 16, 17, 33, 513, 1025, 8191, 8193, 40000, 131073, 200001])
def test_embedding_one_token(cuda, n, d, dtype):
    print(f"case whole one token {n} {d} {dtype}", flush=True)
    index = torch.full((n,), 41, device=cuda)
    check_embedding(index, 77, d, dtype)
    # and with others on both sides of it in the order
    index[::3] = 40
    index[1::7] = 76
    check_embedding(index, 77, d, dtype, scale=0.5, padding=40)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,d", [(5000, 5, 64), (8192, 3, 520), (40000, 5, 12), (131073, 5, 65), (200001, 2, 3),
                                   (70000, 11, 1030)])
def test_embedding_few_tokens(cuda, n, v, d, dtype):
    print(f"case whole few tokens {n} {v} {d} {dtype}", flush=True)
    check_embedding(randint(cuda, v, n, seed=1), v, d, dtype)


@pytest.mark.parametrize("run", [15, 16, 17, 31, 32, 33, 63, 64, 65, 1000])
@pytest.mark.parametrize("n,d", [(5000, 24), (9000, 520), (131072, 8), (65536, 1024)])
def test_embedding_runs(cuda, n, d, run):
    """Equal ids in runs that end at and around the borders of what a wave sums, 16
    entries or 64."""
    print(f"case whole runs {n} {d} {run}", flush=True)
    at = torch.arange(n, device=cuda) // run
    v = int(at[-1]) + 1
    check_embedding(at, v, d, torch.float32)
    check_embedding(at[torch.randperm(n, generator=torch.Generator().manual_seed(run)).to(cuda)], v, d, torch.bfloat16)


ROWS = [(2, 200001), (4, 131073), (6, 262145), (8, 200001), (40, 50000), (72, 16385), (768, 9000), (768, 20001),
        (1000, 5000), (2048, 4097), (4096, 2049), (4104, 1500), (8192, 1500), (16384, 3000), (16392, 1100),
        (20000, 700), (32768, 900), (40000, 1000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,n", ROWS)
def test_layer_norm_parameters(cuda, d, n, dtype):
    """Rows of as many 1 as -1 with eps 0: mean 0, mean square D fl(1 / D), which is 1
    for these D, so that x normalised is x, and dw and db are sums of whole numbers."""
    print(f"case whole norm {d} {n} {dtype}", flush=True)
    assert np.float32(d) * (np.float32(1) / np.float32(d)) == 1
    turn = randint(cuda, d, n, seed=d)[:, None]
    x = torch.where((torch.arange(d, device=cuda) + turn) % d < d // 2, 1.0, -1.0).to(dtype)
    g = whole(cuda, 4, n, d, seed=n).to(dtype)
    w = torch.ones(d, device=cuda, requires_grad=True)
    b = torch.zeros(d, device=cuda, requires_grad=True)
    for leaf in (x, x.clone().requires_grad_(True)):  # the parameters' gradients alone, and with dx
        y = fuselse_amd.layer_norm(leaf, w, b, eps=0.0)
        assert torch.equal(y.detach(), x)
        dw, db = torch.autograd.grad(y, [w, b] + ([leaf] if leaf.requires_grad else []), g)[:2]
        assert torch.equal(db.double(), g.sum(0, dtype=torch.float64))
        assert torch.equal(dw.double(), (g.float() * x.float()).sum(0, dtype=torch.float64))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,k,d", [(50, 3, 7), (200, 8, 40), (300, 2, 512), (300, 8, 520), (100, 3, 1100), (60, 1, 4104),
                                   (40, 2, 8200), (30, 9, 16384), (5, 100, 2100)])
def test_experts_weights(cuda, t, k, d, dtype):
    """Dot products, and sums over a token's choices."""
    print(f"case whole experts {t} {k} {d} {dtype}", flush=True)
    order = fuselse_amd.expert_order(randint(cuda, 9, t, k, seed=2) - 1, 8)
    live = order.position >= 0
    at = torch.where(live, order.position, 0).long()
    rows = whole(cuda, 4, t * k, d, seed=3).to(dtype).requires_grad_(True)
    w = whole(cuda, 2, t, k, seed=4).requires_grad_(True)
    x = torch.zeros(t, d, dtype=dtype, device=cuda, requires_grad=True)
    y = fuselse_amd.expert_combine(rows, w, order)
    g, g_rows = whole(cuda, 4, t, d, seed=5).to(dtype), whole(cuda, 1, t * k, d, seed=6).to(dtype)
    d_w, dx = torch.autograd.grad((y, fuselse_amd.expert_dispatch(x, order)), (w, x), (g, g_rows))
    made = rows.detach().double()[at] * live[..., None]
    assert torch.equal(y.detach(), (made * w.detach()[..., None]).sum(1).to(dtype))
    assert torch.equal(d_w.double(), (made * g.double()[:, None]).sum(-1))
    assert torch.equal(dx, (g_rows.double()[at] * live[..., None]).sum(1).to(dtype))
