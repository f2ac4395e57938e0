"""How the layers around the training losses are called: compiled and Python
paths, graphs, streams, devices, saved-tensor hooks, second derivatives, large
offsets, and a step of a model in which all of them run."""

import math

import pytest
import torch

import fuselse_amd
from fuselse_amd import _lib, layers
from test_gpu_layers import randint, randn
from test_gpu_losses import E23, u, within

pytestmark = pytest.mark.gpu


class _None:
    """Stands in for the compiled calls and leaves every call to Python."""

    def __getattr__(self, name):
        return lambda *args: None


def inputs(cuda, dtype=torch.bfloat16, seed=0):
    n, d, v, e, k = 150, 72, 300, 6, 3
    s = {"ids": randint(cuda, v, n, seed=seed), "table": randn(cuda, v, d, seed=seed + 1).to(dtype),
         "w": randn(cuda, d, seed=seed + 2), "b": randn(cuda, d, seed=seed + 3),
         "index": randint(cuda, e + 1, n, k, seed=seed + 4) - 1, "mask": randint(cuda, 4, n, seed=seed + 5) > 0,
         "gates": torch.softmax(randn(cuda, n, k, seed=seed + 6), -1), "g": randn(cuda, n, d, seed=seed + 7).to(dtype),
         "made": randn(cuda, n * k, d, seed=seed + 8).to(dtype), "experts": e}
    for name in ("table", "w", "b", "gates", "made"):
        s[name].requires_grad_(True)
    return s


def chain(s):
    """Lookup, norm, order, rows to the experts and back: outputs and gradients."""
    x = fuselse_amd.layer_norm(fuselse_amd.embedding(s["ids"], s["table"], scale=1.5, padding_idx=0), s["w"], s["b"])
    order = fuselse_amd.expert_order(s["index"], s["experts"], mask=s["mask"])
    rows = fuselse_amd.expert_dispatch(x, order)
    y = fuselse_amd.expert_combine(rows * s["made"], s["gates"], order)
    grads = torch.autograd.grad(y, [s[name] for name in ("table", "w", "b", "gates", "made")], s["g"])
    return [order.position, order.counts, order.offsets, rows.detach(), y.detach(), *grads]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_compiled_and_python_calls_give_the_same_bits(cuda, monkeypatch, dtype):
    s = inputs(cuda, dtype)
    compiled = chain(s)
    with torch.no_grad():
        plain = fuselse_amd.layer_norm(fuselse_amd.embedding(s["ids"], s["table"]), s["w"], s["b"])
    monkeypatch.setattr(layers, "_common", _None())
    assert same(chain(s), compiled)
    with torch.no_grad():
        assert torch.equal(plain, fuselse_amd.layer_norm(fuselse_amd.embedding(s["ids"], s["table"]), s["w"], s["b"]))


def test_parameters_and_subclasses(cuda, monkeypatch):
    """torch.nn.Parameter takes the compiled call; other subclasses the Python one."""
    s = inputs(cuda)
    want = chain(s)
    for name in ("table", "w", "b"):
        s[name] = torch.nn.Parameter(s[name].detach())
    assert same(chain(s), want)

    class Sub(torch.Tensor):
        pass

    assert layers._bind().layer_norm(s["g"].as_subclass(Sub), s["w"], s["b"], 1e-5) is None
    assert torch.equal(torch.Tensor(fuselse_amd.layer_norm(s["g"].as_subclass(Sub), s["w"], s["b"]).detach().float()),
                       fuselse_amd.layer_norm(s["g"], s["w"], s["b"]).detach().float())


def test_compiled_calls_leave_other_calls(cuda):
    c = layers._bind()
    s = inputs(cuda)
    x, w = s["g"], s["w"]
    order = fuselse_amd.expert_order(s["index"], 6)
    assert c.layer_norm(x.double(), w, None, 1e-5) is None
    assert c.layer_norm(x[:, :40], w[:40], None, 1e-5) is None
    assert c.layer_norm(x, w.half(), None, 1e-5) is None and c.layer_norm(x, w[1:], None, 1e-5) is None
    assert c.layer_norm(x, w, None, -1.0) is None and c.layer_norm(x[:0], w, None, 1e-5) is None
    assert c.layer_norm(x.cpu(), w, None, 1e-5) is None and c.layer_norm(x, w.cpu(), None, 1e-5) is None
    assert c.embedding(s["ids"].int(), s["table"], 1.0, -1) is None
    assert c.embedding(s["ids"], s["table"].t(), 1.0, -1) is None
    assert c.expert_order(s["index"].int(), 6, None) is None and c.expert_order(s["index"], 0, None) is None
    assert c.expert_order(s["index"], 6, s["mask"][1:]) is None and c.expert_order(s["index"], 6, s["mask"].int()) is None
    assert c.expert_dispatch(x[1:], order.position) is None and c.expert_dispatch(x, order.position.long()) is None
    assert c.expert_combine(s["made"], s["gates"].half(), order.position) is None
    assert c.expert_combine(s["made"][1:], s["gates"], order.position) is None
    with pytest.raises(TypeError):
        c.layer_norm(x, w, None, "1e-5")
    with pytest.raises(RuntimeError, match="1024 experts"):
        fuselse_amd.expert_order(s["index"], 1025)


def test_library_that_is_not_built_raises(cuda, monkeypatch):
    import sys

    monkeypatch.setattr(layers, "_common", None)
    monkeypatch.setitem(sys.modules, "fuselse_amd._layers", None)
    monkeypatch.delattr(fuselse_amd, "_layers", raising=False)
    with pytest.raises(_lib.NativeLibraryMissing, match="_layers.so"):
        fuselse_amd.layer_norm(torch.zeros(2, 4, device=cuda))


@pytest.mark.parametrize("python", [False, True])
def test_differentiable_once(cuda, monkeypatch, python):
    if python:
        monkeypatch.setattr(layers, "_common", _None())
    s = inputs(cuda, torch.float32)
    order = fuselse_amd.expert_order(s["index"], 6)
    calls = {"layer_norm": lambda x: fuselse_amd.layer_norm(x, s["w"], s["b"]),
             "dispatch": lambda x: fuselse_amd.expert_dispatch(x, order)}
    for name, f in calls.items():
        x = s["g"].clone().requires_grad_(True)
        y = f(x)
        up = torch.ones_like(y).requires_grad_(True)
        (g,) = torch.autograd.grad(y, x, up, create_graph=True)
        with pytest.raises(RuntimeError, match="once"):
            g.sum().backward()
        # create_graph alone is no error, where nothing differentiates again
        y = f(x)
        (h,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
        assert torch.equal(g.detach(), h.detach()), name


@pytest.mark.parametrize("python", [False, True])
def test_saved_tensor_hooks(cuda, monkeypatch, python):
    """Hooks that give saved tensors back in another layout, or from the host."""
    if python:
        monkeypatch.setattr(layers, "_common", _None())
    s = inputs(cuda)
    want = chain(s)

    def odd(t):
        if t.dim() != 2 or t.dtype not in (torch.bfloat16, torch.float32) or t.shape[1] == 4:
            return t
        return t.t().contiguous().t()

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, odd):
        assert same(chain(s), want)
    with torch.autograd.graph.save_on_cpu():
        assert same(chain(s), want)


def test_a_saved_tensor_that_was_written_is_an_error(cuda):
    s = inputs(cuda)
    x = s["g"].clone().requires_grad_(True) * 1
    y = fuselse_amd.layer_norm(x, s["w"], s["b"])
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_unused_gradients_are_not_made(cuda):
    s = inputs(cuda)
    want = dict(zip(("table", "w", "b", "gates", "made"), chain(s)[5:]))
    x = fuselse_amd.layer_norm(fuselse_amd.embedding(s["ids"], s["table"], scale=1.5, padding_idx=0), s["w"], s["b"])
    order = fuselse_amd.expert_order(s["index"], s["experts"], mask=s["mask"])
    y = fuselse_amd.expert_combine(fuselse_amd.expert_dispatch(x, order) * s["made"], s["gates"], order)
    for name in want:
        (g,) = torch.autograd.grad(y, s[name], s["g"], retain_graph=True)
        assert torch.equal(g, want[name]), name


def test_autocast_keeps_types(cuda):
    s = inputs(cuda)
    want = chain(s)
    with torch.autocast("cuda", torch.float16):
        got = chain(s)
    assert got[4].dtype == torch.bfloat16 and same(got, want)


def test_graph_capture_and_replay(cuda):
    """A captured step, replayed on new values between eager work, gives what the
    eager step gives."""
    s = inputs(cuda)
    fresh = [inputs(cuda, seed=seed) for seed in (20, 40, 60)]
    names = ("ids", "table", "w", "b", "index", "mask", "gates", "g", "made")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            chain(s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = chain(s)
    for _ in range(2):
        for f in fresh:
            with torch.no_grad():
                for name in names:
                    s[name].copy_(f[name])
            graph.replay()
            torch.cuda.synchronize()
            assert same([t.clone() for t in out], chain(f))


def test_two_captured_graphs_and_large_sort(cuda):
    """Two graphs, each with a gradient whose sort takes several launches, replayed
    in turn and on two streams at once."""
    def step(ids, table, g):
        return torch.autograd.grad(fuselse_amd.embedding(ids, table), table, g)[0]

    sets = []
    for seed, n in ((0, 9000), (5, 20000)):
        ids = randint(cuda, 5000, n, seed=seed) // 3
        table = randn(cuda, 5000, 40, seed=seed + 1).requires_grad_(True)
        sets.append((ids, table, randn(cuda, n, 40, seed=seed + 2)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(*a) for a in sets]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step(*a))
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        step(*sets[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_streams(cuda):
    """Two streams at once, with their own workspaces."""
    sets = [inputs(cuda, seed=seed) for seed in (0, 100)]
    want = [chain(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i].append(chain(s))
    torch.cuda.synchronize()
    assert all(same(g, w) for gs, w in zip(got, want) for g in gs)


def test_another_device_than_the_current_one(cuda):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    there = torch.device("cuda:1")
    s = inputs(cuda)
    t = {k: v.detach().to(there).requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) else v
         for k, v in s.items()}
    assert same([a.cpu() for a in chain(t)], [a.cpu() for a in chain(s)])
    with pytest.raises(RuntimeError, match="same device"):
        fuselse_amd.embedding(s["ids"], t["table"])


def test_results_do_not_depend_on_the_run(cuda):
    ids = randint(cuda, 2000, 70000) ** 2 // 2000
    table = randn(cuda, 2000, 1000).bfloat16().requires_grad_(True)
    g = randn(cuda, 70000, 1000, seed=1).bfloat16()
    first = torch.autograd.grad(fuselse_amd.embedding(ids, table), table, g)[0]
    for _ in range(5):
        assert torch.equal(torch.autograd.grad(fuselse_amd.embedding(ids, table), table, g)[0], first)


# ---------------------------------------------------------------------------
# Offsets that pass 32 bits
# ---------------------------------------------------------------------------
def test_large_embedding(cuda):
    """A matrix and a result of more than 2^32 bytes and 2^31 elements."""
    v, d, n = 600000, 4096, 530000
    table = torch.empty(v, d, dtype=torch.bfloat16, device=cuda)
    table.copy_((torch.arange(v, device=cuda) % 251)[:, None].expand(v, d))
    ids = (torch.arange(n, device=cuda) * 7919 + 599999) % v
    table.requires_grad_(True)
    out = fuselse_amd.embedding(ids, table)
    for at in (0, 1, n // 2, n - 2, n - 1):
        assert (out.detach()[at] == int(ids[at]) % 251).all()
    del out
    g = torch.empty(n, d, dtype=torch.bfloat16, device=cuda)
    g.copy_((torch.arange(n, device=cuda) % 127)[:, None].expand(n, d))
    from fuselse_amd import ext

    dw = ext.embedding_backward(g, ids, v)
    want = torch.zeros(v, device=cuda).index_add_(0, ids, (torch.arange(n, device=cuda) % 127).float())
    for c in (0, 1, d // 2, d - 1):
        assert torch.equal(dw[:, c].float(), want.bfloat16().float())


@pytest.mark.parametrize("n", [5000, 9000])
def test_embedding_of_the_largest_vocabulary(cuda, n):
    """Ids of 31 bits, sorted by as many digits as they take."""
    from fuselse_amd import ext

    v = 1 << 30
    table = torch.zeros(v, 1, dtype=torch.float16, device=cuda)
    ids = torch.cat([randint(cuda, v, n - 4), torch.tensor([0, v - 1, v - 1, v // 2], device=cuda)])
    table[ids, 0] = (ids % 1000).half()
    assert torch.equal(fuselse_amd.embedding(ids, table)[:, 0], (ids % 1000).half())
    dw = ext.embedding_backward(torch.ones(n, 1, dtype=torch.float16, device=cuda), ids, v)
    unique, counts = ids.unique(return_counts=True)
    assert torch.equal(dw[unique, 0], counts.half())
    assert int(torch.count_nonzero(dw)) == unique.numel()
    with pytest.raises(RuntimeError, match="2\\^30"):
        ext.embedding_backward(torch.ones(1, 1, dtype=torch.float16, device=cuda), ids[:1], v + 1)


def test_large_layer_norm(cuda):
    n, d = 530000, 4096
    x = torch.empty(n, d, dtype=torch.bfloat16, device=cuda)
    row = randn(cuda, 64, d).bfloat16()
    for first in range(0, n, 64):
        x[first:first + 64] = row[:n - first]
    w, b = randn(cuda, d, seed=1), randn(cuda, d, seed=2)
    small = row.clone().requires_grad_(True)
    want = fuselse_amd.layer_norm(small, w, b)
    y = fuselse_amd.layer_norm(x, w, b)
    for first in (0, 262144 - 64, 529984 - 64):
        assert torch.equal(y[first:first + 64], want.detach()[:64])
    del y
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(fuselse_amd.layer_norm(x, w, b), x, x.detach())
    (ds,) = torch.autograd.grad(want, small, row)
    for first in (0, 262144 - 64, 529984 - 64):
        assert torch.equal(dx[first:first + 64], ds)


def test_large_experts(cuda):
    t, k, e, d = 150000, 8, 64, 2048
    index = randint(cuda, e, t, k)
    order = fuselse_amd.expert_order(index, e)
    x = torch.empty(t, d, dtype=torch.bfloat16, device=cuda)
    x.copy_((torch.arange(t, device=cuda) % 251)[:, None].expand(t, d))
    rows = fuselse_amd.expert_dispatch(x, order)
    token = torch.empty(t * k, dtype=torch.int64, device=cuda)
    token[order.position.reshape(-1).long()] = torch.arange(t, device=cuda).repeat_interleave(k)
    for c in (0, d - 1):
        assert torch.equal(rows[:, c].float(), (token % 251).float())
    w = torch.full((t, k), 0.125, device=cuda)
    assert torch.equal(fuselse_amd.expert_combine(rows, w, order), x)  # eighths of small integers: exact
    rows.requires_grad_(True)
    w.requires_grad_(True)
    d_rows, d_w = torch.autograd.grad(fuselse_amd.expert_combine(rows, w, order), (rows, w), x)
    assert torch.equal(d_rows[:, -1].float(), (token % 251).float() / 8)
    assert torch.equal(d_w, ((torch.arange(t, device=cuda) % 251).float() ** 2 * d)[:, None].expand(t, k))


# ---------------------------------------------------------------------------
# All of them in a step of a model
# ---------------------------------------------------------------------------
def model_state(cuda, seed=0):
    n, d, v, e, k = 96, 64, 211, 5, 2
    s = {"ids": randint(cuda, v, n, seed=seed), "target": randint(cuda, v, n, seed=seed + 1),
         "mask": randint(cuda, 5, n, seed=seed + 2) > 0, "k": k, "experts": e}
    for name, shape, size in (("table", (v, d), 0.5), ("router", (d, e), 0.3), ("up", (e, d, d), 0.125)):
        s[name] = (randn(cuda, *shape, seed=seed + len(name)) * size).requires_grad_(True)
    for i in (1, 2):
        s[f"w{i}"] = (1 + 0.1 * randn(cuda, d, seed=seed + 20 + i)).requires_grad_(True)
        s[f"b{i}"] = (0.1 * randn(cuda, d, seed=seed + 30 + i)).requires_grad_(True)
    s["target"] = torch.where(s["mask"], s["target"], -100)
    return s


LEAVES = ("table", "router", "up", "w1", "b1", "w2", "b2")


def model_step(s):
    """One block of experts between the lookup and the head, whose matrix is the
    lookup's, with the router's losses."""
    d = s["table"].shape[1]
    x = fuselse_amd.embedding(s["ids"], s["table"], scale=math.sqrt(d))
    h = fuselse_amd.layer_norm(x, s["w1"], s["b1"])
    logits = h @ s["router"]
    top = logits.topk(s["k"], -1)
    aux = fuselse_amd.router_balance(logits, top.indices, mask=s["mask"])
    order = fuselse_amd.expert_order(top.indices, s["experts"], mask=s["mask"])
    assert torch.equal(order.counts, aux.counts)
    rows = fuselse_amd.expert_dispatch(h, order)
    ends = order.offsets.tolist()
    made = torch.zeros_like(rows)
    for e in range(s["experts"]):
        part = slice(ends[e], ends[e + 1])
        made = made.index_copy(0, torch.arange(ends[e], ends[e + 1], device=rows.device), rows[part] @ s["up"][e])
    y = x + fuselse_amd.expert_combine(made, torch.softmax(top.values, -1), order)
    out = fuselse_amd.layer_norm(y, s["w2"], s["b2"])
    loss = fuselse_amd.linear_cross_entropy(out, s["table"], s["target"])
    total = loss + 0.01 * aux.balance_loss + 0.001 * aux.z_loss
    return total, torch.autograd.grad(total, [s[name] for name in LEAVES])


def model_exact(s):
    """The same in 64 bits, every token by itself."""
    t = {k: v.detach().double().requires_grad_(True) if k in LEAVES else v for k, v in s.items()}
    d = t["table"].shape[1]
    x = t["table"][t["ids"]] * math.sqrt(d)
    h = torch.nn.functional.layer_norm(x, (d,), t["w1"], t["b1"])
    logits = h @ t["router"]
    top = logits.topk(t["k"], -1)
    mask = t["mask"]
    probs = torch.softmax(logits[mask], -1)
    n = int(mask.sum())
    counts = torch.bincount(top.indices[mask].reshape(-1), minlength=t["experts"]).double()
    balance = t["experts"] * (counts / (n * t["k"]) * probs.mean(0)).sum()
    z = (torch.logsumexp(logits[mask], -1) ** 2).mean()
    gates = torch.softmax(top.values, -1)
    made = (h[:, None, None] @ t["up"][top.indices])[:, :, 0]
    y = x + torch.where(mask[:, None], (gates[..., None] * made).sum(1), 0.0)
    out = torch.nn.functional.layer_norm(y, (d,), t["w2"], t["b2"])
    loss = torch.nn.functional.cross_entropy(out @ t["table"].t(), t["target"], ignore_index=-100)
    total = loss + 0.01 * balance + 0.001 * z
    return total, torch.autograd.grad(total, [t[name] for name in LEAVES])


@pytest.mark.parametrize("seed", [0, 50])
def test_a_models_step(cuda, seed):
    """Loss and gradients of a step in fp32 against 64 bits.

    Tolerance: each of the step's ten layers is off by at most 2^-16 of its
    result's size (64 and 211 terms a sum at 2^-23 a step, 2^-21 a product), the
    norms and softmaxes multiply an error by at most 4 here, so that a gradient is
    off by less than 10 * 4 * 2^-16 < 2^-10 of its largest entry."""
    s = model_state(cuda, seed)
    logits = (fuselse_amd.layer_norm(fuselse_amd.embedding(s["ids"], s["table"], scale=8.0), s["w1"], s["b1"])
              @ s["router"]).detach().sort(-1, descending=True).values
    assert float((logits[:, 1] - logits[:, 2]).min()) > 1e-4  # the choice of experts is not in doubt
    loss, grads = model_step(s)
    want, exact = model_exact(s)
    within(loss, want, 2.0 ** -14 * want.abs().detach(), "loss")
    for name, g, e in zip(LEAVES, grads, exact):
        within(g, e, torch.full_like(e, 2.0 ** -10 * float(e.abs().max())), name)
    # and the same bits again
    again = model_step(s)
    assert torch.equal(loss, again[0]) and same(list(grads), list(again[1]))


def test_gradients_against_differences(cuda):
    """Central differences of each layer's output along a direction, in fp32: the
    step 2^-6 leaves a third-order term of at most 2^-12 of the directions' size
    and a rounding of 2^-23 * 2^6 of the output's."""
    n, d = 12, 48
    w, b = randn(cuda, d, seed=1), randn(cuda, d, seed=2)
    order = fuselse_amd.expert_order(randint(cuda, 4, n, 2, seed=3), 4)
    gates, made, ids = torch.rand(n, 2, device=cuda), randn(cuda, 2 * n, d, seed=4), randint(cuda, 9, n, seed=5)
    cases = {
        "embedding": (lambda t: fuselse_amd.embedding(ids, t, scale=3.0), randn(cuda, 9, d, seed=6)),
        "norm x": (lambda t: fuselse_amd.layer_norm(t, w, b), randn(cuda, n, d, seed=7)),
        "norm w": (lambda t: fuselse_amd.layer_norm(made, t, b), w.clone()),
        "norm b": (lambda t: fuselse_amd.layer_norm(made, w, t), b.clone()),
        "dispatch": (lambda t: fuselse_amd.expert_dispatch(t, order), randn(cuda, n, d, seed=8)),
        "combine rows": (lambda t: fuselse_amd.expert_combine(t, gates, order), made.clone()),
        "combine weights": (lambda t: fuselse_amd.expert_combine(made, t, order), gates.clone()),
    }
    step = 2.0 ** -6
    for name, (f, at) in cases.items():
        at = at.detach().requires_grad_(True)
        y = f(at)
        up, way = randn(cuda, *y.shape, seed=9), randn(cuda, *at.shape, seed=10)
        (g,) = torch.autograd.grad(y, at, up)
        with torch.no_grad():
            change = ((f(at + step * way) - f(at - step * way)).double() * up.double()).sum() / (2 * step)
        size = (y.detach().abs().double() * up.abs().double()).sum() * E23 / step
        size = size + 2.0 ** -9 * (g.abs().double() * way.abs().double()).sum()
        assert abs(float(change - (g.double() * way.double()).sum())) <= float(size), name


def test_tensors_that_are_negated_lazily(cuda):
    """A view whose memory holds the negated values (the imaginary part of a
    conjugate) is taken for what it stands for."""
    d = 24
    view = torch.complex(randn(cuda, 6, d), randn(cuda, 6, d, seed=1)).conj().imag
    assert view.is_neg()
    x = view.clone()
    order = fuselse_amd.expert_order(randint(cuda, 3, 6, 2), 3)
    w = torch.rand(6, 2, device=cuda)
    ids = randint(cuda, 6, 5)
    assert torch.equal(fuselse_amd.layer_norm(view), fuselse_amd.layer_norm(x))
    assert torch.equal(fuselse_amd.embedding(ids, view), fuselse_amd.embedding(ids, x))
    assert torch.equal(fuselse_amd.expert_dispatch(view, order), fuselse_amd.expert_dispatch(x, order))
    rows = torch.cat([x, x]).requires_grad_(True)
    y = fuselse_amd.expert_combine(rows, w, order)
    assert torch.equal(torch.autograd.grad(y, rows, view, retain_graph=True)[0], torch.autograd.grad(y, rows, x)[0])
