"""Rows sorted by path from compact picks and back, with their gradients, against plain numpy and
64-bit torch formulas."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def order_by_hand(picks, paths):
    flat = picks.reshape(-1)
    key = np.where((flat >= 0) & (flat < paths), flat, paths)
    order = np.argsort(key, kind="stable")
    places = np.empty(flat.size, dtype=np.int64)
    places[order] = np.arange(flat.size)
    places = np.where(key < paths, places, -2 - places)
    return places.reshape(picks.shape), np.bincount(key, minlength=paths + 1)[:paths]


def make_picks(T, k, E, kind, seed=0):
    rng = np.random.RandomState(seed)
    if kind == "one path":
        picks = np.full((T, k), E - 1)
    elif kind == "skewed":
        picks = np.minimum((rng.exponential(E / 8 + 0.3, (T, k))).astype(np.int64), E - 1)
    else:
        picks = rng.randint(0, E, (T, k))
    if kind == "dropped":
        picks[rng.rand(T, k) < 0.4] = -1
        picks[rng.rand(T, k) < 0.1] = E + 5
        picks[T // 2] = -7  # a cell that goes nowhere
    if kind == "all dropped":
        picks[:] = -1
    return picks


@pytest.mark.parametrize("kind", ["plain", "skewed", "one path", "dropped", "all dropped"])
@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 8, 64), (31, 3, 7), (33, 1, 1024), (1000, 4, 30),
                                   (1024, 8, 256), (1025, 8, 256), (5000, 2, 1), (40001, 3, 130),
                                   (70000, 8, 1024)])
@pytest.mark.parametrize("wide", [False, True])
def test_order_picks(T, k, E, kind, wide):
    from brainstorm_b200._C import router as R

    picks = make_picks(T, k, E, kind)
    places, loads = R.order_picks(
        torch.tensor(picks, dtype=torch.int64 if wide else torch.int32, device="cuda"), E)
    want_places, want_loads = order_by_hand(picks, E)
    assert places.dtype == loads.dtype == torch.int32
    assert np.array_equal(places.cpu().numpy(), want_places)
    assert np.array_equal(loads.cpu().numpy(), want_loads)


def test_order_picks_of_no_cells_and_of_strided_picks():
    from brainstorm_b200._C import router as R

    places, loads = R.order_picks(torch.empty((0, 2), dtype=torch.int64, device="cuda"), 5)
    assert places.shape == (0, 2) and loads.tolist() == [0] * 5
    picks = torch.tensor(make_picks(300, 8, 12, "plain"), device="cuda")
    part = picks[::2, 1:4]
    places, loads = R.order_picks(part, 12)
    want_places, want_loads = order_by_hand(part.cpu().numpy(), 12)
    assert np.array_equal(places.cpu().numpy(), want_places)
    # far beyond 32 bits, and just past both ends
    odd = torch.tensor([[2 ** 32 + 1, -2 ** 40], [12, 3]], device="cuda")
    places, loads = R.order_picks(odd, 12)
    assert places.tolist() == [[-3, -4], [-5, 0]] and int(loads.sum()) == 1 and int(loads[3]) == 1


def routes(T, k, E, kind, seed=1):
    """places on the device, and (cell, pick, row) of the picks that go somewhere."""
    places, _ = order_by_hand(make_picks(T, k, E, kind, seed), E)
    t, j = np.nonzero(places >= 0)
    return (torch.tensor(places, dtype=torch.int32, device="cuda"),
            torch.tensor(t, device="cuda"), torch.tensor(j, device="cuda"),
            torch.tensor(places[t, j], device="cuda"))


SHAPES = [(1, 1, 3, (1,)), (1, 8, 64, (2048,)), (5, 2, 4, (7,)), (129, 3, 30, (501,)),
          (64, 8, 16, (4, 33)), (300, 2, 5, (1024,)), (17, 4, 9, (5000,)), (40, 1, 6, (16,))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["plain", "dropped", "all dropped"])
@pytest.mark.parametrize("T,k,E,cell", SHAPES)
def test_sort_cells_and_gradient(T, k, E, cell, kind, dtype):
    from brainstorm_b200._C import router as R

    places, t, j, row = routes(T, k, E, kind)
    x = torch.randn(T, *cell, device="cuda").to(dtype).requires_grad_()
    rows = R.sort_cells(x, places)
    want = torch.zeros(T * k, *cell, dtype=dtype, device="cuda")
    want[row] = x.detach()[t]
    assert torch.equal(rows.detach(), want)
    gy = torch.randn(T * k, *cell, device="cuda").to(dtype)
    (gx,) = torch.autograd.grad(rows, x, gy)
    exact = torch.zeros(T, *cell, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(exact)
    exact.index_add_(0, t, gy.double()[row])
    size.index_add_(0, t, gy.double()[row].abs())
    # k fp32 additions, and one rounding to the type
    tol = k * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * exact.abs() + 1e-30
    if dtype == torch.float16:
        tol += 2.0 ** -25  # half a step among its smallest numbers
    assert bool(((gx.double() - exact).abs() <= tol * (1 + 1e-6)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate_type", ["none", "f32", "same"])
@pytest.mark.parametrize("kind", ["plain", "dropped", "all dropped"])
@pytest.mark.parametrize("T,k,E,cell", SHAPES)
def test_unsort_cells_and_gradients(T, k, E, cell, kind, dtype, gate_type):
    from brainstorm_b200._C import router as R

    places, t, j, row = routes(T, k, E, kind)
    rows = torch.randn(T * k, *cell, device="cuda").to(dtype).requires_grad_()
    gates = None
    weight = torch.ones(t.numel(), dtype=torch.float64, device="cuda")
    if gate_type != "none":
        gates = torch.rand(T, k, device="cuda").to(
            torch.float32 if gate_type == "f32" else dtype)
        gates[places < 0] = float("nan")  # not looked at
        weight = gates[t, j].double()
        gates.requires_grad_()
    ones = (1,) * len(cell)
    out = R.unsort_cells(rows, places, gates)
    terms = rows.detach().double()[row] * weight.view(-1, *ones)
    exact = torch.zeros(T, *cell, dtype=torch.float64, device="cuda").index_add_(0, t, terms)
    size = torch.zeros_like(exact).index_add_(0, t, terms.abs())
    half = torch.finfo(dtype).eps / 2
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    tol = k * 2.0 ** -24 * size + half * exact.abs() + least
    assert out.dtype == dtype
    assert bool(((out.detach().double() - exact).abs() <= tol * (1 + 1e-6)).all())

    gy = torch.randn(T, *cell, device="cuda").to(dtype)
    grads = torch.autograd.grad(out, [rows] + ([gates] if gates is not None else []), gy)
    want = torch.zeros(T * k, *cell, dtype=torch.float64, device="cuda")
    want[row] = gy.double()[t] * weight.view(-1, *ones)
    tol = (2.0 ** -24 + half) * want.abs() + least
    assert bool(((grads[0].double() - want).abs() <= tol * (1 + 1e-6)).all())
    if gates is not None:
        dots = (gy.double()[t] * rows.detach().double()[row]).flatten(1)
        want = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        want[t, j] = dots.sum(1)
        size = torch.zeros_like(want)
        size[t, j] = dots.abs().sum(1)
        gate_half = torch.finfo(gates.dtype).eps / 2
        tol = (dots.size(1) + 5) * 2.0 ** -24 * size + gate_half * want.abs() + least
        assert grads[1].dtype == gates.dtype
        assert bool(((grads[1].double() - want).abs() <= tol * (1 + 1e-6)).all())


def test_gradients_agree_with_differences():
    from brainstorm_b200._C import router as R

    torch.manual_seed(3)
    picks = torch.tensor([[0, 2], [2, -1], [1, 1], [0, 1]], device="cuda")
    places, _ = R.order_picks(picks, 3)
    x = torch.randn(4, 6, device="cuda", requires_grad=True)
    gates = torch.rand(4, 2, device="cuda", requires_grad=True)
    mix = torch.randn(8, 6, device="cuda")
    probe = torch.randn(4, 6, device="cuda")

    def f(x, gates):
        return (R.unsort_cells(R.sort_cells(x, places) * mix, places, gates) * probe).sum()

    gx, gg = torch.autograd.grad(f(x, gates), (x, gates))
    step = 2.0 ** -6  # f is linear in x and in the gates: a difference is exact but for rounding
    for leaf, grad in ((x, gx), (gates, gg)):
        for i in range(leaf.numel()):
            moved = leaf.detach().clone().view(-1)
            moved[i] += step
            moved = moved.view(leaf.shape)
            other = f(moved, gates) if leaf is x else f(x, moved)
            slope = float((other - f(x, gates)).detach()) / step
            # sums of about 50 terms below 20 in fp32, twice, over the step
            assert abs(slope - float(grad.view(-1)[i])) < 2 * 50 * 20 * 2.0 ** -24 / step


def test_places_set_to_minus_one_and_outside_the_buffer_are_skipped():
    from brainstorm_b200._C import router as R

    x = torch.arange(8, dtype=torch.float32, device="cuda").view(4, 2) + 1
    places, _ = R.order_picks(torch.tensor([[0, 1], [1, 0], [0, 1], [1, 0]], device="cuda"), 2)
    places[1, 0] = -1
    places[2, 1] = 8
    places[3, 0] = -2 - 8
    gates = torch.full((4, 2), 2.0, device="cuda")
    rows = torch.randn(8, 2, device="cuda")
    want = torch.zeros(4, 2, device="cuda")
    for t in range(4):
        for j in range(2):
            if 0 <= int(places[t, j]) < 8:
                want[t] += 2 * rows[int(places[t, j])]
    assert torch.allclose(R.unsort_cells(rows, places, gates), want, rtol=1e-6, atol=1e-6)
    got = R.sort_cells(x, places)
    for t in range(4):
        for j in range(2):
            if 0 <= int(places[t, j]) < 8:
                assert torch.equal(got[int(places[t, j])], x[t])


def test_infinities_in_unrouted_rows_stay_there():
    from brainstorm_b200._C import router as R

    picks = torch.tensor([[0, -1], [-1, -1], [1, 0]], device="cuda")
    places, loads = R.order_picks(picks, 2)
    rows = torch.randn(6, 40, device="cuda")
    rows[int(loads.sum()):] = float("inf")
    gates = torch.rand(3, 2, device="cuda").requires_grad_()
    rows.requires_grad_()
    out = R.unsort_cells(rows, places, gates)
    assert bool(torch.isfinite(out).all()) and bool((out[1] == 0).all())
    gr, gg = torch.autograd.grad(out.sum(), (rows, gates))
    assert bool(torch.isfinite(gr).all()) and bool(torch.isfinite(gg).all())
    assert bool((gr[int(loads.sum()):] == 0).all())
    x = torch.randn(3, 40, device="cuda")
    x[1] = float("nan")  # goes nowhere
    assert bool(torch.isfinite(R.sort_cells(x, places)).all())


def test_layouts_streams_and_slices():
    from brainstorm_b200._C import router as R

    places, t, j, row = routes(200, 2, 8, "plain")
    base = torch.randn(200, 100, device="cuda")
    for x in (base[:, 3:71], base.t().contiguous().t(), base.flatten()[1:13601].view(200, 68)):
        want = torch.zeros(400, x.size(1), device="cuda")
        want[row] = x[t]
        assert torch.equal(R.sort_cells(x, places), want)
    side = torch.cuda.Stream()
    x = torch.randn(200, 2048, device="cuda").bfloat16()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        rows = R.sort_cells(x, places)
        back = R.unsort_cells(rows, places)
    side.synchronize()
    assert torch.equal(back, (x.float() * 2).bfloat16())


def test_captured_routes_replay_with_new_picks_beside_another_graph():
    from brainstorm_b200._C import router as R

    T, k, E = 6000, 4, 40
    made = []
    for seed in (5, 6):
        picks = torch.tensor(make_picks(T, k, E, "dropped", seed), device="cuda")
        x = torch.randn(T, 64, device="cuda")
        graph = torch.cuda.CUDAGraph()
        R.order_picks(picks, E)  # loads the kernels
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            places, loads = R.order_picks(picks, E)
            rows = R.sort_cells(x, places)
        made.append((graph, picks, x, places, loads, rows))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    fresh = [make_picks(T, k, E, "skewed", seed) for seed in (7, 8)]
    for (graph, picks, *_), new in zip(made, fresh):
        picks.copy_(torch.tensor(new))
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (graph, *_) in zip(streams, made):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, picks, x, places, loads, rows), new in zip(made, fresh):
        want, want_loads = order_by_hand(new, E)
        assert np.array_equal(places.cpu().numpy(), want)
        assert np.array_equal(loads.cpu().numpy(), want_loads)
        assert torch.equal(rows[places.long().flatten()], x.repeat_interleave(k, 0))


def test_captured_training_pass():
    from brainstorm_b200._C import router as R

    T, k, E, d = 500, 2, 8, 256
    picks = torch.tensor(make_picks(T, k, E, "dropped"), device="cuda")
    x = torch.randn(T, d, device="cuda").bfloat16()
    gates = torch.rand(T, k, device="cuda")
    gy = torch.randn(T, d, device="cuda").bfloat16()

    def step():
        a, g = x.detach().requires_grad_(), gates.detach().requires_grad_()
        places, _ = R.order_picks(picks, E)
        out = R.unsort_cells(R.sort_cells(a, places), places, g)
        return (out.detach(),) + torch.autograd.grad(out, (a, g), gy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    picks.copy_(torch.tensor(make_picks(T, k, E, "plain", 9)))
    x.copy_(torch.randn(T, d, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


@pytest.fixture(params=["native", "python"])
def host_side(request, monkeypatch):
    """The operators with their native host side, and with the Python that takes what it declines."""
    from brainstorm_b200 import _lib

    if request.param == "python":
        monkeypatch.setattr(_lib, "_host", _lib._DeclinesAll())
    return request.param


@pytest.mark.parametrize("gate_type", [None, torch.float32, torch.bfloat16])
def test_both_host_sides(host_side, gate_type):
    from brainstorm_b200._C import router as R

    torch.manual_seed(4)
    T, k, E, d = 90, 3, 11, 160
    picks = torch.tensor(make_picks(T, k, E, "dropped"), device="cuda")
    places, loads = R.order_picks(picks, E)
    want, want_loads = order_by_hand(picks.cpu().numpy(), E)
    assert np.array_equal(places.cpu().numpy(), want)
    assert np.array_equal(loads.cpu().numpy(), want_loads)
    x = torch.randn(T, d, device="cuda").bfloat16().requires_grad_()
    gates = None if gate_type is None else \
        torch.rand(T, k, device="cuda").to(gate_type).requires_grad_()
    rows = R.sort_cells(x, places)
    out = R.unsort_cells(rows, places, gates)
    gy = torch.randn(T, d, device="cuda").bfloat16()
    leaves = [x] if gates is None else [x, gates]
    grads = torch.autograd.grad(out, leaves, gy)
    live = (places >= 0).float()
    weight = live if gates is None else live * gates.detach().float()
    # sums of up to 3 products of bf16 values: the products are exact in fp32 but for fp32 gates
    # (2^-24), the sums are off by 2^-23 of their terms, and each result is rounded to bf16: twice
    # on the way back
    size = weight.sum(1, keepdim=True)
    plain = x.detach().float() * size
    assert bool(((out.detach().float() - plain).abs() <= 2.0 ** -8 * plain.abs() * 1.01).all())
    plain = gy.float() * size
    tol = 2.0 ** -8 * 2.01 * (gy.float().abs() * size) + 1e-30
    assert bool(((grads[0].float() - plain).abs() <= tol).all())
    if gates is not None:
        dots = (gy.double() * x.detach().double()).sum(1, keepdim=True) * live
        size = (gy.double() * x.detach().double()).abs().sum(1, keepdim=True)
        half = torch.finfo(gate_type).eps / 2
        assert bool(((grads[1].double() - dots).abs()
                     <= (d + 5) * 2.0 ** -24 * size + half * dots.abs() * 1.01).all())
    codes, scales = R.sort_cells_fp8(x.detach(), places)
    assert codes.shape == (T * k, d) and scales.stride() == (1, T * k)
    # a gradient that comes expanded, and one of the leaves alone
    (g,) = torch.autograd.grad(R.sort_cells(x, places).sum(), (x,))
    assert torch.equal(g.float(), live.sum(1, keepdim=True).expand(T, d))
    if gates is not None:
        out = R.unsort_cells(rows.detach(), places, gates)
        (g,) = torch.autograd.grad(out, (gates,), gy)
        assert torch.equal(g, grads[1])


def test_second_gradients_are_refused(host_side):
    from brainstorm_b200._C import router as R

    places, _ = R.order_picks(torch.tensor([[0, 1], [1, 0]], device="cuda"), 2)
    x = torch.randn(2, 16, device="cuda", requires_grad=True)
    gates = torch.rand(2, 2, device="cuda", requires_grad=True)
    out = R.unsort_cells(R.sort_cells(x, places), places, gates)
    gx, gg = torch.autograd.grad(out.square().sum(), (x, gates), create_graph=True)
    assert bool(torch.isfinite(gx).all()) and bool(torch.isfinite(gg).all())
    with pytest.raises(RuntimeError, match="differentia"):
        torch.autograd.grad(gg.sum(), x)


def test_an_edited_input_is_noticed_by_the_backward_pass(host_side):
    from brainstorm_b200._C import router as R

    places, _ = R.order_picks(torch.tensor([[0, 1], [1, 0]], device="cuda"), 2)
    rows = torch.randn(4, 16, device="cuda")
    gates = torch.rand(2, 2, device="cuda", requires_grad=True)
    out = R.unsort_cells(rows, places, gates)
    rows.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """The leaves' accumulators belong to the eager graph's stream; autograd would tie that stream to
    the captured one.  The operator says so before, and both go on to work."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    picks = torch.randint(0, 4, (64, 2), device="cuda")
    places, loads = R.order_picks(picks, 4)
    x = torch.randn(64, 32, device="cuda").bfloat16().requires_grad_()
    gates = torch.rand(64, 2, device="cuda").requires_grad_()
    w = (torch.randn(4, 48, 32, device="cuda") / 8).requires_grad_()

    def layer():
        y = X.expert_linear_fp8(R.sort_cells(x, places), w, loads)
        return R.unsort_cells(y, places, gates)

    steps = {
        "sort": (lambda: R.sort_cells(x, places), (x,)),
        "unsort": (lambda: R.unsort_cells(torch.ones(128, 32, device="cuda"), places, gates),
                   (gates,)),
        "layer": (layer, (w,)),
    }
    for name, (step, leaves) in steps.items():
        alive = step()  # an eager graph that lives on
        torch.autograd.grad(alive.float().sum(), leaves, retain_graph=True)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="being captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                out = step()
                torch.autograd.grad(out, leaves, torch.ones_like(out))
        torch.cuda.synchronize()
        (want,) = torch.autograd.grad(alive.float().sum(), leaves)
        del alive, out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
            (got,) = torch.autograd.grad(out, leaves, torch.ones_like(out))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), name
