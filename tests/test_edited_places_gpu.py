"""Places that were edited after ``order_picks``: the rows that nothing names any more are zeros, in
the operators' results and in their gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def host_side(request, monkeypatch):
    from brainstorm_b200 import _lib

    if request.param == "python":
        monkeypatch.setattr(_lib, "_host", _lib._DeclinesAll())
    return request.param


def foul(*sizes):
    """Leaves NaN in the memory that the next allocations of these numbers of bytes get."""
    held = [torch.full((n,), 0xff, dtype=torch.uint8, device="cuda") for n in sizes for _ in "12"]
    del held


def edited(T, k, E, how, seed=0):
    """(places, loads, live [T, k], rows that are still named by a live place)"""
    from brainstorm_b200._C import router as R

    gen = torch.Generator().manual_seed(seed)
    picks = torch.randint(-1, E, (T, k), generator=gen).cuda()
    places, loads = R.order_picks(picks, E)
    cut = (torch.rand(T, k, generator=gen) < {"few": 0.02, "most": 0.9, "all": 2.0, "none": -1.0,
                                              "outside": 0.3, "twice": 0.1}[how]).cuda()
    if how == "outside":
        places[cut] = T * k + 3
        places[0, 0] = -2 - T * k
    elif how == "twice":
        places[cut] = places[0, 0].clone()
    else:
        places[cut] = -1
    live = (places >= 0) & (places < T * k)
    return places, loads, live


# few cells; whole cells; rows of 4- and 2-byte accesses; as many rows as one CTA searches and one more;
# narrow rows, many of them; cells of many picks
SHAPES = [(1, 1, 3, 16), (5, 3, 4, 48), (300, 8, 16, 2048), (3000, 2, 30, 501), (6000, 3, 40, 640),
          (8192, 1, 5, 33), (2731, 3, 5, 80), (30000, 4, 64, 17), (50000, 2, 7, 144),
          (9, 1700, 5, 272)]


@pytest.mark.parametrize("how", ["few", "most", "all", "none", "outside"])
@pytest.mark.parametrize("T,k,E,d", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_no_place_names_are_zeros(host_side, T, k, E, d, how, dtype):
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    places, _, live = edited(T, k, E, how)
    t, j = torch.nonzero(live, as_tuple=True)
    row = places[t, j].long()
    x = torch.randn(T, d, device="cuda").to(dtype)
    want = torch.zeros(T * k, d, dtype=dtype, device="cuda")
    want[row] = x[t]
    foul(want.numel() * want.element_size())
    assert torch.equal(R.sort_cells(x, places), want)
    if d % 16 == 0:
        codes, scales = X.quantize_rows(want)
        foul(codes.numel(), scales.numel() * 4)
        got_codes, got_scales = R.sort_cells_fp8(x, places)
        assert torch.equal(got_codes.float(), codes.float()) and torch.equal(got_scales, scales)

    gates = torch.rand(T, k, device="cuda")
    for g in (gates, None):
        rows = torch.randn(T * k, d, device="cuda").to(dtype).requires_grad_()
        leaves = [rows] if g is None else [rows, g.requires_grad_()]
        out = R.unsort_cells(rows, places, g)
        gy = torch.randn(T, d, device="cuda").to(dtype)
        foul(want.numel() * want.element_size())
        grads = torch.autograd.grad(out, leaves, gy)
        want = torch.zeros(T * k, d, dtype=dtype, device="cuda")
        want[row] = gy[t] if g is None else (g.detach()[t, j].unsqueeze(1) * gy[t].float()).to(dtype)
        assert torch.equal(grads[0], want)
        if g is not None:
            assert bool((grads[1][~live] == 0).all()) and bool(torch.isfinite(grads[1]).all())


def test_a_row_named_twice_leaves_no_row_unwritten(host_side):
    """Which of the two cells such a row gets is open; every other row is as it should be."""
    from brainstorm_b200._C import router as R

    T, k, E, d = 700, 2, 9, 96
    places, _, live = edited(T, k, E, "twice")
    t, j = torch.nonzero(live, as_tuple=True)
    row = places[t, j].long()
    x = torch.randn(T, d, device="cuda")
    named = torch.bincount(row, minlength=T * k)
    foul(T * k * d * 4)
    got = R.sort_cells(x, places)
    assert bool((got[named == 0] == 0).all())
    once = named[row] == 1
    assert torch.equal(got[row[once]], x[t[once]])


def test_dropped_rows_add_nothing_to_the_weights_gradient(host_side):
    """A pick that is taken out of the places after it was counted in the loads: its row is still one
    of its expert's, with a gradient of zero."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    T, k, E, d, n = 500, 2, 6, 128, 64
    places, loads, live = edited(T, k, E, "few")
    x = torch.randn(T, d, device="cuda").bfloat16()
    rows = R.sort_cells(x, places)
    out = torch.randn(T * k, n, device="cuda").bfloat16().requires_grad_()
    gates = torch.rand(T, k, device="cuda", requires_grad=True)
    back = R.unsort_cells(out, places, gates)
    gy = torch.randn(T, n, device="cuda").bfloat16()
    foul(T * k * n * 2)
    (gr, _) = torch.autograd.grad(back, (out, gates), gy)
    got = X.grouped_expert_weight_grad(gr, rows, loads, dtype=torch.float32)
    first = 0
    t, j = torch.nonzero(live, as_tuple=True)
    row = places[t, j].long()
    for e, load in enumerate(loads.tolist()):
        mine = (row >= first) & (row < first + load)
        a = (gates.detach()[t, j][mine].unsqueeze(1) * gy[t][mine].float()).bfloat16().double()
        b = x[t][mine].double()
        want, size = a.t() @ b, a.abs().t() @ b.abs()
        assert bool(((got[e].double() - want).abs() <= (load + 2) * 2.0 ** -23 * size).all())
        first += load


def test_more_rows_than_the_windows_of_one_search():
    from brainstorm_b200._C import router as R

    T, k, E, d = 700_000, 8, 9, 16
    places, _, live = edited(T, k, E, "few")
    x = torch.randn(T, d, device="cuda").bfloat16()
    t, j = torch.nonzero(live, as_tuple=True)
    want = torch.zeros(T * k, d, dtype=x.dtype, device="cuda")
    want[places[t, j].long()] = x[t]
    foul(want.numel() * 2)
    assert torch.equal(R.sort_cells(x, places), want)


@pytest.mark.parametrize("T", [4000, 20000])
def test_rows_named_twice_in_place_of_others_with_the_same_sums(T):
    """0, 3, 5 and 6 have the sum and the squares' sum of 1, 2, 4 and 7."""
    from brainstorm_b200._C import router as R

    k, d = 2, 64
    places, _ = R.order_picks(torch.randint(0, 5, (T, k), device="cuda"), 5)
    flat = places.view(-1)
    for a, b in ((0, 1), (3, 2), (5, 4), (6, 7)):
        flat[flat == a] = b
    x = torch.randn(T, d, device="cuda")
    foul(T * k * d * 4)
    got = R.sort_cells(x, places)
    assert bool((got[[0, 3, 5, 6]] == 0).all()) and bool(torch.isfinite(got).all())


def test_captured_training_pass_over_edited_places():
    """More rows than one CTA searches: the search beside the kernels that move rows, replayed with other
    picks and other edits."""
    from brainstorm_b200._C import router as R

    T, k, E, d = 6000, 3, 12, 96
    gen = torch.Generator(device="cuda").manual_seed(3)

    def fresh():
        return (torch.randint(-1, E, (T, k), device="cuda", generator=gen),
                torch.rand(T, k, device="cuda", generator=gen) < 0.2,
                torch.randn(T, d, device="cuda", generator=gen).bfloat16(),
                torch.rand(T, k, device="cuda", generator=gen),
                torch.randn(T, d, device="cuda", generator=gen).bfloat16())

    held = fresh()

    def step(picks, cut, x, gates, gy):
        x, gates = x.detach().requires_grad_(), gates.detach().requires_grad_()
        places, _ = R.order_picks(picks, E)
        places = torch.where(cut, -1, places)
        rows = R.sort_cells(x, places)
        leaf = rows.detach().requires_grad_()
        out = R.unsort_cells(leaf, places, gates)
        grads = torch.autograd.grad(out, (leaf, gates), gy)
        return (rows.detach(), out.detach()) + grads + torch.autograd.grad(rows, (x,), grads[0])

    step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for _ in range(4):
        for a, b in zip(held, fresh()):
            a.copy_(b)
        for a in got:
            a.view(torch.uint8).fill_(0xff)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(*held)):
            assert torch.equal(a, b) and bool(torch.isfinite(a).all())
