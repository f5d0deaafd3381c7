"""Expert products in which every CTA or pair walks over several tiles of different experts, with several
blocks of the summed axis each, against 64 bits on every row."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def spread(scales, size, dim):
    return scales.double().repeat_interleave(128, dim).narrow(dim, 0, size)


def uneven(E, most, seed):
    """Loads with runs of more than four empty experts, some of one row, some of whole tiles."""
    rng = np.random.RandomState(seed)
    loads = rng.randint(1, most + 1, E)
    loads[rng.rand(E) < 0.15] = 0
    loads[5:12] = 0
    loads[E - 6:] = 0
    loads[0], loads[13], loads[14] = 1, min(256, most), 128
    loads[20:26] = 0
    return loads


# (experts, largest load): single CTAs take up to 192 rows per expert on average, or in a padded slot;
# pairs take more
@pytest.mark.parametrize("E,most", [(128, 180), (128, 250), (60, 1100)])
@pytest.mark.parametrize("N,K", [(2000, 144), (2000, 400), (2064, 272), (1168, 1040)])
@pytest.mark.parametrize("padded", [False, True])
def test_products_of_many_tiles(E, most, N, K, padded):
    from brainstorm_b200._C import expert as X

    loads = uneven(E, most, N + K)
    slot = int(loads.max()) + 5 if padded else 0
    L = slot * E if padded else int(loads.sum()) + 77
    gen = torch.Generator(device="cuda").manual_seed(N * K + E)

    def codes(*shape):
        x = torch.randn(*shape, device="cuda", generator=gen) * 60
        return x.clamp(-448, 448).to(torch.float8_e4m3fn)

    rows, weights = codes(L, K), codes(E, N, K)
    rs = torch.rand(-(-K // 128), L, device="cuda", generator=gen).t() + 0.1
    ws = torch.rand(E, -(-N // 128), -(-K // 128), device="cuda", generator=gen) - 0.3
    counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
    starts = [e * slot for e in range(E)] if padded else \
        list(np.cumsum(np.concatenate([[0], loads]))[:-1])
    used = torch.zeros(L, dtype=torch.bool, device="cuda")
    want = torch.zeros(L, N, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for e in range(E):
        at = slice(int(starts[e]), int(starts[e] + loads[e]))
        used[at] = True
        x = rows[at].double() * spread(rs[at], K, 1)
        w = weights[e].double() * spread(spread(ws[e], K, 1), N, 0)
        want[at], size[at] = x @ w.t(), x.abs() @ w.abs().t()
    # up to 128 additions in tensor memory and one per block in fp32, each off by at most 2^-23; two
    # roundings of the scale; one to bf16
    tol = (128 + 2 * rs.size(1) + 2) * 2.0 ** -23 * size + 1e-30
    for relu in (False, True):
        exact = want.clamp(min=0) if relu else want
        out = torch.full((L, N), 7.0, dtype=torch.bfloat16, device="cuda")
        X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot, relu, out)
        X.check_status()
        off = (out.double() - exact).abs()[used]
        assert bool((off <= tol[used] + 2.0 ** -8 * exact.abs()[used]).all())
        assert bool((out[~used] == 7).all())
        filled = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot, relu,
                                             zero_unused=True)
        assert torch.equal(filled[used], out[used]) and bool((filled[~used] == 0).all())
    # the same products once more: nothing depends on the order in which CTAs run
    again = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot, True)
    assert torch.equal(again[used], out[used])


# features: an odd number of blocks up to 5 goes to single CTAs, other numbers to pairs; more than 256
# experts are taken in the order they come
@pytest.mark.parametrize("E,most,N,K", [(60, 1500, 368, 1040), (60, 700, 640, 528), (40, 2300, 400, 1040),
                                        (60, 500, 1040, 784), (300, 150, 144, 272),
                                        (300, 90, 336, 528)])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weight_gradients_of_many_tiles(E, most, N, K, padded, dtype):
    from brainstorm_b200._C import expert as X

    loads = uneven(E, most, N + K)
    slot = int(loads.max()) + 3 if padded else 0
    L = slot * E if padded else int(loads.sum()) + 70
    gen = torch.Generator(device="cuda").manual_seed(N * K + E)
    rows = torch.randn(L, K, device="cuda", generator=gen).bfloat16()
    grads = torch.randn(L, N, device="cuda", generator=gen).bfloat16()
    starts = [e * slot for e in range(E)] if padded else \
        list(np.cumsum(np.concatenate([[0], loads]))[:-1])
    used = torch.zeros(L, dtype=torch.bool, device="cuda")
    for e in range(E):
        used[int(starts[e]):int(starts[e] + loads[e])] = True
    rows[~used] = float("nan")  # not looked at
    grads[~used] = float("inf")
    counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
    got = X.grouped_expert_weight_grad(grads, rows, counts, padded, slot, dtype)
    X.check_status()
    half = torch.finfo(dtype).eps / 2
    for e in range(E):
        at = slice(int(starts[e]), int(starts[e] + loads[e]))
        g, x = grads[at].double(), rows[at].double()
        want, size = g.t() @ x, g.abs().t() @ x.abs()
        tol = (int(loads[e]) + 1) * 2.0 ** -23 * size + half * want.abs() + 1e-30
        assert bool(((got[e].double() - want).abs() <= tol).all()), (e, loads[e])
    again = X.grouped_expert_weight_grad(grads, rows, counts, padded, slot, dtype)
    assert torch.equal(again, got)


def test_layer_of_all_operators_within_twice_the_codes_error():
    """A feed-forward layer of experts against 64 bits, the tolerance twice the error that is expected of
    the codes.  A code's error is uniform within a step of 2^-3 of the power of two below its value:
    0.0255 rms of the value, so a product of two coded operands is off by e = 0.036 of its norm.
    ReLU passes the gradient where the coded product is positive: a share e / pi of all signs differ,
    which is 2 e / pi of what passes, 0.15 in the norm."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    torch.manual_seed(5)
    T, k, E, d, hidden = 900, 2, 6, 384, 640
    cells = torch.randn(T, d, device="cuda").bfloat16().requires_grad_()
    up = (torch.randn(E, hidden, d, device="cuda") / 20).bfloat16().requires_grad_()
    down = (torch.randn(E, d, hidden, device="cuda") / 25).bfloat16().requires_grad_()
    score = torch.randn(T, E, device="cuda", requires_grad=True)
    leaves = (cells, up, down, score)
    gy = torch.randn(T, d, device="cuda")

    top, picks = torch.topk(score, k, dim=1)
    places, loads = R.order_picks(picks, E)
    mid = torch.relu(X.expert_linear_fp8(R.sort_cells(cells, places), up, loads))
    got = R.unsort_cells(X.expert_linear_fp8(mid, down, loads), places, torch.softmax(top, 1))
    got_grads = torch.autograd.grad(got, leaves, gy.bfloat16())
    X.check_status()

    gates = torch.softmax(torch.topk(score.double(), k, dim=1).values, 1)
    want = torch.zeros(T, d, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, j = torch.nonzero(picks == e, as_tuple=True)
        y = torch.relu(cells.double()[t] @ up[e].double().t()) @ down[e].double().t()
        want = want.index_add(0, t, y * gates[t, j].unsqueeze(1))
    want_grads = torch.autograd.grad(want, leaves, gy.double())

    e, signs = 0.036, 0.15
    expected = {
        "out": 2 ** 0.5 * e,                           # two products
        "cells": (2 * e ** 2 + signs ** 2) ** 0.5,     # two products and the signs between them
        "up": (e ** 2 + signs ** 2) ** 0.5,
        "down": e,                                     # of the rows that go in
        "score": 2 ** 0.5 * e,
    }
    for name, a, b in zip(expected, (got,) + got_grads, (want,) + want_grads):
        a, b = a.detach().double(), b.detach().double()
        off = float((a - b).norm() / b.norm())
        assert off < 2 * expected[name], (name, off, expected[name])


@pytest.mark.parametrize("padded", [False, True])
def test_loads_beyond_the_buffer_and_below_zero_are_cut(padded):
    """Loads are on the device and not checked: no row outside the buffer, or outside its slot, is read or
    written."""
    from brainstorm_b200._C import expert as X

    E, N, K = 4, 144, 272
    slot = 70 if padded else 0
    L = slot * E if padded else 300
    given = [40, -3, 2 ** 31 - 1, 2 ** 31 - 1]
    real = [40, 0, 70, 70] if padded else [40, 0, 260, 0]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(L, K, device="cuda", generator=gen).bfloat16()
    g = torch.randn(L, N, device="cuda", generator=gen).bfloat16()
    rows, rs = X.quantize_rows(x)
    w, ws = X.quantize_expert_weights(torch.randn(E, N, K, device="cuda", generator=gen))
    counts, cut = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in (given, real))
    for zero in (False, True):
        outs = []
        for loads in (counts, cut):
            out = torch.full((L, N), 7.0, dtype=torch.bfloat16, device="cuda")
            outs.append(X.grouped_expert_linear_fp8(rows, rs, w, ws, loads, padded, slot, out=out,
                                                    zero_unused=zero))
        assert torch.equal(*outs)
    assert torch.equal(X.grouped_expert_weight_grad(g, x, counts, padded, slot),
                       X.grouped_expert_weight_grad(g, x, cut, padded, slot))
    X.check_status()


@pytest.mark.parametrize("padded", [False, True])
def test_no_expert_has_a_row(padded):
    from brainstorm_b200._C import expert as X

    E, N, K, L = 5, 272, 144, 500
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(L, K, device="cuda", generator=gen).bfloat16()
    loads = torch.zeros(E, dtype=torch.int32, device="cuda")
    w = torch.randn(E, N, K, device="cuda", generator=gen).requires_grad_()
    x.requires_grad_()
    out = X.expert_linear_fp8(x, w, loads, padded)
    grads = torch.autograd.grad(out, (x, w), torch.full_like(out, float("nan")))
    X.check_status()
    assert bool((out == 0).all()) and all(bool((t == 0).all()) for t in grads)
