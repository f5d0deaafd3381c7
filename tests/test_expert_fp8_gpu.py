"""8-bit codes with a scale for each block of 128, the grouped expert product over them and the
gradient of the experts' weights, against 64-bit formulas."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FLOOR = 2.0 ** -100


def spread(scales, size, dim):
    return scales.double().repeat_interleave(128, dim).narrow(dim, 0, size)


def check_codes(codes, scales, x, dims):
    """Scales within fp32's rounding of max / 448, codes the nearest e4m3 value of x / scale: half a
    step (2^-4 relative, 2^-10 among the smallest) and fp32's roundings of the quotient."""
    block = torch.nn.functional.pad(x.double().abs(), sum(
        ([0, -n % 128 if d in dims else 0] for d, n in reversed(list(enumerate(x.shape)))), []))
    for d in dims:
        block = block.unflatten(d, (-1, 128)).amax(d + 1)
    amax = block.clamp(min=FLOOR)
    assert scales.shape == amax.shape and scales.dtype == torch.float32
    assert bool(((scales.double() - amax / 448).abs() <= 2.0 ** -24 * amax / 448).all())
    full = scales.double()
    for d in dims:
        full = spread(full, x.size(d), d)
    value, want = codes.double(), x.double() / full
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    tol = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10))
    assert bool(((value - want).abs() <= tol * (1 + 2.0 ** -10)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,width", [(1, 16), (1, 128), (3, 144), (257, 1040), (1000, 2048),
                                     (7, 8208), (0, 64)])
def test_quantize_rows(L, width, dtype):
    from brainstorm_b200._C import expert as X

    x = (torch.randn(L, width, device="cuda") * torch.exp(torch.randn(width, device="cuda")))
    if L > 2:
        x[1] = 0
        x[2] *= 1e-4
    x = x.to(dtype)
    codes, scales = X.quantize_rows(x)
    if L == 0:
        assert codes.shape == (0, width) and scales.shape == (0, 1)
        return
    check_codes(codes, scales, x, (1,))
    if L > 2:
        assert bool((codes[1].float() == 0).all())


def test_quantize_extremes():
    from brainstorm_b200._C import expert as X

    x = torch.randn(6, 256, device="cuda")
    x[0, 5] = float("nan")
    x[1, 130] = float("inf")
    x[2] = 3e38
    x[3] = 1e-44
    x[4, :128] = -448.0
    codes, scales = X.quantize_rows(x)
    assert bool(torch.isnan(codes[0, 5].float())) and int(torch.isnan(codes[0].float()).sum()) == 1
    assert torch.isinf(scales[1, 1]) and bool(torch.isnan(codes[1, 130].float()))
    assert bool((codes[2].float() == 448).all()) and bool(torch.isfinite(scales[2]).all())
    assert bool((codes[3].float() == 0).all()) and bool((scales[3] > 0).all())
    assert bool((codes[4, :128].float() == -448).all()) and float(scales[4, 0]) == 1.0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("E,N,K", [(1, 16, 16), (3, 128, 256), (2, 144, 400), (5, 1040, 272)])
def test_quantize_expert_weights(E, N, K, dtype, transposed):
    from brainstorm_b200._C import expert as X

    w = (torch.randn(E, N, K, device="cuda") * 0.02).to(dtype)
    w[0, 0, 0] = 3.0
    codes, scales = X.quantize_expert_weights(w, transposed)
    check_codes(codes, scales, w.transpose(1, 2) if transposed else w, (1, 2))


@pytest.mark.parametrize("T,k,E,width", [(1, 8, 64, 2048), (33, 2, 5, 144), (300, 4, 16, 1040)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sort_cells_fp8_is_sort_then_quantize(T, k, E, width, dtype):
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    picks = torch.randint(-1, E, (T, k), device="cuda")
    x = torch.randn(T, width, device="cuda").to(dtype)
    places, _ = R.order_picks(picks, E)
    codes, scales = R.sort_cells_fp8(x, places)
    want_codes, want_scales = X.quantize_rows(R.sort_cells(x, places))
    assert torch.equal(codes.float(), want_codes.float()) and torch.equal(scales, want_scales)
    assert scales.stride() == want_scales.stride()


def codes_of(*shape):
    x = torch.randn(*shape, device="cuda") * 60
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def starts(loads, slot):
    if slot:
        return [e * slot for e in range(len(loads))]
    return list(np.cumsum([0] + list(loads))[:-1])


LOADS = {
    "one row": [0, 0, 1, 0],
    "one each": [1] * 7,
    "ragged": [0, 37, 256, 1, 300, 0, 129, 511, 16, 0],
    "one expert": [700],
    "few large": [1025, 90],
}


@pytest.mark.parametrize("kind", list(LOADS))
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("N,K", [(128, 128), (256, 256), (16, 16), (400, 1040), (2000, 144),
                                 (640, 4096)])
def test_grouped_expert_linear_fp8(kind, padded, N, K):
    from brainstorm_b200._C import expert as X

    loads = LOADS[kind]
    E = len(loads)
    slot = max(loads) + 3 if padded else 0
    L = slot * E if padded else sum(loads) + 5
    torch.manual_seed(L + N + K)
    rows, weights = codes_of(L, K), codes_of(E, N, K)
    rs = torch.rand(-(-K // 128), L, device="cuda").t() + 0.1  # any fp32 numbers
    ws = torch.rand(E, -(-N // 128), -(-K // 128), device="cuda") - 0.3
    counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
    for relu in (False, True):
        out = torch.full((L, N), 7.0, dtype=torch.bfloat16, device="cuda")
        got = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot, relu, out)
        X.check_status()
        assert got is out
        used = torch.zeros(L, dtype=torch.bool, device="cuda")
        for e, (first, load) in enumerate(zip(starts(loads, slot), loads)):
            at = slice(first, first + load)
            used[at] = True
            x = rows[at].double() * spread(rs[at], K, 1)
            w = weights[e].double() * spread(spread(ws[e], K, 1), N, 0)
            want, size = x @ w.t(), x.abs() @ w.abs().t()
            if relu:
                want = want.clamp(min=0)
            # up to 128 additions in tensor memory and one per block in fp32, each off by at most
            # 2^-23 (additions in the tensor cores need not round to nearest); two roundings of the
            # scale; one to bf16
            tol = (128 + 2 * rs.size(1) + 2) * 2.0 ** -23 * size + 2.0 ** -8 * want.abs() + 1e-30
            assert bool(((out[at].double() - want).abs() <= tol).all()), (e, load)
        assert bool((out[~used] == 7).all())  # left as they were
    if kind == "ragged":
        filled = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot,
                                             zero_unused=True)
        plain = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts, padded, slot)
        assert bool((filled[~used] == 0).all()) and torch.equal(filled[used], plain[used])


def test_products_with_scales_in_any_layout_and_nan_beside_the_loads():
    from brainstorm_b200._C import expert as X

    loads, N, K = [3, 0, 60], 256, 384
    L = 80
    rows, weights = codes_of(L, K), codes_of(3, N, K)
    rs = torch.rand(L, 3, device="cuda") + 0.1
    ws = torch.rand(3, 2, 3, device="cuda") + 0.1
    counts = torch.tensor(loads, device="cuda")  # int64 loads
    want = X.grouped_expert_linear_fp8(rows, rs, weights, ws, counts)
    for other in (rs.t().contiguous().t(), torch.cat([rs, rs], 1)[:, :3],
                  rs.repeat_interleave(2, 0)[::2]):
        assert torch.equal(X.grouped_expert_linear_fp8(rows, other, weights, ws, counts)[:63],
                           want[:63])
    odd = rs.clone()
    odd[63:] = float("nan")
    nan = rows.clone()
    nan[63:] = torch.full((17, K), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    assert torch.equal(X.grouped_expert_linear_fp8(nan, odd, weights, ws, counts)[:63], want[:63])
    # loads that promise more rows than there are
    more = torch.tensor([3, 0, 600], dtype=torch.int32, device="cuda")
    assert torch.equal(X.grouped_expert_linear_fp8(rows, rs, weights, ws, more)[:63], want[:63])


@pytest.mark.parametrize("kind", list(LOADS))
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("N,K", [(128, 128), (16, 16), (256, 512), (400, 1040), (2000, 144)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grouped_expert_weight_grad(kind, padded, N, K, dtype):
    from brainstorm_b200._C import expert as X

    loads = LOADS[kind]
    E = len(loads)
    slot = max(loads) + 3 if padded else 0
    L = slot * E if padded else sum(loads) + 5
    torch.manual_seed(L + N + K)
    rows = torch.randn(L, K, device="cuda").bfloat16()
    grads = torch.randn(L, N, device="cuda").bfloat16()
    used = torch.zeros(L, dtype=torch.bool, device="cuda")
    for first, load in zip(starts(loads, slot), loads):
        used[first:first + load] = True
    rows[~used] = float("nan")  # not looked at
    grads[~used] = float("inf")
    counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
    got = X.grouped_expert_weight_grad(grads, rows, counts, padded, slot, dtype)
    X.check_status()
    assert got.dtype == dtype and got.shape == (E, N, K)
    for e, (first, load) in enumerate(zip(starts(loads, slot), loads)):
        g, x = grads[first:first + load].double(), rows[first:first + load].double()
        want, size = g.t() @ x, g.abs().t() @ x.abs()
        half = torch.finfo(dtype).eps / 2
        tol = (load + 1) * 2.0 ** -23 * size + half * want.abs() + 1e-30
        assert bool(((got[e].double() - want).abs() <= tol).all()), (e, load)


def test_expert_linear_fp8_gradients():
    """Against the same steps in 64 bits on the codes the operators themselves return."""
    from brainstorm_b200._C import expert as X

    loads, N, K, slot = [5, 0, 130, 64], 272, 400, 140
    E = len(loads)
    for padded in (False, True):
        L = slot * E if padded else sum(loads) + 9
        x = torch.randn(L, K, device="cuda").bfloat16().requires_grad_()
        w = (torch.randn(E, N, K, device="cuda") * 0.05).requires_grad_()
        counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
        out = X.expert_linear_fp8(x, w, counts, padded, slot if padded else 0)
        gy = torch.randn(L, N, device="cuda").bfloat16()
        gx, gw = torch.autograd.grad(out, (x, w), gy)
        X.check_status()
        assert gx.dtype == torch.bfloat16 and gw.dtype == torch.float32
        with torch.no_grad():
            xq, xs = X.quantize_rows(x)
            wq, ws = X.quantize_expert_weights(w)
            gq, gs = X.quantize_rows(gy)
        used = torch.zeros(L, dtype=torch.bool, device="cuda")
        for e, (first, load) in enumerate(zip(starts(loads, slot if padded else 0), loads)):
            at = slice(first, first + load)
            used[at] = True
            xd = xq[at].double() * spread(xs[at], K, 1)
            wd = wq[e].double() * spread(spread(ws[e], K, 1), N, 0)
            gd = gq[at].double() * spread(gs[at], N, 1)
            for got, a, b in ((out[at], xd, wd.t()), (gx[at], gd, wd),
                              (gw[e], gy[at].double().t(), x[at].double())):
                want, size = a @ b, a.abs() @ b.abs()
                half = torch.finfo(got.dtype).eps / 2
                terms = max(a.size(1), 128) + 20
                tol = terms * 2.0 ** -23 * size + half * want.abs() + 1e-30
                assert bool(((got.double() - want).abs() <= tol).all()), (padded, e)
        assert bool((out[~used] == 0).all()) and bool((gx[~used] == 0).all())


def test_layer_of_all_operators_and_its_gradients():
    """A feed-forward layer of experts from scores to cells, against 64 bits: both expert layers
    in 8 bits, so the tolerance is that of the codes (2^-4 relative to a block's values, and
    independent for the terms of a sum)."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    torch.manual_seed(0)
    T, k, E, d, hidden = 700, 2, 6, 256, 512
    cells = torch.randn(T, d, device="cuda").bfloat16().requires_grad_()
    up = (torch.randn(E, hidden, d, device="cuda") / 16).bfloat16().requires_grad_()
    down = (torch.randn(E, d, hidden, device="cuda") / 22).bfloat16().requires_grad_()
    score = torch.randn(T, E, device="cuda", requires_grad=True)

    def layer(dtype, linear):
        top, picks = torch.topk(score, k, dim=1)
        gates = torch.softmax(top, dim=1)
        return linear(picks, gates, cells.to(dtype), up.to(dtype), down.to(dtype))

    def fp8(picks, gates, cells, up, down):
        places, loads = R.order_picks(picks, E)
        rows = R.sort_cells(cells, places)
        mid = torch.relu(X.expert_linear_fp8(rows, up, loads))
        return R.unsort_cells(X.expert_linear_fp8(mid, down, loads), places, gates)

    def plain(picks, gates, cells, up, down):
        out = torch.zeros_like(cells)
        for e in range(E):
            t, j = torch.nonzero(picks == e, as_tuple=True)
            y = torch.relu(cells[t] @ up[e].t()) @ down[e].t()
            out = out.index_add(0, t, y * gates.double()[t, j].unsqueeze(1))
        return out

    leaves = (cells, up, down, score)
    gy = torch.randn(T, d, device="cuda")
    got = layer(torch.bfloat16, fp8)
    want = layer(torch.float64, plain)
    got_grads = torch.autograd.grad(got, leaves, gy.bfloat16())
    want_grads = torch.autograd.grad(want, leaves, gy.double())
    X.check_status()
    for a, b in zip((got,) + got_grads, (want,) + want_grads):
        off = (a.detach().double() - b.detach().double()).norm() / b.detach().double().norm()
        # each product's operands are off by at most 2^-4 of a value (0.036 rms of it) and four
        # such roundings are behind the deepest gradient
        assert float(off) < 4 * 2 * 2.0 ** -4, float(off)
        assert bool(torch.isfinite(a).all())


def test_captured_step_of_the_8_bit_layer():
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    T, k, E, d = 64, 4, 8, 256
    x = torch.randn(T, d, device="cuda").bfloat16()
    picks = torch.randint(0, E, (T, k), device="cuda")
    w, ws = X.quantize_expert_weights(torch.randn(E, d, d, device="cuda"))

    def step():
        places, loads = R.order_picks(picks, E)
        rows, rs = R.sort_cells_fp8(x, places)
        return R.unsort_cells(X.grouped_expert_linear_fp8(rows, rs, w, ws, loads), places)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(torch.randn(T, d, device="cuda"))
        picks.copy_(torch.randint(0, E, (T, k), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


@pytest.fixture(params=["native", "python"])
def host_side(request, monkeypatch):
    """The operators with their native host side, and with the Python that takes what it declines."""
    from brainstorm_b200 import _lib

    if request.param == "python":
        monkeypatch.setattr(_lib, "_host", _lib._DeclinesAll())
    return request.param


def test_both_host_sides(host_side):
    from brainstorm_b200._C import expert as X

    loads, N, K, slot = [3, 0, 40], 144, 272, 48
    L = slot * len(loads)
    x = torch.randn(L, K, device="cuda").bfloat16()
    g = torch.randn(L, N, device="cuda").bfloat16()
    w, ws = X.quantize_expert_weights(torch.randn(3, N, K, device="cuda"))
    counts = torch.tensor(loads, dtype=torch.int32, device="cuda")
    rows, rs = X.quantize_rows(x)
    check_codes(rows, rs, x, (1,))
    out = torch.full((L, N), 7.0, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):  # the first call makes the error word that the native side wants
        got = X.grouped_expert_linear_fp8(rows, rs, w, ws, counts, True, slot, out=out)
        filled = X.grouped_expert_linear_fp8(rows, rs, w, ws, counts, True, slot, True,
                                             zero_unused=True)
        grad = X.grouped_expert_weight_grad(g, x, counts, True, slot, torch.float32)
        half = X.grouped_expert_weight_grad(g, x, counts, True, 0)  # the slot from the sizes
    assert got is out and half.dtype == torch.bfloat16 and torch.equal(half, grad.bfloat16())
    for e, load in enumerate(loads):
        at, rest = slice(e * slot, e * slot + load), slice(e * slot + load, (e + 1) * slot)
        a = rows[at].double() * spread(rs[at], K, 1)
        b = w[e].double() * spread(spread(ws[e], K, 1), N, 0)
        want, size = a @ b.t(), a.abs() @ b.abs().t()
        tol = 140 * 2.0 ** -23 * size + 2.0 ** -8 * want.abs() + 1e-30
        assert bool(((out[at].double() - want).abs() <= tol).all())
        assert bool(((filled[at].double() - want.clamp(min=0)).abs() <= tol).all())
        assert bool((out[rest] == 7).all()) and bool((filled[rest] == 0).all())
        want = g[at].double().t() @ x[at].double()
        size = g[at].double().abs().t() @ x[at].double().abs()
        assert bool(((grad[e].double() - want).abs() <= (load + 2) * 2.0 ** -23 * size).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_between_two_codes_go_to_the_even_one(dtype):
    """bf16 and fp16 blocks whose maximum is a multiple of 7 hold many exact ties."""
    from brainstorm_b200._C import expert as X

    x = torch.arange(-140, 140, device="cuda").repeat(200)[:40 * 1280].view(40, 1280) / 128
    x[:, ::128] = 140 / 128  # scale 5 / 2048, exact in fp32
    x = x.to(dtype)
    codes, scales = X.quantize_rows(x)
    assert bool((scales == 5 / 2048).all())
    assert torch.equal(codes.float(), (x.double() / (5 / 2048)).float()
                       .to(torch.float8_e4m3fn).float())
    w, _ = X.quantize_expert_weights(x[:, :1280].repeat(4, 1).view(1, 160, 1280), True)
    want = codes.float().repeat(4, 1).view(160, 1280)
    assert torch.equal(w[0].float().t(), want)
