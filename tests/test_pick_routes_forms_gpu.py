"""Sort, unsort and codes in the forms that many cells take, with row ends that cut an item, at every
access width, against 64-bit formulas."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(T, k, E, seed):
    from brainstorm_b200._C import router as R

    gen = torch.Generator().manual_seed(seed)
    picks = torch.randint(-1, E, (T, k), generator=gen)
    picks[T // 3] = -1  # a cell that goes nowhere
    flat = picks.flatten().numpy()
    key = np.where(flat >= 0, flat, E)
    order = np.argsort(key, kind="stable")
    row = np.empty_like(order)
    row[order] = np.arange(order.size)
    places, loads = R.order_picks(picks.cuda(), E)
    want = torch.tensor(np.where(key < E, row, -2 - row)).view(T, k)
    assert torch.equal(places.cpu().long(), want)
    t, j = torch.nonzero(places >= 0, as_tuple=True)
    return places, t, j, places[t, j].long()


def shifted(t, by):
    """The values of `t` in memory that begins `by` elements behind a 16-byte boundary."""
    held = torch.empty(t.numel() + by, dtype=t.dtype, device=t.device)
    out = held[by:].view(t.shape)
    out.copy_(t)
    return out


# widths: whole items of four accesses; of three; cut ends; 4- and 2-byte accesses
WIDTHS = [(torch.float32, 501), (torch.float32, 1024), (torch.float32, 516), (torch.bfloat16, 501),
          (torch.bfloat16, 1002), (torch.bfloat16, 1040), (torch.bfloat16, 1288),
          (torch.bfloat16, 2056), (torch.bfloat16, 2048), (torch.float16, 1026),
          (torch.float16, 1288)]


@pytest.mark.parametrize("gate_type", ["none", "f32", "same"])
@pytest.mark.parametrize("by", [0, 2, 1])
@pytest.mark.parametrize("dtype,d", WIDTHS)
def test_long_forms(dtype, d, by, gate_type):
    from brainstorm_b200._C import router as R

    T, k, E = 3000, 2, 30
    places, t, j, row = make(T, k, E, d)
    gen = torch.Generator(device="cuda").manual_seed(d + by)

    def normal(*shape):
        return shifted(torch.randn(*shape, device="cuda", generator=gen).to(dtype), by)

    x = normal(T, d).requires_grad_()
    rows = R.sort_cells(x, places)
    want = torch.zeros(T * k, d, dtype=dtype, device="cuda")
    want[row] = x.detach()[t]
    assert torch.equal(rows.detach(), want)
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 1e-30
    gy = normal(T * k, d)
    (gx,) = torch.autograd.grad(rows, x, gy)
    exact = torch.zeros(T, d, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(exact)
    exact.index_add_(0, t, gy.double()[row])
    size.index_add_(0, t, gy.double()[row].abs())
    assert bool(((gx.double() - exact).abs()
                 <= (k * 2.0 ** -24 * size + half * exact.abs() + least) * (1 + 1e-6)).all())

    rows = normal(T * k, d).requires_grad_()
    gates, weight = None, torch.ones(t.numel(), dtype=torch.float64, device="cuda")
    if gate_type != "none":
        gates = torch.rand(T, k, device="cuda", generator=gen).to(
            torch.float32 if gate_type == "f32" else dtype)
        weight = gates[t, j].double()
        gates.requires_grad_()
    out = R.unsort_cells(rows, places, gates)
    terms = rows.detach().double()[row] * weight.unsqueeze(1)
    exact = torch.zeros(T, d, dtype=torch.float64, device="cuda").index_add_(0, t, terms)
    size = torch.zeros_like(exact).index_add_(0, t, terms.abs())
    assert bool(((out.detach().double() - exact).abs()
                 <= (k * 2.0 ** -24 * size + half * exact.abs() + least) * (1 + 1e-6)).all())
    gy = normal(T, d)
    grads = torch.autograd.grad(out, [rows] + ([gates] if gates is not None else []), gy)
    want = torch.zeros(T * k, d, dtype=torch.float64, device="cuda")
    want[row] = gy.double()[t] * weight.unsqueeze(1)
    assert bool(((grads[0].double() - want).abs()
                 <= ((2.0 ** -24 + half) * want.abs() + least) * (1 + 1e-6)).all())
    if gates is not None:
        dots = gy.double()[t] * rows.detach().double()[row]
        want = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        want[t, j] = dots.sum(1)
        size = torch.zeros_like(want)
        size[t, j] = dots.abs().sum(1)
        tol = (d + 5) * 2.0 ** -24 * size + torch.finfo(gates.dtype).eps / 2 * want.abs() + least
        assert bool(((grads[1].double() - want).abs() <= tol * (1 + 1e-6)).all())


def check_codes(codes, scales, x):
    """Scales within fp32's rounding of max / 448; codes the nearest e4m3 value of x / scale."""
    blocks = torch.nn.functional.pad(x.double(), (0, -x.size(1) % 128)).unflatten(1, (-1, 128))
    amax = blocks.abs().amax(2).clamp(min=2.0 ** -100)
    assert bool(((scales.double() - amax / 448).abs() <= 2.0 ** -24 * amax / 448).all())
    want = x.double() / scales.double().repeat_interleave(128, 1)[:, :x.size(1)]
    tol = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10))
    assert bool(((codes.double() - want).abs() <= tol * (1 + 2.0 ** -10)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,width", [(1000, 1040), (1000, 1296), (700, 656), (900, 2064), (600, 1024)])
def test_codes_of_many_rows(L, width, dtype):
    from brainstorm_b200._C import expert as X

    x = torch.randn(L, width, device="cuda") * torch.exp(torch.randn(width, device="cuda"))
    x[7] = 0
    x = x.to(dtype)
    check_codes(*X.quantize_rows(x), x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,k,E,width", [(1, 8, 64, 2048), (33, 2, 5, 144), (300, 4, 16, 1040),
                                         (900, 3, 9, 656), (2000, 2, 30, 1024)])
def test_sorted_codes(T, k, E, width, dtype):
    from brainstorm_b200._C import router as R

    places, t, j, row = make(T, k, E, width)
    x = (torch.randn(T, width, device="cuda") * torch.exp(torch.randn(width, device="cuda"))).to(dtype)
    want = torch.zeros(T * k, width, dtype=dtype, device="cuda")
    want[row] = x[t]
    check_codes(*R.sort_cells_fp8(x, places), want)
