"""Buffers of more than 2^31 elements: their last rows are as right as their first."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_sorted_rows_beyond_31_bits():
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    T, k, d, E = 1_050_000, 2, 1024, 3  # 2.15e9 elements of rows
    picks = (torch.arange(T, device="cuda") % E).view(T, 1).repeat(1, k)
    places, loads = R.order_picks(picks, E)
    assert loads.tolist() == [T * k // E] * E
    x = (torch.arange(T, device="cuda") % 251).bfloat16().view(T, 1).expand(T, d).contiguous()
    rows = R.sort_cells(x, places)
    back = R.unsort_cells(rows, places)
    assert torch.equal(back, (x * 2).to(back.dtype))
    codes, scales = X.quantize_rows(rows)
    at = torch.tensor([0, 1, T * k // 2, T * k - 2, T * k - 1], device="cuda")
    value = codes[at].float() * scales[at].repeat_interleave(128, 1)
    # equal values fill a block: each is its maximum, code 448, off by the scale's rounding
    assert bool(((value - rows[at].float()).abs() <= 2.0 ** -23 * rows[at].float()).all())
    codes2, scales2 = R.sort_cells_fp8(x, places)
    assert torch.equal(codes2[at].float(), codes[at].float())
    assert torch.equal(scales2[at], scales[at])


def test_expert_products_beyond_31_bits():
    from brainstorm_b200._C import expert as X

    L, N, K, E = 540_000, 4096, 128, 4  # 2.2e9 elements of output
    rows = torch.zeros(L, K, device="cuda").to(torch.float8_e4m3fn)
    rows[-300:] = torch.randn(300, K, device="cuda").to(torch.float8_e4m3fn)
    scales = torch.rand(L, 1, device="cuda") + 0.5
    w, ws = X.quantize_expert_weights(torch.randn(E, N, K, device="cuda"))
    loads = torch.full((E,), L // E, dtype=torch.int32, device="cuda")
    out = X.grouped_expert_linear_fp8(rows, scales, w, ws, loads)
    X.check_status()
    a = rows[-300:].double() * scales[-300:].double()
    b = w[-1].double() * ws[-1].double().repeat_interleave(128, 0)
    want, size = a @ b.t(), a.abs() @ b.abs().t()
    # 128 additions in tensor memory, each off by at most 2^-23, and the rounding to bf16
    assert bool(((out[-300:].double() - want).abs()
                 <= 132 * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all())
    assert bool((out[:-300][::997] == 0).all())


def test_weight_gradients_beyond_31_bits():
    from brainstorm_b200._C import expert as X

    E, N, K, L = 120, 4096, 4608, 240  # 2.3e9 elements
    grads = torch.randn(L, N, device="cuda").bfloat16()
    rows = torch.randn(L, K, device="cuda").bfloat16()
    loads = torch.full((E,), L // E, dtype=torch.int32, device="cuda")
    out = X.grouped_expert_weight_grad(grads, rows, loads)
    X.check_status()
    for e in (0, 57, E - 1):
        g, x = grads[2 * e:2 * e + 2].double(), rows[2 * e:2 * e + 2].double()
        want, size = g.t() @ x, g.abs().t() @ x.abs()
        assert bool(((out[e].double() - want).abs()
                     <= 3 * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all())
