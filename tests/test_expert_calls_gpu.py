"""Calls of the expert layers that touch more than their numbers: buffers that autograd has saved, NaN
under a fused ReLU, operands that want gradients or carry forward-mode derivatives, first calls under
capture."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def host_side(request, monkeypatch):
    from brainstorm_b200 import _lib

    if request.param == "python":
        monkeypatch.setattr(_lib, "_host", _lib._DeclinesAll())
    return request.param


def layer(L=96, N=128, K=128, E=3, seed=0):
    """Operands of one expert layer in 8 bits and in bf16, 32 rows each but for the last expert."""
    from brainstorm_b200._C import expert as X

    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(L, K, device="cuda", generator=gen).bfloat16()
    w = (torch.randn(E, N, K, device="cuda", generator=gen) / 8).bfloat16()
    loads = torch.full((E,), L // E, dtype=torch.int32, device="cuda")
    return X.quantize_rows(x) + X.quantize_expert_weights(w), (x, w), loads


def products():
    from brainstorm_b200._C import expert as X

    fp8, bf16, loads = layer()
    return {
        "fp8": lambda **kw: X.grouped_expert_linear_fp8(*fp8, loads, **kw),
        "bf16": lambda **kw: X.grouped_expert_linear(*bf16, loads, **kw),
    }


# ------------------------------------------------------------------------------ buffers of the caller
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_a_saved_buffer_that_is_written_again_is_noticed(host_side, kind):
    """One buffer for the rows of two micro-batches: the first one's backward pass must not take the
    second one's rows."""
    from brainstorm_b200._C import router as R

    product = products()[kind]
    picks = torch.arange(96, device="cuda").view(48, 2) % 3
    places, _ = R.order_picks(picks, 3)
    gates = torch.rand(48, 2, device="cuda", requires_grad=True)
    buf = torch.empty(96, 128, dtype=torch.bfloat16, device="cuda")
    for _ in range(2):  # the first call makes what the native side wants
        before = buf._version
        assert product(out=buf) is buf and buf._version == before + 1
    out = R.unsort_cells(buf, places, gates)
    product(out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_buffers_made_in_inference_mode(host_side, kind):
    product = products()[kind]
    want = product()
    with torch.inference_mode():
        buf = torch.empty_like(want)
        assert torch.equal(product(out=buf), want)
        buf.zero_()
    assert torch.equal(product(out=buf), want)


# ------------------------------------------------------------------------------------------- ReLU
@pytest.mark.parametrize("rows_per_expert", [5, 40, 300])
def test_relu_keeps_nan_8_bit(host_side, rows_per_expert):
    """NaN in a row, in a weight and in a scale, and infinities of both signs that meet: what
    torch.relu makes of the product without it."""
    from brainstorm_b200._C import expert as X

    E, N, K = 3, 272, 272
    L = E * rows_per_expert
    torch.manual_seed(1)
    xq, xs = X.quantize_rows(torch.randn(L, K, device="cuda"))
    wq, ws = X.quantize_expert_weights(torch.randn(E, N, K, device="cuda"))
    nan = torch.tensor(float("nan"), device="cuda").to(torch.float8_e4m3fn)
    xq[3, 200] = nan
    wq[1, 17, 5] = nan
    xs = xs.clone()
    xs[rows_per_expert * 2 + 1, 0] = float("nan")
    xs[4, 0], xs[4, 1] = float("inf"), float("-inf")
    loads = torch.full((E,), rows_per_expert, dtype=torch.int32, device="cuda")
    for _ in range(2):
        plain = X.grouped_expert_linear_fp8(xq, xs, wq, ws, loads)
        got = X.grouped_expert_linear_fp8(xq, xs, wq, ws, loads, relu=True)
    X.check_status()
    assert bool(plain[3].isnan().all()) and bool(plain[rows_per_expert:, 17][:5].isnan().all())
    assert bool(plain[rows_per_expert * 2 + 1].isnan().all()) and bool(plain[4].isnan().any())
    assert torch.equal(got.isnan(), plain.isnan())
    assert torch.equal(got.nan_to_num(), torch.relu(plain).nan_to_num())
    assert bool((plain.nan_to_num() < 0).any())


@pytest.mark.parametrize("rows_per_expert", [5, 40, 300])
@pytest.mark.parametrize("N", [128, 256])
def test_relu_keeps_nan_bf16(rows_per_expert, N):
    from brainstorm_b200._C import expert as X

    E, K = 3, 128
    L = E * rows_per_expert
    torch.manual_seed(2)
    x = torch.randn(L, K, device="cuda").bfloat16()
    w = torch.randn(E, N, K, device="cuda").bfloat16()
    x[3, 100] = float("nan")
    w[1, 17, 5] = float("nan")
    x[4, 0], x[4, 1] = float("inf"), float("inf")  # weights of both signs: inf - inf
    loads = torch.full((E,), rows_per_expert, dtype=torch.int32, device="cuda")
    plain = X.grouped_expert_linear(x, w, loads)
    got = X.grouped_expert_linear(x, w, loads, relu=True)
    X.check_status()
    assert bool(plain[3].isnan().all()) and bool(plain[4].isnan().any())
    assert torch.equal(got.isnan(), plain.isnan())
    assert torch.equal(got.nan_to_num(), torch.relu(plain).nan_to_num())


# ------------------------------------------------------------------------------------ derivatives
@pytest.mark.parametrize("which", range(4))
def test_the_8_bit_product_refuses_operands_that_want_gradients(host_side, which):
    from brainstorm_b200._C import expert as X

    fp8, _, loads = layer()
    want = X.grouped_expert_linear_fp8(*fp8, loads)
    leaf = fp8[which].float().requires_grad_()
    operands = list(fp8)
    operands[which] = leaf.to(fp8[which].dtype)  # still part of the leaf's graph
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no gradient"):
            X.grouped_expert_linear_fp8(*operands, loads)
    with torch.no_grad():
        assert torch.equal(X.grouped_expert_linear_fp8(*operands, loads), want)


def test_the_8_bit_product_refuses_a_buffer_that_wants_a_gradient(host_side):
    from brainstorm_b200._C import expert as X

    fp8, _, loads = layer()
    want = X.grouped_expert_linear_fp8(*fp8, loads)
    buf = torch.zeros_like(want).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        X.grouped_expert_linear_fp8(*fp8, loads, out=buf)
    assert bool((buf == 0).all())
    with torch.no_grad():
        assert X.grouped_expert_linear_fp8(*fp8, loads, out=buf) is buf
    assert torch.equal(buf.detach(), want)


FORWARD = ["sort_cells", "sort_cells_fp8", "unsort_cells", "unsort_cells gates", "quantize_rows",
           "quantize_expert_weights", "linear rows' scales", "linear weights' scales", "weight_grad",
           "weight_grad rows", "expert_linear_fp8", "expert_linear_fp8 weights"]


@pytest.mark.parametrize("wants_grad", [False, True])
@pytest.mark.parametrize("name", FORWARD)
def test_forward_mode_derivatives_are_refused(host_side, name, wants_grad):
    """They would vanish without a word: no operator here has a forward-mode derivative."""
    import torch.autograd.forward_ad as fw

    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    fp8, (x, w), loads = layer()
    X.grouped_expert_linear_fp8(*fp8, loads)
    places, _ = R.order_picks(torch.arange(96, device="cuda").view(48, 2) % 3, 3)
    cells, gates = x[:48].contiguous(), torch.rand(48, 2, device="cuda")
    grads = torch.randn(96, 128, device="cuda").bfloat16()
    calls = {
        "sort_cells": (cells, lambda t: R.sort_cells(t, places)),
        "sort_cells_fp8": (cells, lambda t: R.sort_cells_fp8(t, places)),
        "unsort_cells": (x, lambda t: R.unsort_cells(t, places)),
        "unsort_cells gates": (gates, lambda t: R.unsort_cells(x, places, t)),
        "quantize_rows": (x, X.quantize_rows),
        "quantize_expert_weights": (w, X.quantize_expert_weights),
        "linear rows' scales": (
            fp8[1], lambda t: X.grouped_expert_linear_fp8(fp8[0], t, *fp8[2:], loads)),
        "linear weights' scales": (
            fp8[3], lambda t: X.grouped_expert_linear_fp8(*fp8[:3], t, loads)),
        "weight_grad": (grads, lambda t: X.grouped_expert_weight_grad(t, x, loads)),
        "weight_grad rows": (x, lambda t: X.grouped_expert_weight_grad(grads, t, loads)),
        "expert_linear_fp8": (x, lambda t: X.expert_linear_fp8(t, w, loads)),
        "expert_linear_fp8 weights": (w, lambda t: X.expert_linear_fp8(x, t, loads)),
    }
    value, call = calls[name]
    call(value)
    value = value.detach().clone().requires_grad_(wants_grad)
    with fw.dual_level():
        dual = fw.make_dual(value, torch.ones_like(value))
        with pytest.raises((RuntimeError, NotImplementedError), match="forward|no gradient|jvp"):
            call(dual)
        call(value.detach())  # without a tangent all is as ever


@pytest.mark.parametrize("name", ["sort_cells", "unsort_cells", "unsort_cells gates", "layer"])
def test_forward_mode_derivatives_of_gradients_are_refused(host_side, name):
    import torch.autograd.forward_ad as fw

    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    _, (x, w), loads = layer()
    places, _ = R.order_picks(torch.arange(96, device="cuda").view(48, 2) % 3, 3)
    leaf = (x[:48] if name == "sort_cells" else x).detach().clone().requires_grad_()
    gates = torch.rand(48, 2, device="cuda") if name.endswith("gates") else None
    out = {"sort_cells": lambda: R.sort_cells(leaf, places),
           "layer": lambda: X.expert_linear_fp8(leaf, w, loads)}.get(
               name, lambda: R.unsort_cells(leaf, places, gates))()
    gy = torch.randn_like(out)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, leaf, fw.make_dual(gy, torch.ones_like(gy)),
                                retain_graph=True)
        torch.autograd.grad(out, leaf, gy)


# ---------------------------------------------------------------------------------------- capture
def test_a_report_survives_the_replays_of_a_graph_captured_before_any_eager_call(monkeypatch):
    """The word that reports a wait which ran out is made by the first call.  When that call is
    captured, replays must not wipe out what a kernel reported in between."""
    from brainstorm_b200 import _lib
    from brainstorm_b200._C import expert as X

    fp8, _, loads = layer()
    want = X.grouped_expert_linear_fp8(*fp8, loads)
    torch.cuda.synchronize()
    monkeypatch.setattr(X, "_error_words", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = X.grouped_expert_linear_fp8(*fp8, loads)
    torch.cuda.synchronize()
    X.check_status()  # zero before the graph has run once
    graph.replay()
    X.check_status()
    assert torch.equal(out, want)
    (word,) = X._error_words.values()
    word.fill_(7)
    graph.replay()
    with pytest.raises(_lib.BrtError):
        X.check_status()
    X.check_status()


def test_a_report_is_not_written_by_what_else_a_graph_computes(monkeypatch):
    """Nor may the word share memory with what the capture that made it has let go."""
    from brainstorm_b200._C import expert as X

    fp8, _, loads = layer()
    want = X.grouped_expert_linear_fp8(*fp8, loads)
    torch.cuda.synchronize()
    monkeypatch.setattr(X, "_error_words", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for n in (1, 100, 1000, 100000):
            gone = torch.full((n,), 5, dtype=torch.int32, device="cuda")
            del gone
        out = X.grouped_expert_linear_fp8(*fp8, loads)
    for _ in range(2):
        graph.replay()
        X.check_status()
    assert torch.equal(out, want)


def test_the_first_product_of_a_process_may_be_captured():
    """Then even the library's kernels and its word are loaded under capture."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from brainstorm_b200._C import expert as X
rows, scales = torch.randn(96, 128, device="cuda").to(torch.float8_e4m3fn), torch.ones(96, 1, device="cuda")
w, ws = torch.randn(3, 128, 128, device="cuda").to(torch.float8_e4m3fn), torch.ones(3, 1, 1, device="cuda")
loads = torch.full((3,), 32, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = X.grouped_expert_linear_fp8(rows, scales, w, ws, loads)
graph.replay()
X.check_status()
assert torch.equal(out, X.grouped_expert_linear_fp8(rows, scales, w, ws, loads))
print("fine")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


# ------------------------------------------------------------------------------------- empty batches
@pytest.mark.parametrize("padded", [False, True])
def test_a_batch_without_rows(host_side, padded):
    """Serving and training of no cells at all: empty results, weights' gradients of zeros."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    E, N, K = 3, 128, 256
    picks = torch.empty(0, 2, dtype=torch.int64, device="cuda")
    cells = torch.empty(0, K, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    gates = torch.empty(0, 2, device="cuda", requires_grad=True)
    w = torch.randn(E, N, K, device="cuda", requires_grad=True)
    places, loads = R.order_picks(picks, E)
    with torch.no_grad():
        wq, ws = X.quantize_expert_weights(w)
        for _ in range(2):
            codes, scales = R.sort_cells_fp8(cells, places)
            y = X.grouped_expert_linear_fp8(codes, scales, wq, ws, loads, padded)
            assert y.shape == (0, N) and R.unsort_cells(y, places, gates).shape == (0, N)
            grad = X.grouped_expert_weight_grad(y, R.sort_cells(cells, places), loads, padded)
            assert grad.shape == (E, N, K) and bool((grad == 0).all())
    y = X.expert_linear_fp8(R.sort_cells(cells, places), w, loads, padded)
    out = R.unsort_cells(y, places, gates)
    grads = torch.autograd.grad(out, (cells, gates, w), torch.empty_like(out))
    assert grads[0].shape == (0, K) and grads[1].shape == (0, 2)
    assert bool((grads[2] == 0).all())
    X.check_status()


def test_no_experts_are_refused(host_side):
    from brainstorm_b200._C import expert as X

    rows = torch.randn(8, 32, device="cuda").bfloat16()
    codes, scales = X.quantize_rows(rows)
    wq, ws = X.quantize_expert_weights(torch.empty(0, 32, 32, device="cuda"))
    loads = torch.empty(0, dtype=torch.int32, device="cuda")
    for padded in (False, True):
        with pytest.raises(RuntimeError):
            X.grouped_expert_linear_fp8(codes, scales, wq, ws, loads, padded)
        with pytest.raises(RuntimeError):
            X.grouped_expert_weight_grad(rows, rows, loads, padded)


# ----------------------------------------------------------------------------------- calls at once
def test_layers_on_two_streams_at_once():
    """Everything that a layer launches, on two streams with inputs of their own, again and again."""
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    T, k, E, d, n = 6000, 2, 12, 256, 384
    made = []
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        made.append((torch.randint(-1, E, (T, k), device="cuda", generator=gen),
                     torch.randn(T, d, device="cuda", generator=gen).bfloat16(),
                     torch.randn(E, n, d, device="cuda", generator=gen).bfloat16(),
                     torch.rand(T, k, device="cuda", generator=gen),
                     torch.randn(T, n, device="cuda", generator=gen).bfloat16()))

    def step(picks, x, w, gates, gy):
        x, w, gates = (t.detach().requires_grad_() for t in (x, w, gates))
        places, loads = R.order_picks(picks, E)
        out = R.unsort_cells(X.expert_linear_fp8(R.sort_cells(x, places), w, loads), places, gates)
        return (out.detach(),) + torch.autograd.grad(out, (x, w, gates), gy)

    want = [step(*m) for m in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(step(*made[i]))
    torch.cuda.synchronize()
    X.check_status()
    for i in (0, 1):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
