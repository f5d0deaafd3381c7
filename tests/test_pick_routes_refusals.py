"""What the operators over compact picks and 8-bit codes refuse, before anything is launched."""
import pytest
import torch

P = 4096  # stands for an address: the refusals come before it is used


@pytest.mark.parametrize("name,args,words", [
    ("brt_order_picks", (P, 0, 8, 0, P, P, None, 0, None), "path_num 0"),
    ("brt_order_picks", (P, 0, 8, 1025, P, P, None, 0, None), "path_num 1025"),
    ("brt_order_picks", (P, 0, 2 ** 31, 4, P, P, None, 0, None), "32 bits"),
    ("brt_order_picks", (P, 0, 100000, 4, P, P, None, 0, None), "scratch holds 0"),
    ("brt_order_picks", (P, 0, 8, 4, P, None, None, 0, None), "loads is null"),
    ("brt_order_picks", (None, 0, 8, 4, P, P, None, 0, None), "null pointer"),
    ("brt_sort_cells", (P, P, P, 4, 2, 8, 7, None), "dtype 7"),
    ("brt_sort_cells", (P, P, P, 4, 0, 8, 0, None), "bad shape"),
    ("brt_sort_cells", (P, P, P, 2 ** 30, 8, 8, 0, None), "32 bits"),
    ("brt_sort_cells", (P, P, None, 4, 2, 8, 0, None), "null pointer"),
    ("brt_sort_cells_fp8", (P, P, P, P, 4, 2, 24, 2, None), "multiple of 16"),
    ("brt_sort_cells_fp8", (P + 8, P, P, P, 4, 2, 32, 2, None), "aligned"),
    ("brt_unsort_cells", (P, P, P, P, 4, 2, 8, 2, 1, None), "gates are"),
    ("brt_unsort_cells_backward", (P, P, P, P, P, P, 4, 2, 8, 2, 1, None), "gates are"),
    ("brt_unsort_cells_backward", (P, None, P, P, P, P, 4, 2, 8, 2, 0, None), "null pointer"),
    ("brt_quantize_rows", (P, P, P, 4, 40, 2, None), "multiple of 16"),
    ("brt_quantize_rows", (P, P, None, 4, 32, 2, None), "null pointer"),
    ("brt_quantize_expert_weights", (P, P, P, 2, 40, 32, 0, 2, None), "multiples of 16"),
    ("brt_quantize_expert_weights", (P, P, P, 70000, 32, 32, 0, 2, None), "path_num"),
    ("brt_grouped_expert_gemm_fp8",
     (P, P, 1, 1, P, P, P, P, 2000, 8, 0, 128, 128, 0, 0, P, None), "path_num 2000"),
    ("brt_grouped_expert_gemm_fp8",
     (P, P, 1, 1, P, P, P, P, 2, 8, 0, 136, 128, 0, 0, P, None), "in_features % 16"),
    ("brt_grouped_expert_gemm_fp8",
     (P + 4, P, 1, 1, P, P, P, P, 2, 8, 0, 128, 128, 0, 0, P, None), "aligned"),
    ("brt_grouped_expert_gemm_fp8",
     (P, P, 1, 1, P, P, P, P, 2, 8, -1, 128, 128, 0, 0, P, None), "negative"),
    ("brt_grouped_expert_gemm_fp8",
     (P, P, 1, 1, P, P, P, None, 2, 8, 0, 128, 128, 0, 0, P, None), "loads"),
    ("brt_grouped_expert_weight_grad",
     (P, P, P, P, 2, 8, 0, 128, 120, 0, P, None), "out_features % 16"),
    ("brt_grouped_expert_weight_grad",
     (P, P, P, P, 2, 8, 0, 128, 128, 1, P, None), "out_dtype 1"),
    ("brt_grouped_expert_weight_grad",
     (P, P + 8, P, P, 2, 8, 0, 128, 128, 0, P, None), "aligned"),
])
def test_the_library_refuses(name, args, words):
    from brainstorm_b200 import _lib

    with pytest.raises(_lib.BrtError, match=words):
        _lib.call(name, *args)


def test_nothing_to_do_needs_no_gpu():
    from brainstorm_b200 import _lib

    _lib.call("brt_sort_cells", None, None, None, 0, 2, 8, 0, None)
    _lib.call("brt_unsort_cells", None, None, None, None, 0, 2, 8, 0, 0, None)
    _lib.call("brt_quantize_rows", None, None, None, 0, 32, 0, None)
    _lib.call("brt_grouped_expert_gemm_fp8", None, None, 1, 1, None, None, None, P, 2, 0, 0, 128,
              128, 0, 0, P, None)
    assert _lib.query("brt_pick_order_scratch_bytes", 8, 64) == 0
    assert _lib.query("brt_pick_order_scratch_bytes", 1 << 20, 64) >= 65 * 4


def test_operators_refuse_cpu_tensors():
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    picks = torch.zeros(4, 2, dtype=torch.int32)
    rows = torch.zeros(8, 32)
    codes, scales = rows.to(torch.float8_e4m3fn), torch.zeros(8, 1)
    weights = torch.zeros(2, 32, 32)
    loads = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: R.order_picks(picks, 2), lambda: R.sort_cells(rows[:4], picks),
                 lambda: R.sort_cells_fp8(rows[:4], picks), lambda: R.unsort_cells(rows, picks),
                 lambda: X.quantize_rows(rows), lambda: X.quantize_expert_weights(weights),
                 lambda: X.grouped_expert_linear_fp8(codes, scales, weights.to(codes.dtype),
                                                     torch.zeros(2, 1, 1), loads),
                 lambda: X.grouped_expert_weight_grad(rows, rows, loads),
                 lambda: X.expert_linear_fp8(rows, weights, loads)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


@pytest.mark.gpu
def test_operators_refuse_wrong_arguments():
    from brainstorm_b200._C import expert as X
    from brainstorm_b200._C import router as R

    picks = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    places, _ = R.order_picks(picks, 2)
    x = torch.zeros(4, 32, device="cuda")
    rows = torch.zeros(8, 32, device="cuda")
    codes, scales = X.quantize_rows(rows)
    w, ws = X.quantize_expert_weights(torch.zeros(2, 32, 32, device="cuda"))
    loads = torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    half = rows.bfloat16()
    with pytest.raises(RuntimeError, match="int32 or int64"):
        R.order_picks(picks.float(), 2)
    with pytest.raises(RuntimeError, match="cells, k"):
        R.order_picks(picks[0], 2)
    with pytest.raises(RuntimeError, match="path_num 0"):
        R.order_picks(picks, 0)
    with pytest.raises(RuntimeError, match="path_num"):
        R.order_picks(picks, 1025)
    with pytest.raises(RuntimeError, match="5 cells"):
        R.sort_cells(torch.zeros(5, 32, device="cuda"), places)
    with pytest.raises(NotImplementedError):
        R.sort_cells(x.double(), places)
    with pytest.raises(RuntimeError, match="int32 tensor of order_picks"):
        R.sort_cells(x, places.long())
    with pytest.raises(NotImplementedError, match="multiple of 16"):
        R.sort_cells_fp8(x[:, :24], places)
    with pytest.raises(RuntimeError, match="no gradient"):
        R.sort_cells_fp8(x.clone().requires_grad_(), places)
    with pytest.raises(RuntimeError, match="7 rows"):
        R.unsort_cells(rows[:7], places)
    with pytest.raises(RuntimeError, match="shape and device"):
        R.unsort_cells(rows, places, torch.zeros(4, 3, device="cuda"))
    with pytest.raises(RuntimeError, match="float32 or match"):
        R.unsort_cells(rows, places, torch.zeros(4, 2, device="cuda").half())
    with pytest.raises(NotImplementedError, match="multiples of 16"):
        X.quantize_rows(rows[:, :24])
    with pytest.raises(RuntimeError, match="no gradient"):
        X.quantize_rows(rows.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="float8_e4m3fn"):
        X.grouped_expert_linear_fp8(rows, scales, w, ws, loads)
    with pytest.raises(RuntimeError, match="row_scales"):
        X.grouped_expert_linear_fp8(codes, scales[:7], w, ws, loads)
    with pytest.raises(RuntimeError, match="loads must hold"):
        X.grouped_expert_linear_fp8(codes, scales, w, ws, loads[:1])
    with pytest.raises(RuntimeError, match="padded buffer"):
        X.grouped_expert_linear_fp8(codes, scales, w, ws, loads, True, 5)
    with pytest.raises(RuntimeError, match="out must be"):
        X.grouped_expert_linear_fp8(codes, scales, w, ws, loads, out=half[:, :16])
    with pytest.raises(NotImplementedError, match="bf16"):
        X.grouped_expert_weight_grad(rows, rows, loads)
    with pytest.raises(RuntimeError, match="expected grads"):
        X.grouped_expert_weight_grad(half[:7], half, loads)
    with pytest.raises(NotImplementedError, match="bf16 rows"):
        X.expert_linear_fp8(rows, torch.zeros(2, 32, 32, device="cuda"), loads)
