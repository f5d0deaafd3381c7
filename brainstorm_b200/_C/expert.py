"""The expert side of the dispatched layout: a grouped linear layer on the tensor cores.

No counterpart in the reference's ``brt._C.router``: there the experts run as horizontally
fused kernels compiled by its JIT (``brt._C.jit`` ``homo_invoke``,
src/backend/torch/jit.cc:54-75; benchmark/switch_moe/switch_expert.py:62-99 builds the FFN of
a Switch layer from them).  This op consumes the same buffer and the same per-expert loads,
with the loads staying on the device.
"""
import ctypes

import torch

from .. import _lib

_error_words = {}


class _Word:
    """An int32 at an address on the device, as ``torch.as_tensor`` takes it without a copy."""

    def __init__(self, address: int):
        self.__cuda_array_interface__ = {"shape": (1,), "typestr": "<i4", "data": (address, False),
                                         "version": 2}


def _error_word(device: torch.device) -> torch.Tensor:
    word = _error_words.get(device.index)
    if word is None:
        # the library's own memory: what is allocated while a graph is captured belongs to the graph,
        # whose replays write to it
        at = ctypes.c_void_p()
        with _lib.device_guard(device):
            _lib.call("brt_expert_error_word", ctypes.byref(at))
            word = torch.as_tensor(_Word(at.value), device=device)
        _error_words[device.index] = word
    return word


def _written(out: torch.Tensor) -> torch.Tensor:
    """``out``, a buffer of the caller's that has just been written: autograd notices when it had saved
    what was in it."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)
    return out


def grouped_expert_linear(rows: torch.Tensor, weights: torch.Tensor, loads: torch.Tensor,
                          max_path_padding: bool = False, max_path_load: int = 0,
                          relu: bool = False, out: torch.Tensor = None) -> torch.Tensor:
    """``out[r] = act(rows[r] @ weights[e].T)`` for the first ``loads[e]`` rows of every expert
    ``e`` of a dispatched buffer.

    ``rows`` [L, in] bf16 as ``dispatch_with_indices_and_loads`` returns it (padded to
    ``max_path_load`` rows per expert with ``max_path_padding``, else packed), ``weights``
    [E, out, in] bf16, ``loads`` [E] int32 on the device.  Returns [L, out] bf16; rows beyond an
    expert's load are left unwritten (combine never reads them).  ``in`` must be a multiple of
    64 and ``out`` of 128 (``NotImplementedError`` otherwise).  ``out``: a contiguous [L, out]
    bf16 tensor to write instead of a new one (e.g. ``expert_output_buffer`` of the
    expert-parallel exchange, which the fused combine pulls from)."""
    if not rows.is_cuda or not weights.is_cuda or not loads.is_cuda:
        raise RuntimeError("rows, weights and loads must be CUDA tensors")
    if rows.dtype != torch.bfloat16 or weights.dtype != torch.bfloat16:
        raise NotImplementedError("the tensor-core expert GEMM takes bf16 rows and weights")
    if rows.dim() != 2 or weights.dim() != 3 or weights.size(2) != rows.size(1) or \
            loads.numel() != weights.size(0):
        raise RuntimeError("expected rows [L, in], weights [E, out, in] and loads [E]")
    E, n_out, n_in = weights.shape
    L = rows.size(0)
    if max_path_padding:
        mpl = int(max_path_load) if max_path_load > 0 else L // E
        if mpl * E != L:
            raise RuntimeError("a padded buffer must hold max_path_load rows per expert")
    else:
        mpl = 0
    dev = rows.device
    with _lib.device_guard(dev):
        x = rows if rows.is_contiguous() else rows.contiguous()
        w = weights if weights.is_contiguous() else weights.contiguous()
        counts = loads if (loads.dtype == torch.int32 and loads.is_contiguous()) \
            else loads.to(torch.int32).contiguous()
        given = out is not None
        if not given:
            out = torch.empty((L, n_out), dtype=torch.bfloat16, device=dev)
        elif out.shape != (L, n_out) or out.dtype != torch.bfloat16 or \
                not out.is_contiguous() or out.device != dev:
            raise RuntimeError("out must be a contiguous [L, out_features] bf16 tensor on the "
                               "device of the rows")
        try:
            _lib.call("brt_grouped_expert_gemm", x.data_ptr(), w.data_ptr(), out.data_ptr(),
                      counts.data_ptr(), E, L, mpl, n_in, n_out, int(bool(relu)),
                      _error_word(dev).data_ptr(), _lib.raw_stream(dev))
        except _lib.BrtError as exc:
            if exc.status == 4:  # BRT_ERR_UNSUPPORTED: feature counts the tiles do not divide
                raise NotImplementedError(str(exc)) from None
            raise
    return _written(out) if given else out


_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_BLOCK = 128


def _blocks(n: int) -> int:
    return (n + _BLOCK - 1) // _BLOCK


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous and on a 16-byte boundary."""
    if not t.is_contiguous():
        return t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_features(*features: int) -> None:
    for n in features:
        if n < 1 or n % 16 != 0:
            raise NotImplementedError(f"features must be multiples of 16, got {n}")


def _no_gradient(name: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no gradient: use expert_linear_fp8, or no_grad()")
    _lib.refuse_tangents(name, *tensors)


def _slot(max_path_padding: bool, max_path_load: int, total_rows: int, path_num: int) -> int:
    if not max_path_padding or total_rows == 0:
        return 0
    slot = int(max_path_load) if max_path_load > 0 else total_rows // max(path_num, 1)
    if slot * path_num != total_rows or slot < 1:
        raise RuntimeError("a padded buffer must hold max_path_load rows per expert")
    return slot


def _loads(loads: torch.Tensor, path_num: int, dev: torch.device) -> torch.Tensor:
    if loads.numel() != path_num or loads.device != dev:
        raise RuntimeError(f"loads must hold one number for each of {path_num} experts, on the "
                           "device of the rows")
    return loads if loads.dtype == torch.int32 and loads.is_contiguous() \
        else loads.to(torch.int32).contiguous()


def quantize_rows(rows: torch.Tensor):
    """Rows [L, width] (fp32, fp16 or bf16) to 8-bit floating point with an fp32 scale for each
    128 neighbouring values: (codes [L, width] float8_e4m3fn, scales [L, ceil(width / 128)]), a
    value is ``code * scale``.  ``scale = max(max |x|, 2**-100) / 448`` and the code is the nearest to
    ``x / scale``.  The scales of a block lie together for all rows (strides (1, L)), as the products
    read them.  A NaN stays NaN by itself; an infinity makes its block's scale infinite and its codes
    NaN.  The width must be a multiple of 16."""
    done = _lib.host_ops().quantize_rows(rows)
    if done is not None:
        return done
    if not rows.is_cuda:
        raise RuntimeError("rows must be a CUDA tensor")
    if rows.dtype not in _DT:
        raise NotImplementedError(f"rows of {rows.dtype} are not supported")
    if rows.dim() != 2:
        raise RuntimeError(f"rows must be [L, width], got {tuple(rows.shape)}")
    _no_gradient("quantize_rows", rows)
    L, width = rows.shape
    _check_features(width)
    dev = rows.device
    with _lib.device_guard(dev):
        src = _aligned(rows)
        codes = torch.empty((L, width), dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty((_blocks(width), L), dtype=torch.float32, device=dev)
        _lib.call("brt_quantize_rows", src.data_ptr(), codes.data_ptr(), scales.data_ptr(), L,
                  width, _DT[rows.dtype], _lib.raw_stream(dev))
    return codes, scales.t()


def quantize_expert_weights(weights: torch.Tensor, transposed: bool = False):
    """Weights [E, out, in] (fp32, fp16 or bf16) to 8-bit floating point with an fp32 scale for
    each 128 x 128: (codes [E, out, in] float8_e4m3fn, scales [E, ceil(out / 128),
    ceil(in / 128)]).  ``transposed`` gives both with in and out exchanged: the weights with which
    the product takes gradients of the output to gradients of the rows.  Multiples of 16."""
    if not weights.is_cuda:
        raise RuntimeError("weights must be a CUDA tensor")
    if weights.dtype not in _DT:
        raise NotImplementedError(f"weights of {weights.dtype} are not supported")
    if weights.dim() != 3:
        raise RuntimeError(f"weights must be [E, out, in], got {tuple(weights.shape)}")
    _no_gradient("quantize_expert_weights", weights)
    E, n_out, n_in = weights.shape
    _check_features(n_out, n_in)
    dev = weights.device
    shape = (E, n_in, n_out) if transposed else (E, n_out, n_in)
    with _lib.device_guard(dev):
        src = _aligned(weights)
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev)
        scales = torch.empty((E, _blocks(shape[1]), _blocks(shape[2])), dtype=torch.float32,
                             device=dev)
        _lib.call("brt_quantize_expert_weights", src.data_ptr(), codes.data_ptr(),
                  scales.data_ptr(), E, n_in, n_out, int(bool(transposed)), _DT[weights.dtype],
                  _lib.raw_stream(dev))
    return codes, scales


def grouped_expert_linear_fp8(rows: torch.Tensor, row_scales: torch.Tensor,
                              weights: torch.Tensor, weight_scales: torch.Tensor,
                              loads: torch.Tensor, max_path_padding: bool = False,
                              max_path_load: int = 0, relu: bool = False,
                              out: torch.Tensor = None,
                              zero_unused: bool = False) -> torch.Tensor:
    """``grouped_expert_linear`` over 8-bit rows and weights with a scale for each block of 128.

    ``rows`` [L, in] float8_e4m3fn with ``row_scales`` [L, ceil(in / 128)] fp32 (any strides), as
    ``sort_cells_fp8`` or ``quantize_rows`` return them; ``weights`` [E, out, in] float8_e4m3fn with
    ``weight_scales`` [E, ceil(out / 128), ceil(in / 128)] fp32.  The scales may be any fp32
    numbers whose products are in fp32's normal range; sums run in fp32.  Returns [L, out] bf16.
    Rows beyond an expert's load are left unwritten, or set to zero with ``zero_unused``.  ``in``
    and ``out`` are multiples of 16.  The other arguments are those of ``grouped_expert_linear``.
    No gradient: train through ``expert_linear_fp8``."""
    word = _error_words.get(rows.get_device())
    if word is not None and (not max_path_padding or max_path_load > 0):
        done = _lib.host_ops().grouped_expert_linear_fp8(
            rows, row_scales, weights, weight_scales, loads,
            max_path_load if max_path_padding else 0, relu, out, zero_unused, word)
        if done is not None:
            return done
    for t in (rows, row_scales, weights, weight_scales, loads):
        if not t.is_cuda:
            raise RuntimeError("rows, weights, their scales and loads must be CUDA tensors")
    if rows.dtype != torch.float8_e4m3fn or weights.dtype != torch.float8_e4m3fn:
        raise NotImplementedError("the 8-bit expert GEMM takes float8_e4m3fn rows and weights")
    if rows.dim() != 2 or weights.dim() != 3 or weights.size(2) != rows.size(1):
        raise RuntimeError("expected rows [L, in] and weights [E, out, in]")
    E, n_out, n_in = weights.shape
    L = rows.size(0)
    _check_features(n_out, n_in)
    if row_scales.dtype != torch.float32 or weight_scales.dtype != torch.float32 or \
            row_scales.shape != (L, _blocks(n_in)) or \
            weight_scales.shape != (E, _blocks(n_out), _blocks(n_in)):
        raise RuntimeError("expected fp32 row_scales [L, in / 128] and weight_scales "
                           "[E, out / 128, in / 128], rounded up")
    _no_gradient("grouped_expert_linear_fp8", rows, row_scales, weights, weight_scales,
                 *(() if out is None else (out,)))
    dev = rows.device
    if any(t.device != dev for t in (row_scales, weights, weight_scales)):
        raise RuntimeError("rows, weights and their scales are on different devices")
    slot = _slot(max_path_padding, max_path_load, L, E)
    with _lib.device_guard(dev):
        counts = _loads(loads, E, dev)
        x, w = _aligned(rows), _aligned(weights)
        ws = weight_scales if weight_scales.is_contiguous() else weight_scales.contiguous()
        given = out is not None
        if not given:
            out = torch.empty((L, n_out), dtype=torch.bfloat16, device=dev)
        elif out.shape != (L, n_out) or out.dtype != torch.bfloat16 or \
                not out.is_contiguous() or out.device != dev or out.data_ptr() % 16 != 0:
            raise RuntimeError("out must be a contiguous, 16-byte aligned [L, out_features] bf16 "
                               "tensor on the device of the rows")
        _lib.call("brt_grouped_expert_gemm_fp8", x.data_ptr(), row_scales.data_ptr(),
                  row_scales.stride(0), row_scales.stride(1), w.data_ptr(), ws.data_ptr(),
                  out.data_ptr(), counts.data_ptr(), E, L, slot, n_in, n_out, int(bool(relu)),
                  int(bool(zero_unused)), _error_word(dev).data_ptr(), _lib.raw_stream(dev))
    return _written(out) if given else out


def grouped_expert_weight_grad(grads: torch.Tensor, rows: torch.Tensor, loads: torch.Tensor,
                               max_path_padding: bool = False, max_path_load: int = 0,
                               dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The gradient of an expert layer's weights: ``out[e] = grads[rows of e].T @ rows[rows of
    e]``, for ``grads`` [L, out] bf16 (the gradient of the layer's output) and ``rows`` [L, in] bf16
    (what went into it), laid out and counted by ``loads`` as for ``grouped_expert_linear``.
    Returns [E, out, in] in ``dtype`` (bf16 or fp32), fp32 sums rounded once; zeros for an expert
    without rows.  Rows beyond an expert's load are not looked at.  Multiples of 16."""
    word = _error_words.get(rows.get_device())
    if word is not None and (not max_path_padding or max_path_load > 0) and \
            dtype in (torch.bfloat16, torch.float32):
        done = _lib.host_ops().grouped_expert_weight_grad(
            grads, rows, loads, max_path_load if max_path_padding else 0,
            dtype == torch.float32, word)
        if done is not None:
            return done
    if not grads.is_cuda or not rows.is_cuda or not loads.is_cuda:
        raise RuntimeError("grads, rows and loads must be CUDA tensors")
    if grads.dtype != torch.bfloat16 or rows.dtype != torch.bfloat16 or \
            dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("the weight gradient takes bf16 grads and rows and gives bf16 "
                                  "or fp32")
    if grads.dim() != 2 or rows.dim() != 2 or grads.size(0) != rows.size(0) or loads.dim() != 1 \
            or loads.numel() < 1 or grads.device != rows.device:
        raise RuntimeError("expected grads [L, out], rows [L, in] and loads [E] on one device")
    _no_gradient("grouped_expert_weight_grad", grads, rows)
    L, n_out = grads.shape
    n_in, E = rows.size(1), loads.numel()
    _check_features(n_out, n_in)
    slot = _slot(max_path_padding, max_path_load, L, E)
    dev = rows.device
    with _lib.device_guard(dev):
        counts = _loads(loads, E, dev)
        g, x = _aligned(grads), _aligned(rows)
        out = torch.empty((E, n_out, n_in), dtype=dtype, device=dev)
        _lib.call("brt_grouped_expert_weight_grad", g.data_ptr(), x.data_ptr(), out.data_ptr(),
                  counts.data_ptr(), E, L, slot, n_in, n_out, _DT[dtype],
                  _error_word(dev).data_ptr(), _lib.raw_stream(dev))
    return out


class _ExpertLinearFp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, loads, max_path_padding, max_path_load):
        ctx.save_for_backward(rows, weights, loads)
        ctx.layout = (max_path_padding, max_path_load)
        return grouped_expert_linear_fp8(*quantize_rows(rows), *quantize_expert_weights(weights),
                                         loads, *ctx.layout, zero_unused=True)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grads):
        rows, weights, loads = ctx.saved_tensors
        _lib.host_ops().check_capture(ctx.next_functions)
        row_grads = weight_grads = None
        if ctx.needs_input_grad[0]:
            back = quantize_expert_weights(weights, transposed=True)
            row_grads = grouped_expert_linear_fp8(*quantize_rows(grads), *back, loads, *ctx.layout,
                                                  zero_unused=True)
        if ctx.needs_input_grad[1]:
            weight_grads = grouped_expert_weight_grad(grads, rows, loads, *ctx.layout,
                                                      dtype=weights.dtype)
        return row_grads, weight_grads, None, None, None


def expert_linear_fp8(rows: torch.Tensor, weights: torch.Tensor, loads: torch.Tensor,
                      max_path_padding: bool = False, max_path_load: int = 0) -> torch.Tensor:
    """One expert layer for training, its products over rows in 8 bits: quantises ``rows`` [L, in]
    bf16 and ``weights`` [E, out, in] (bf16 or fp32) in blocks of 128 and multiplies them
    (``grouped_expert_linear_fp8``).  The gradient of the rows is the product of the quantised
    gradient of the output with the quantised transposed weights, the gradient of the weights the
    bf16 product of that gradient with the rows; the roundings to 8 bits count as the identity.
    Rows beyond an expert's load come out as zeros, and so do their gradients."""
    if not rows.is_cuda or not weights.is_cuda or not loads.is_cuda:
        raise RuntimeError("rows, weights and loads must be CUDA tensors")
    if rows.dtype != torch.bfloat16 or weights.dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("expert_linear_fp8 takes bf16 rows and bf16 or fp32 weights")
    if rows.dim() != 2 or weights.dim() != 3 or weights.size(2) != rows.size(1):
        raise RuntimeError("expected rows [L, in] and weights [E, out, in]")
    _lib.refuse_tangents("expert_linear_fp8", rows, weights)
    return _ExpertLinearFp8.apply(rows, weights, loads, bool(max_path_padding),
                                  int(max_path_load))


def check_status(device=None) -> None:
    """Synchronise and raise if a bounded wait inside an expert GEMM ran out."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    word = _error_words.get(dev.index)
    if word is not None and int(word.item()) != 0:
        word.zero_()
        raise _lib.BrtError("an expert GEMM gave up a bounded wait; its output is incomplete", 7)
