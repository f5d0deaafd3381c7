"""Operators of a mixture-of-experts layer over compact picks, as measurable cases.

Each case's ``op`` names the operator:

``sort``      picks of a top-k -> places and loads, and the cells as rows sorted by path; with
              ``train`` the gradient of the cells too, with ``fp8`` the rows as 8-bit codes with
              a scale for each block of 128
``unsort``    rows back to cells, weighted by the gates; with ``train`` the gradients of rows
              and gates too
``quantize``  a matrix of rows, or the experts' weights (transposed), to 8-bit codes with scales
``linear``    one expert layer in 8 bits: rows and weights as codes with a scale for each block
``wgrad``     the gradient of the experts' weights from the rows and the gradient of the output

With ``own`` false the operators are computed in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100  # smallest maximum that a block's scale is made from
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a serving batch, 8 of 64 experts, rows handed to the 8-bit expert layer
        dict(name="sort_one_token_fp8", op="sort", cells=1, k=8, paths=64, width=2048,
             dtype="bf16", bias="none", dropped=0.0, fp8=True, train=False, wide=True),
        # the benchmark's headline routing, 32768 tokens to 2 of 32 experts, in a training step
        dict(name="sort_train_top2", op="sort", cells=32768, k=2, paths=32, width=1024,
             dtype="bf16", bias="normal", dropped=0.0, fp8=False, train=True, wide=False),
        # odd everything: rows of 2004 bytes, picks that a padded batch leaves out
        dict(name="sort_ragged_f32", op="sort", cells=9001, k=3, paths=30, width=501,
             dtype="f32", bias="normal", dropped=0.1, fp8=False, train=True, wide=True),
        # a decode batch back from its experts: latency
        dict(name="unsort_decode", op="unsort", cells=64, k=8, paths=64, width=2048,
             dtype="bf16", bias="none", dropped=0.0, train=False, wide=False),
        # a training batch with 8 experts per token: the most rows
        dict(name="unsort_train_top8", op="unsort", cells=16384, k=8, paths=64, width=2048,
             dtype="bf16", bias="normal", dropped=0.0, train=True, wide=False),
        # the rows of a long prompt before an expert layer
        dict(name="quantize_rows", op="quantize", rows=65536, inner=2048, paths=0, outer=0,
             dtype="bf16"),
        # all experts' weights as the backward pass of a training step wants them
        dict(name="quantize_weights", op="quantize", rows=0, inner=1024, paths=32, outer=4096,
             dtype="bf16"),
        # one token at 8 of 64 experts: reading their weights is the cost
        dict(name="linear_one_token", op="linear", rows=8, paths=64, inner=2048, outer=4096,
             bias="one", padded=False, relu=False),
        # blocks that are cut at the end of both axes, uneven loads, slots of fixed size
        dict(name="linear_ragged", op="linear", rows=9001, paths=30, inner=1040, outer=2000,
             bias="normal", padded=True, relu=True),
        # a long prompt: the tensor cores are the cost
        dict(name="linear_prefill", op="linear", rows=65536, paths=32, inner=4096, outer=4096,
             bias="normal", padded=False, relu=False),
        # uneven experts of a small training batch, odd widths
        dict(name="wgrad_ragged", op="wgrad", rows=9001, paths=30, inner=1040, outer=2000,
             bias="zipf", wide=True),
        # the benchmark's batch at its expert layer
        dict(name="wgrad_top2", op="wgrad", rows=65536, paths=32, inner=1024, outer=4096,
             bias="normal", wide=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_any(rng):
    op = rng.choice(["sort", "sort", "unsort", "quantize", "linear", "linear", "wgrad"])
    bias = rng.choice(["none", "normal", "zipf"])
    if op in ("sort", "unsort"):
        paths = _log_int(rng, 2, 256)
        fp8 = op == "sort" and rng.random() < 0.4
        width = 16 * _log_int(rng, 4, 256) if fp8 or rng.random() < 0.6 else _log_int(rng, 24, 4096)
        case = dict(op=op, cells=_log_int(rng, 1, 65536), k=rng.choice([1, 2, 3, 4, 6, 8]),
                    paths=paths, width=width, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    bias=bias, dropped=rng.choice([0.0, 0.0, 0.05, 0.5]))
        if op == "sort":
            case["fp8"] = fp8
        return dict(case, train=not fp8 and rng.random() < 0.6, wide=rng.random() < 0.5)
    if op == "quantize":
        if rng.random() < 0.5:
            return dict(op=op, rows=_log_int(rng, 1, 65536), inner=16 * _log_int(rng, 8, 512),
                        paths=0, outer=0, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
        return dict(op=op, rows=0, inner=16 * _log_int(rng, 8, 256), paths=_log_int(rng, 1, 64),
                    outer=16 * _log_int(rng, 8, 256), dtype=rng.choice(["bf16", "bf16", "f32"]))
    sizes = dict(op=op, rows=_log_int(rng, 1, 65536), paths=_log_int(rng, 1, 128),
                 inner=16 * _log_int(rng, 8, 256), outer=16 * _log_int(rng, 8, 256), bias=bias)
    if op == "linear":
        return dict(sizes, padded=rng.random() < 0.3, relu=rng.random() < 0.3)
    return dict(sizes, wide=rng.random() < 0.4)


def draw(rng):
    """One more case of the ranges above, none dearer than the largest listed one of its op."""
    limits = {}
    for case in listed():
        w = work(case)
        old = limits.get(case["op"], {"bytes": 0, "flops": 0})
        limits[case["op"]] = {key: max(old[key], w[key]) for key in w}
    while True:
        case = _draw_any(rng)
        w, limit = work(case), limits[case["op"]]
        if w["bytes"] <= limit["bytes"] and w["flops"] <= limit["flops"]:
            return case


# ------------------------------------------------------------------------------------ inputs
def _loads(case):
    """Rows per expert, the same for every seed: what the work of a case goes by."""
    E, rows = case["paths"], case["rows"]
    rng = np.random.RandomState(7)
    if case["bias"] == "one":  # the picks of one token: as many experts with a row each
        loads = np.zeros(E, dtype=np.int64)
        loads[rng.permutation(E)[:rows]] = 1
        return loads
    if case["bias"] == "zipf":
        p = 1.0 / np.arange(1, E + 1) ** 1.1
        p = p[rng.permutation(E)]
    else:
        p = np.exp(rng.randn(E) * (0.5 if case["bias"] == "normal" else 0.05))
    return rng.multinomial(rows, p / p.sum())


def _slot(case):
    """Rows of an expert's slot in a padded buffer, 0 when the rows are packed."""
    return int(-(-int(_loads(case).max()) // 8) * 8) if case.get("padded") else 0


def _picks(case, gen):
    T, E, k = case["cells"], case["paths"], case["k"]
    logits = torch.randn(T, E, device="cuda", generator=gen)
    if case["bias"] == "normal":
        logits += 0.5 * torch.randn(E, device="cuda", generator=gen)
    elif case["bias"] == "zipf":
        logits -= 1.1 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    score, picks = torch.topk(logits, min(k, E), dim=1)
    if k > E:  # more picks than paths: the same paths again
        picks = picks.repeat(1, -(-k // E))[:, :k]
        score = score.repeat(1, -(-k // E))[:, :k]
    if case["dropped"]:
        picks = picks.masked_fill(
            torch.rand(T, k, device="cuda", generator=gen) < case["dropped"], -1)
    return picks if case["wide"] else picks.to(torch.int32), torch.softmax(score, dim=1)


def _codes(x):
    """8-bit codes and scales of [..., K] values, a block of 128 along K each (prepared data)."""
    K = x.size(-1)
    blocks = torch.nn.functional.pad(x, (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1).clamp(min=AMAX_FLOOR)
    codes = (blocks * (E4M3_MAX / amax).unsqueeze(-1)).clamp(-E4M3_MAX, E4M3_MAX).flatten(-2)
    return codes[..., :K].to(E4M3).contiguous(), amax / E4M3_MAX


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen).to(dtype)

    op = case["op"]
    if op in ("sort", "unsort"):
        dtype = DTYPES[case["dtype"]]
        T, L, d = case["cells"], case["cells"] * case["k"], case["width"]
        picks, gates = _picks(case, gen)
        state.update(picks=picks)
        if op == "sort":
            # activations have channels of very different size
            state["cells"] = (normal(T, d) * torch.exp(normal(d))).to(dtype)
            if case["train"]:
                state["cells"].requires_grad_()
                state["row_grads"] = normal(L, d, dtype=dtype)
        else:
            state["rows"] = normal(L, d, dtype=dtype)
            state["gates"] = gates
            state["places"], _ = _order(picks, case["paths"])
            if case["train"]:
                state["rows"].requires_grad_()
                state["gates"].requires_grad_()
                state["cell_grads"] = normal(T, d, dtype=dtype)
        return state
    if op == "quantize":
        dtype = DTYPES[case["dtype"]]
        if case["rows"]:
            x = normal(case["rows"], case["inner"])
            state["rows"] = (x * torch.exp(normal(case["inner"]))).to(dtype)
        else:
            w = normal(case["paths"], case["outer"], case["inner"])
            state["weights"] = (w * (0.02 * torch.exp(0.5 * normal(case["outer"], 1)))).to(dtype)
        return state
    loads, slot = _loads(case), _slot(case)
    L = slot * case["paths"] if slot else case["rows"]
    state["loads"] = torch.tensor(loads, dtype=torch.int32, device="cuda")
    state["slot"] = slot
    if op == "linear":
        rows, scales = _codes(normal(L, case["inner"]) * torch.exp(normal(case["inner"])))
        state["rows"], state["row_scales"] = rows, scales.t().contiguous().t()
        E, N, K = case["paths"], case["outer"], case["inner"]
        state["weights"] = torch.empty(E, N, K, dtype=E4M3, device="cuda")
        blocks = [-(-N // BLOCK), -(-K // BLOCK)]
        state["weight_scales"] = torch.empty(E, *blocks, device="cuda")
        for e in range(E):
            w = torch.nn.functional.pad(0.02 * normal(N, K), (0, -K % BLOCK, 0, -N % BLOCK))
            w = w.unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
            amax = w.abs().amax((1, 3)).clamp(min=AMAX_FLOOR)
            w = (w * (E4M3_MAX / amax)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
            state["weights"][e] = w.flatten(2).flatten(0, 1)[:N, :K].to(E4M3)
            state["weight_scales"][e] = amax / E4M3_MAX
        # rows that no expert reaches stay as they are in a buffer that the program keeps
        state["out"] = torch.zeros(L, N, dtype=torch.bfloat16, device="cuda")
    else:
        state["rows"] = normal(L, case["inner"], dtype=torch.bfloat16)
        state["grads"] = normal(L, case["outer"], dtype=torch.bfloat16)
    return state


# --------------------------------------------------------------------------- the plain forms
def _order(picks, paths):
    """places [T, k] and loads [E] of a stable sort by path.  Picks that are no path come last;
    -2 - row stands for them: the row that stays empty in their place."""
    flat = picks.reshape(-1).long()
    valid = (flat >= 0) & (flat < paths)
    key = torch.where(valid, flat, paths)
    order = torch.argsort(key, stable=True)
    places = torch.empty_like(flat)
    places[order] = torch.arange(flat.numel(), device=flat.device)
    places = torch.where(valid, places, -2 - places)
    loads = torch.zeros(paths + 1, dtype=torch.int32, device=flat.device)
    loads.index_add_(0, key, torch.ones_like(key, dtype=torch.int32))
    return places.view(picks.shape).to(torch.int32), loads[:paths]


def _taken(rows, places):
    """[T, k, d]: the row at each place in fp32, zeros where there is none."""
    got = rows.float()[places.clamp(min=0).long()]
    return torch.where((places >= 0).unsqueeze(-1), got, torch.zeros((), device=rows.device))


def _placed(values, places):
    """[T * k, d]: values [T, k, d] written to their places, zeros elsewhere."""
    L = places.numel()
    out = torch.zeros(L + 1, values.size(-1), dtype=values.dtype, device=values.device)
    flat = places.reshape(-1).long()
    out[torch.where(flat >= 0, flat, L)] = values.reshape(L, -1)
    return out[:L]


def _quantized(x):
    """x [..., K] -> codes and scales, a scale for each block of 128 along the last axis."""
    K = x.size(-1)
    blocks = torch.nn.functional.pad(x.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1).clamp(min=AMAX_FLOOR)
    codes = blocks * (E4M3_MAX / amax).unsqueeze(-1)
    codes = codes.clamp(-E4M3_MAX, E4M3_MAX).to(E4M3).flatten(-2)[..., :K]
    return codes, amax / E4M3_MAX


def _quantized_weights(w):
    """w [E, N, K] -> codes [E, N, K] and scales [E, N / 128, K / 128]."""
    E, N, K = w.shape
    w = torch.nn.functional.pad(w.float(), (0, -K % BLOCK, 0, -N % BLOCK))
    w = w.unflatten(1, (-1, BLOCK)).unflatten(3, (-1, BLOCK))
    amax = w.abs().amax((2, 4)).clamp(min=AMAX_FLOOR)
    codes = (w * (E4M3_MAX / amax)[:, :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)
    return codes.flatten(3).flatten(1, 2)[:, :N, :K], amax / E4M3_MAX


def _at(loads, slot):
    """Which expert each row with one belongs to, its number there, and its place."""
    counts = loads.long()
    expert = torch.repeat_interleave(torch.arange(counts.numel(), device=loads.device), counts)
    first = torch.cumsum(counts, 0) - counts
    seat = torch.arange(expert.numel(), device=loads.device) - first[expert]
    place = expert * slot + seat if slot else torch.arange(expert.numel(), device=loads.device)
    return expert, seat, place


def _by_expert(values, at, paths, most):
    """[E, most, n]: each expert's rows, zeros behind them."""
    expert, seat, place = at
    out = torch.zeros(paths, most, values.size(1), dtype=values.dtype, device=values.device)
    out[expert, seat] = values[place]
    return out


def _plain(state):
    case = state["case"]
    op = case["op"]
    with torch.no_grad():
        if op == "sort":
            places, loads = _order(state["picks"], case["paths"])
            cells = state["cells"].unsqueeze(1).expand(-1, case["k"], -1)
            if case["fp8"]:
                rows, scales = _quantized(_placed(cells, places))
                return places, loads, rows, scales
            rows = _placed(cells, places)
            if not case["train"]:
                return places, loads, rows
            grad = _taken(state["row_grads"], places).sum(1).to(rows.dtype)
            return places, loads, rows, grad
        if op == "unsort":
            places, gates = state["places"], state["gates"]
            taken = _taken(state["rows"], places)
            out = (taken * gates.unsqueeze(-1)).sum(1).to(state["rows"].dtype)
            if not case["train"]:
                return out
            g = state["cell_grads"].float().unsqueeze(1)
            rows_grad = _placed((g * gates.unsqueeze(-1)).to(out.dtype), places)
            return out, rows_grad, (g * taken).sum(-1)
        if op == "quantize":
            if case["rows"]:
                return _quantized(state["rows"])
            return _quantized_weights(state["weights"].transpose(1, 2))
        loads = state["loads"]
        at, most = _at(loads, state["slot"]), int(loads.max())
        if op == "linear":
            x = state["rows"].float() * _spread(state["row_scales"], case["inner"], 1)
            w = state["weights"].float() * _spread(
                _spread(state["weight_scales"], case["inner"], 2), case["outer"], 1)
            y = torch.bmm(_by_expert(x, at, case["paths"], most), w.transpose(1, 2))
            if case["relu"]:
                y = y.clamp(min=0)
            out = torch.zeros_like(state["out"])
            out[at[2]] = y[at[0], at[1]].to(out.dtype)
            return out
        x = _by_expert(state["rows"].float(), at, case["paths"], most)
        g = _by_expert(state["grads"].float(), at, case["paths"], most)
        grad = torch.bmm(g.transpose(1, 2), x)
        return grad if case["wide"] else grad.to(torch.bfloat16)


def _spread(scales, size, dim):
    """Scales of blocks -> of every one of `size` values along `dim`."""
    return scales.repeat_interleave(BLOCK, dim).narrow(dim, 0, size)


# ------------------------------------------------------------------- the framework's operators
def _framework(state):
    from brainstorm_b200._C import expert, router

    case = state["case"]
    op = case["op"]
    if op == "sort":
        places, loads = router.order_picks(state["picks"], case["paths"])
        if case["fp8"]:
            rows, scales = router.sort_cells_fp8(state["cells"], places)
            return places, loads, rows, scales
        rows = router.sort_cells(state["cells"], places)
        if not case["train"]:
            return places, loads, rows
        (grad,) = torch.autograd.grad(rows, state["cells"], state["row_grads"])
        return places, loads, rows.detach(), grad
    if op == "unsort":
        out = router.unsort_cells(state["rows"], state["places"], state["gates"])
        if not case["train"]:
            return out
        grads = torch.autograd.grad(out, (state["rows"], state["gates"]), state["cell_grads"])
        return (out.detach(), *grads)
    if op == "quantize":
        if case["rows"]:
            return expert.quantize_rows(state["rows"])
        return expert.quantize_expert_weights(state["weights"], transposed=True)
    slot = state["slot"]
    if op == "linear":
        return expert.grouped_expert_linear_fp8(
            state["rows"], state["row_scales"], state["weights"], state["weight_scales"],
            state["loads"], max_path_padding=slot > 0, max_path_load=slot, relu=case["relu"],
            out=state["out"])
    return expert.grouped_expert_weight_grad(
        state["grads"], state["rows"], state["loads"],
        dtype=torch.float32 if case["wide"] else torch.bfloat16)


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------------- floors
def work(case):
    """Bytes and operations of one pass: every input read once, every output written once."""
    op = case["op"]
    if op in ("sort", "unsort"):
        size = 4 if case["dtype"] == "f32" else 2
        T, L, d = case["cells"], case["cells"] * case["k"], case["width"]
        if op == "sort":
            index = L * (8 if case["wide"] else 4) + 4 * L + 4 * case["paths"]
            row = d + 4 * -(-d // BLOCK) if case["fp8"] else d * size
            moved = T * d * size + L * row
            if case["train"]:
                moved += L * d * size + T * d * size
            return {"bytes": index + moved, "flops": L * d if case["train"] else T * d}
        moved = L * d * size + T * d * size + 8 * L
        if case["train"]:  # the rows and the cells' gradients in, the rows' and gates' out
            moved += T * d * size + L * d * size + 4 * L
        return {"bytes": moved, "flops": (5 if case["train"] else 2) * L * d}
    if op == "quantize":
        size = 4 if case["dtype"] == "f32" else 2
        if case["rows"]:
            n, scales = case["rows"] * case["inner"], case["rows"] * -(-case["inner"] // BLOCK)
        else:
            n = case["paths"] * case["inner"] * case["outer"]
            scales = case["paths"] * -(-case["inner"] // BLOCK) * -(-case["outer"] // BLOCK)
        return {"bytes": n * size + n + 4 * scales, "flops": 3 * n}
    E, K, N, rows = case["paths"], case["inner"], case["outer"], case["rows"]
    if op == "linear":
        used = int((_loads(case) > 0).sum())
        k_blocks, n_blocks = -(-K // BLOCK), -(-N // BLOCK)
        return {"bytes": rows * (K + 4 * k_blocks + 2 * N) + used * (N * K + 4 * k_blocks * n_blocks)
                + 4 * E, "flops": 2 * rows * N * K}
    return {"bytes": 2 * rows * (N + K) + E * N * K * (4 if case["wide"] else 2) + 4 * E,
            "flops": 2 * rows * N * K}


# -------------------------------------------------------------------------- values in 64 bits
def exact(case, seed):
    """What ``run`` returns, from the definitions in 64 bits."""
    state = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](case, state)


def _exact_routes(picks, paths):
    """(cell, pick number, row) of all routes: counted path by path."""
    flat = picks.reshape(-1).cpu().numpy().astype(np.int64)
    rows = np.concatenate([np.nonzero(flat == e)[0] for e in range(paths)])
    routes = torch.from_numpy(rows).cuda()
    k = picks.size(1)
    return routes // k, routes % k, torch.arange(routes.numel(), device="cuda")


def _exact_block_codes(x, dims):
    """x (a multiple of 128 along `dims` after padding with zeros) -> code values and scales."""
    pads, shape = [], list(x.shape)
    for dim in range(x.dim() - 1, -1, -1):
        pads += [0, -shape[dim] % BLOCK if dim in dims else 0]
    padded = torch.nn.functional.pad(x.double(), pads)
    split, inside = [], []
    for dim, n in enumerate(padded.shape):
        if dim in dims:
            inside.append(len(split) + 1)
            split += [n // BLOCK, BLOCK]
        else:
            split.append(n)
    scales = padded.reshape(split).abs().amax(inside, keepdim=True)
    scales = torch.where(scales < AMAX_FLOOR, AMAX_FLOOR, scales) / E4M3_MAX
    scaled = padded.reshape(split) / scales
    # e4m3: 3 bits behind the leading one, the smallest step 2^-9, ties to even
    step = torch.exp2(torch.floor(torch.log2(scaled.abs().clamp(min=2.0 ** -6))) - 3)
    codes = (torch.round(scaled / step) * step).reshape(padded.shape)
    for dim in dims:
        codes = codes.narrow(dim, 0, shape[dim])
    return codes, scales.reshape([n // BLOCK if d in dims else n
                                  for d, n in enumerate(padded.shape)])


def _exact_sort(case, state):
    cell, pick, row = _exact_routes(state["picks"], case["paths"])
    x = state["cells"].double()
    rows = torch.zeros(case["cells"] * case["k"], case["width"], dtype=torch.float64,
                       device="cuda")
    rows[row] = x[cell]
    if case["fp8"]:
        return (None, None, *_exact_block_codes(rows, (1,)))
    if not case["train"]:
        return None, None, rows
    grad = torch.zeros_like(x).index_add_(0, cell, state["row_grads"].double()[row])
    return None, None, rows, grad


def _exact_unsort(case, state):
    cell, pick, row = _exact_routes(state["picks"], case["paths"])
    gates, rows = state["gates"].double(), state["rows"].double()
    weight = gates[cell, pick].unsqueeze(1)
    out = torch.zeros(case["cells"], case["width"], dtype=torch.float64, device="cuda")
    out.index_add_(0, cell, rows[row] * weight)
    if not case["train"]:
        return out
    back = state["cell_grads"].double()[cell]
    rows_grad = torch.zeros_like(rows)
    rows_grad[row] = back * weight
    gates_grad = torch.zeros_like(gates)
    gates_grad[cell, pick] = torch.einsum("rd,rd->r", back, rows[row])
    return out, rows_grad, gates_grad


def _exact_quantize(case, state):
    if case["rows"]:
        return _exact_block_codes(state["rows"], (1,))
    return _exact_block_codes(state["weights"].transpose(1, 2), (1, 2))


def _exact_linear(case, state):
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    K, N = case["inner"], case["outer"]
    block_k = torch.arange(K, device="cuda") // BLOCK
    block_n = torch.arange(N, device="cuda") // BLOCK
    first = 0
    for e, load in enumerate(_loads(case).tolist()):
        if load:
            at = slice(e * state["slot"], e * state["slot"] + load) if state["slot"] else \
                slice(first, first + load)
            x = state["rows"][at].double() * state["row_scales"][at].double()[:, block_k]
            w = state["weights"][e].double()
            w *= state["weight_scales"][e].double()[block_n][:, block_k]
            y = x @ w.t()
            out[at] = torch.relu(y) if case["relu"] else y
        first += load
    return out


def _exact_wgrad(case, state):
    out = torch.zeros(case["paths"], case["outer"], case["inner"], dtype=torch.float64,
                      device="cuda")
    first = 0
    for e, load in enumerate(_loads(case).tolist()):
        at = slice(first, first + load)
        out[e] = state["grads"][at].double().t() @ state["rows"][at].double()
        first += load
    return out


_EXACT = {"sort": _exact_sort, "unsort": _exact_unsort, "quantize": _exact_quantize,
          "linear": _exact_linear, "wgrad": _exact_wgrad}
