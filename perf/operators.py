"""The expert operators of one GPU, as cases that can be timed and compared.

Where a GPU holds the experts that its tokens go to, their rows need no transport: the tokens are
sorted by expert, multiplied, and brought back.  The cases are calls of these operators:

* ``permute``       sort the routing by expert and copy every token to the rows of its experts;
                    with ``grad`` the gradient of the tokens from that of the rows as well
* ``permute_int8``  the same with the tokens quantised to 8-bit integers on the way
* ``unpermute``     the weighted sum of each token's rows; with ``grad`` the gradients of the rows
                    and of the weights as well
* ``quantize``      rows to 8-bit integers, one scale per row
* ``gemm``          the experts' product of 8-bit integers, one scale per token and per channel
* ``layer``         all of them in a row: the experts of an int8 MoE layer

Keys of a case:

  op                      one of the above
  experts, topk, hidden   of the model; ``ffn`` the width of an expert (gemm, layer)
  tokens                  tokens of the pass
  dtype                   of the tokens, rows and results: "bf16", "fp16" or "fp32"
  zipf                    exponent of the expert popularity, 0 for uniform routing
  away                    share of the routing that names no expert of this GPU
  capacity                rows that an expert takes at most (rows are then [experts, capacity]),
                          0 for as many as it gets, one expert's rows after the other's
  grad                    permute, unpermute: forward and backward
  padded                  gemm, quantize: rows as [experts, capacity] with a count each, otherwise
                          one expert's rows after the other's
  up                      gemm: gate and up projection with SwiGLU, otherwise the down projection
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (experts, top-k, hidden, expert width): Mixtral-8x7B, Qwen3-30B-A3B, DeepSeek-V3's experts on one
# of eight GPUs, DeepSeek-V2-Lite.
MODELS = [(8, 2, 4096, 14336), (128, 8, 2048, 768), (32, 8, 7168, 2048), (64, 6, 2048, 1408)]
TINY = 1e-30  # smallest largest value of a row that its scale follows


def _permute(op, experts, topk, hidden, tokens, dtype="bf16", zipf=0.0, away=0.0, capacity=0,
             grad=False):
    return {"op": op, "experts": experts, "topk": topk, "hidden": hidden, "tokens": tokens,
            "dtype": dtype, "zipf": zipf, "away": away, "capacity": capacity, "grad": grad}


def _quantize(rows, width, dtype="bf16", experts=1, padded=False):
    return {"op": "quantize", "experts": experts, "rows": rows, "width": width, "dtype": dtype,
            "padded": padded}


def _gemm(model, tokens, up, dtype="bf16", zipf=0.0, padded=False):
    experts, topk, hidden, ffn = model
    return {"op": "gemm", "experts": experts, "topk": topk, "hidden": hidden, "ffn": ffn,
            "tokens": tokens, "up": up, "dtype": dtype, "zipf": zipf, "padded": padded}


def _layer(model, tokens, dtype="bf16", zipf=0.0):
    experts, topk, hidden, ffn = model
    return {"op": "layer", "experts": experts, "topk": topk, "hidden": hidden, "ffn": ffn,
            "tokens": tokens, "dtype": dtype, "zipf": zipf}


def listed() -> list[dict]:
    mixtral, qwen3, v3share, v2lite = MODELS
    return [
        # Decode of a single sequence: the latency of sorting eight entries and copying one token.
        {"name": "permute-1", **_permute("permute", 256, 8, 7168, 1)},
        # A training step's way to the experts and the gradient back, with a capacity that skewed
        # experts overflow.
        {"name": "permute-train-4096", **_permute("permute", 64, 6, 2048, 4096, zipf=0.6,
                                                  capacity=512, grad=True)},
        # A ragged decode batch on its way to int8 experts, three quarters of which are elsewhere.
        {"name": "permute-int8-77", **_permute("permute_int8", 256, 8, 7168, 77, away=0.75)},
        # Prefill.
        {"name": "permute-int8-4096", **_permute("permute_int8", 256, 8, 7168, 4096)},
        # Decode of a small batch in half precision: the way back.
        {"name": "unpermute-16", **_permute("unpermute", 128, 8, 2048, 16, dtype="fp16")},
        # A training step's way back and the gradients of rows and weights.
        {"name": "unpermute-train-4095", **_permute("unpermute", 256, 8, 7168, 4095, grad=True)},
        # The intermediate of a decode batch.
        {"name": "quantize-61", **_quantize(488, 768)},
        # Expert weights as they are loaded: a row for each output channel, in 32 bits.
        {"name": "quantize-load", **_quantize(28672, 4096, dtype="fp32")},
        # Decode of a small batch: nearly every row meets an expert of its own.
        {"name": "gemm-down-3", **_gemm(qwen3, 3, False)},
        # The batch layout of the all-to-all: a row count for each expert, skewed.
        {"name": "gemm-up-1000", **_gemm(v2lite, 1000, True, zipf=1.2, padded=True)},
        # Prefill through few wide experts.
        {"name": "gemm-up-4096", **_gemm(mixtral, 4096, True)},
        # The experts of one GPU in a full decode step of a large deployment.
        {"name": "layer-1021", **_layer(v3share, 1021)},
    ]


def draw(rng: random.Random) -> dict:
    op = rng.choice(["permute", "permute_int8", "unpermute", "quantize", "gemm", "layer"])
    zipf = rng.choice([0.0, 0.0, 0.6, 1.2])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "quantize":
        width = rng.choice([768, 1408, 2048, 7168, 14336, _log_uniform(rng, 16, 16384)])
        experts = rng.choice([1, 1, 8, 64])
        rows = _log_uniform(rng, 1, max(1, min(32768, (1 << 27) // width // experts)))
        return _quantize(rows, width, rng.choice(["bf16", "fp16", "fp32"]), experts, experts > 1)
    if op in ("gemm", "layer"):
        model = rng.choice(MODELS)
        tokens = _log_uniform(rng, 1, 2048 if op == "gemm" else 1024)
        if op == "layer":
            return _layer(model, tokens, dtype, zipf)
        return _gemm(model, tokens, rng.random() < 0.5, dtype, zipf, rng.random() < 0.5)
    experts, topk, hidden = rng.choice([(8, 2, 4096), (128, 8, 2048), (256, 8, 7168), (64, 6, 2048)])
    if rng.random() < 0.3:
        hidden = _log_uniform(rng, 64, 4096)
    if op != "permute_int8" and rng.random() < 0.25:
        dtype = "fp32"
    tokens = _log_uniform(rng, 1, 2047 if dtype == "fp32" else 4095)
    capacity = 0
    if rng.random() < 0.3:
        capacity = max(1, int(1.25 * tokens * topk / experts))
    return _permute(op, experts, topk, hidden, tokens, dtype, zipf, rng.choice([0.0, 0.0, 0.5]),
                    capacity, op != "permute_int8" and rng.random() < 0.5)


def _log_uniform(rng: random.Random, low: int, high: int) -> int:
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


# ------------------------------------------------------------------------- inputs ----


def _routing(case: dict, gen: torch.Generator) -> torch.Tensor:
    """[tokens, topk] int32, distinct experts per token; -1 for those of other GPUs."""
    m, experts, dev = case["tokens"], case["experts"], gen.device
    ranks = torch.arange(1, experts + 1, device=dev, dtype=torch.float32)
    u = torch.rand(m, experts, generator=gen, device=dev).clamp_(1e-20, 1.0)
    noise = -torch.log((-torch.log(u)).clamp_(min=1e-20))
    idx = (noise - case["zipf"] * torch.log(ranks)).topk(case["topk"], dim=1).indices
    if case.get("away"):
        there = torch.rand(m, case["topk"], generator=gen, device=dev) >= case["away"]
        idx = torch.where(there, idx, -1)
    return idx.to(torch.int32)


def _weights_int8(gen: torch.Generator, experts: int, rows: int, k: int):
    """int8 expert weights with a scale per channel, such that products keep their inputs' size."""
    dev = gen.device
    w = torch.empty(experts, rows, k, dtype=torch.int8, device=dev)
    for e in range(experts):
        v = torch.randn(rows, k, generator=gen, device=dev)
        w[e] = (v * 30).round_().clamp_(-127, 127).to(torch.int8)
    s = (0.5 + torch.rand(experts, rows, generator=gen, device=dev)) / (30 * math.sqrt(k))
    return w, s


def _tokens(gen: torch.Generator, rows: int, width: int, dtype: torch.dtype) -> torch.Tensor:
    """Activations: rows of different size, a few large columns."""
    dev = gen.device
    x = torch.randn(rows, width, generator=gen, device=dev)
    x *= torch.exp2(2 * torch.rand(rows, 1, generator=gen, device=dev) - 1)
    if width >= 256:
        x[:, :: width // 4] *= 8
    return x.to(dtype)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s: dict = dict(case)
    op = case["op"]
    if op == "quantize":
        E, rows, width = case["experts"], case["rows"], case["width"]
        s["x"] = _tokens(gen, E * rows, width, dtype)
        s["counts"] = None
        if case["padded"]:
            s["x"] = s["x"].view(E, rows, width)
            s["counts"] = torch.randint(0, rows + 1, (E,), generator=gen, device=dev,
                                        dtype=torch.int32)
        # The rows beyond an expert's count keep what the buffers hold.
        s["q"] = torch.zeros(s["x"].shape, dtype=torch.int8, device=dev)
        s["scale"] = torch.zeros(s["x"].shape[:-1], device=dev)
        return s
    m, topk, E, hidden = case["tokens"], case["topk"], case["experts"], case["hidden"]
    s["indices"] = _routing(case, gen)
    if op in ("gemm", "layer"):
        ffn = case["ffn"]
        if op == "layer":
            s["x"] = _tokens(gen, m, hidden, dtype)
            s["weights"] = torch.softmax(torch.randn(m, topk, generator=gen, device=dev), dim=-1)
            s["w13"], s["w13_scale"] = _weights_int8(gen, E, 2 * ffn, hidden)
            s["w2"], s["w2_scale"] = _weights_int8(gen, E, hidden, ffn)
            s["most"] = _most_rows(s)
            return s
        k, n = (hidden, ffn) if case["up"] else (ffn, hidden)
        s["w"], s["w_scale"] = _weights_int8(gen, E, 2 * n if case["up"] else n, k)
        s["counts"], s["offsets"], _ = _order(s["indices"], E, 0)
        s["most"] = _most_rows(s)
        shape = (E, m) if case["padded"] else (m * topk,)
        q = torch.randn(*shape, k, generator=gen, device=dev)
        s["xq"] = (q * 32).round_().clamp_(-127, 127).to(torch.int8)
        s["x_scale"] = (0.5 + torch.rand(*shape, generator=gen, device=dev)) / 32
        s["out"] = torch.zeros(*shape, n, dtype=dtype, device=dev)
        return s
    if op == "unpermute":
        cap = case["capacity"]
        s["counts"], s["offsets"], s["row_of"] = _order(s["indices"], E, cap)
        shape = (E, cap) if cap else (m * topk,)
        s["y"] = _tokens(gen, math.prod(shape), hidden, dtype).view(*shape, hidden)
        s["weights"] = torch.softmax(torch.randn(m, topk, generator=gen, device=dev), dim=-1)
        if case["grad"]:
            s["grad_out"] = torch.randn(m, hidden, generator=gen, device=dev).to(dtype)
        return s
    s["x"] = _tokens(gen, m, hidden, dtype)
    if case["grad"]:
        shape = (E, case["capacity"]) if case["capacity"] else (m * topk,)
        s["grad_rows"] = torch.randn(*shape, hidden, generator=gen, device=dev).to(dtype)
    return s


def _most_rows(s: dict) -> int:
    """Rows of the expert that has most: what a program that pads its experts sizes them for."""
    return int(torch.bincount(s["indices"].flatten().long(), minlength=1).max())


# -------------------------------------------------------------------- plain forms ----


def _order(indices: torch.Tensor, experts: int, capacity: int):
    """(counts [E], offsets [E + 1], row of every (token, k), -1 for none), in token order."""
    flat = indices.flatten().long()
    there = (flat >= 0) & (flat < experts)
    key = torch.where(there, flat, experts)
    perm = torch.argsort(key, stable=True)
    at = torch.empty_like(perm)
    at[perm] = torch.arange(flat.numel(), device=flat.device)
    n = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    n.index_add_(0, key, torch.ones_like(key))
    first = torch.cumsum(n, 0) - n
    row = at
    counts = n[:experts]
    offsets = first
    if capacity:
        pos = at - first[key]
        there = there & (pos < capacity)
        row = key * capacity + pos
        counts = counts.clamp(max=capacity)
        offsets = torch.arange(experts + 1, device=flat.device) * capacity
    row = torch.where(there, row, -1)
    return (counts.to(torch.int32), offsets.to(torch.int32),
            row.to(torch.int32).view(indices.shape))


def _token_of(row_of: torch.Tensor, rows: int) -> torch.Tensor:
    """Token of every row, -1 for a row without one."""
    m, topk = row_of.shape
    token = torch.full((rows + 1,), -1, dtype=torch.int64, device=row_of.device)
    row = row_of.flatten().long()
    token[torch.where(row < 0, rows, row)] = torch.arange(m * topk, device=row.device) // topk
    return token[:rows]


def _rows_shape(s: dict) -> tuple:
    if s["capacity"]:
        return s["experts"], s["capacity"]
    return (s["tokens"] * s["topk"],)


def _spread(x: torch.Tensor, token: torch.Tensor) -> torch.Tensor:
    """Row of x for every token number, zero for -1."""
    got = x[token.clamp(min=0)]
    return torch.where((token >= 0).view(-1, *[1] * (x.dim() - 1)), got, torch.zeros_like(got))


def _plain_quantize(x: torch.Tensor):
    v = x.float()
    amax = v.abs().amax(dim=-1).clamp(min=TINY)
    q = torch.round(v * (127.0 / amax).unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    return q, amax / 127.0


def _plain_gemm(s, xq, x_scale, w, w_scale, counts, offsets, padded, up, dtype):
    """[rows, n] of `dtype`; padded: rows beyond an expert's count are zero."""
    E, n_w, _ = w.shape
    n = n_w // 2 if up else n_w
    if not padded and xq.size(0) <= E:  # few rows: each with its own copy of its expert's weights
        e = _expert_of(offsets, xq.size(0))
        y = torch.bmm(w[e].float(), xq.float().unsqueeze(2)).squeeze(2)
        y = y * x_scale[:, None] * w_scale[e]
    else:
        if padded:
            a, a_scale = xq[:, : s["most"]], x_scale[:, : s["most"]]
        else:
            at = offsets[:E, None].long() + torch.arange(s["most"], device=w.device)
            at = at.clamp(max=xq.size(0) - 1)
            a, a_scale = xq[at], x_scale[at]
        y = torch.bmm(a.float(), w.float().transpose(1, 2))
        y = y * a_scale[:, :, None] * w_scale[:, None, :]
    if up:
        gate, value = y[..., :n], y[..., n:]
        y = gate / (1 + torch.exp(-gate)) * value
    y = y.to(dtype)
    if padded:
        live = torch.arange(s["most"], device=w.device) < counts[:, None]
        s["out"][:, : s["most"]] = torch.where(live[:, :, None], y, torch.zeros_like(y))
        return s["out"]
    if y.dim() == 2:
        return y
    e = _expert_of(offsets, xq.size(0))
    pos = torch.arange(xq.size(0), device=w.device) - offsets[e]
    return y[e, pos]


def _expert_of(offsets: torch.Tensor, rows: int) -> torch.Tensor:
    row = torch.arange(rows, device=offsets.device)
    return (row[:, None] >= offsets[None, 1:]).sum(1)


def _plain_sum(y, row_of, weights, dtype):
    picked = _spread(y.flatten(0, -2).float(), row_of.flatten().long())
    picked = picked.view(*row_of.shape, -1)
    if weights is not None:
        picked = picked * weights[:, :, None]
    return picked.sum(1).to(dtype)


def _plain(s: dict) -> dict:
    op, dtype = s["op"], DTYPES[s["dtype"]]
    if op == "quantize":
        q, scale = _plain_quantize(s["x"])
        if s["counts"] is not None:
            live = torch.arange(q.size(1), device=q.device) < s["counts"][:, None]
            q, scale = torch.where(live[:, :, None], q, 0), torch.where(live, scale, 0.0)
        return {"q": q, "scale": scale}
    if op == "gemm":
        return {"out": _plain_gemm(s, s["xq"], s["x_scale"], s["w"], s["w_scale"], s["counts"],
                                   s["offsets"], s["padded"], s["up"], dtype)}
    E = s["experts"]
    if op == "layer":
        counts, offsets, row_of = _order(s["indices"], E, 0)
        token = _token_of(row_of, row_of.numel())
        q, scale = _plain_quantize(s["x"])
        h = _plain_gemm(s, q[token], scale[token], s["w13"], s["w13_scale"], counts, offsets,
                        False, True, dtype)
        hq, h_scale = _plain_quantize(h)
        y = _plain_gemm(s, hq, h_scale, s["w2"], s["w2_scale"], counts, offsets, False, False,
                        dtype)
        return {"out": _plain_sum(y, row_of, s["weights"], dtype)}
    if op == "unpermute":
        out = {"out": _plain_sum(s["y"], s["row_of"], s["weights"], dtype)}
        if s["grad"]:
            y, g, w = s["y"].flatten(0, -2), s["grad_out"].float(), s["weights"]
            row = s["row_of"].flatten().long()
            each = (w[:, :, None] * g[:, None, :]).flatten(0, 1)  # of every (token, k)
            slot = _token_of(s["row_of"].view(-1, 1), y.size(0))
            out["grad_rows"] = _spread(each, slot).to(dtype).view(s["y"].shape)
            picked = _spread(y.float(), row).view(*s["row_of"].shape, -1)
            out["grad_weights"] = (picked * g[:, None, :]).sum(-1)
        return out
    counts, offsets, row_of = _order(s["indices"], E, s["capacity"])
    shape = _rows_shape(s)
    token = _token_of(row_of, math.prod(shape))
    out = {"counts": counts, "offsets": offsets, "row_of": row_of}
    if op == "permute_int8":
        q, scale = _plain_quantize(s["x"])
        out["rows"] = _spread(q, token).view(*shape, -1)
        out["scale"] = _spread(scale, token).view(shape)
        return out
    out["rows"] = _spread(s["x"], token).view(*shape, -1)
    if s["grad"]:
        out["grad_x"] = _plain_sum(s["grad_rows"], row_of, None, dtype)
    return out


# --------------------------------------------------------- the framework's operators ----


def _own(s: dict) -> dict:
    from pplx_kernels_b200.ops.expert_rows import (
        ExpertRows,
        permute_tokens,
        permute_tokens_int8,
        sort_by_expert,
        unpermute_tokens,
    )
    from pplx_kernels_b200.ops.grouped_gemm import grouped_gemm_int8
    from pplx_kernels_b200.ops.quant import quantize_rows_int8

    op, dtype, E = s["op"], DTYPES[s["dtype"]], s["experts"]
    if op == "quantize":
        q, scale = quantize_rows_int8(s["x"], counts=s["counts"], out=s["q"], out_scale=s["scale"])
        return {"q": q, "scale": scale}
    if op == "gemm":
        return {"out": grouped_gemm_int8(
            s["xq"], s["x_scale"], s["w"], s["w_scale"], s["counts"],
            offsets=None if s["padded"] else s["offsets"], swiglu=s["up"], out=s["out"],
            expected_rows=s["tokens"] * s["topk"])}
    if op == "layer":
        rows = sort_by_expert(s["indices"], E)
        q, scale = permute_tokens_int8(s["x"], rows)
        h = grouped_gemm_int8(q, scale, s["w13"], s["w13_scale"], rows.counts,
                              offsets=rows.offsets, swiglu=True, out_dtype=dtype)
        hq, h_scale = quantize_rows_int8(h)
        y = grouped_gemm_int8(hq, h_scale, s["w2"], s["w2_scale"], rows.counts,
                              offsets=rows.offsets, out_dtype=dtype)
        return {"out": unpermute_tokens(y, rows, s["weights"])}
    if op == "unpermute":
        rows = ExpertRows(s["counts"], s["offsets"], s["row_of"], s["capacity"])
        if not s["grad"]:
            return {"out": unpermute_tokens(s["y"], rows, s["weights"])}
        y, w = s["y"].detach().requires_grad_(), s["weights"].detach().requires_grad_()
        out = unpermute_tokens(y, rows, w)
        out.backward(s["grad_out"])
        return {"out": out.detach(), "grad_rows": y.grad, "grad_weights": w.grad}
    rows = sort_by_expert(s["indices"], E, capacity=s["capacity"])
    out = {"counts": rows.counts, "offsets": rows.offsets, "row_of": rows.row_of}
    rest = bool(s["away"] or s["capacity"])  # rows without a token are compared as well
    if op == "permute_int8":
        out["rows"], out["scale"] = permute_tokens_int8(s["x"], rows, zero_rest=rest)
        return out
    if not s["grad"]:
        out["rows"] = permute_tokens(s["x"], rows, zero_rest=rest)
        return out
    x = s["x"].detach().requires_grad_()
    got = permute_tokens(x, rows)
    got.backward(s["grad_rows"])
    out["rows"], out["grad_x"] = got.detach(), x.grad
    return out


def run(state: dict) -> dict:
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------- work, exact values ----


def work(case: dict) -> dict:
    op, size = case["op"], DTYPES[case["dtype"]].itemsize
    if op == "quantize":
        n = case["experts"] * case["rows"] * (0.5 if case["padded"] else 1)
        return {"bytes": n * (case["width"] * (size + 1) + 4), "flops": 3 * n * case["width"]}
    m, topk, E, hidden = case["tokens"], case["topk"], case["experts"], case["hidden"]
    if op in ("gemm", "layer"):
        ffn, touched = case["ffn"], _experts_touched(case)
        routed = m * topk
        if op == "layer":
            return {"bytes": touched * 3 * hidden * ffn + m * hidden * 2 * size + m * topk * 8,
                    "flops": 2 * 3 * routed * hidden * ffn}
        k, n = (hidden, ffn) if case["up"] else (ffn, hidden)
        n_w = 2 * n if case["up"] else n
        return {"bytes": touched * n_w * (k + 4) + routed * (k + 4 + n * size) + E * 4,
                "flops": 2 * routed * k * n_w}
    rows = m * topk * (1 - case["away"])  # that a token is copied to
    every = E * case["capacity"] if case["capacity"] else m * topk  # that the result has
    if case["capacity"]:
        rows = min(rows, every)
    table = m * topk * 4
    if op == "unpermute":
        n = {"bytes": (rows + m) * hidden * size + 2 * table, "flops": 2 * rows * hidden}
        if case["grad"]:
            n["bytes"] += (m + rows + every) * hidden * size + 3 * table
            n["flops"] += 3 * rows * hidden
        return n
    out = 1 if op == "permute_int8" else size
    n = {"bytes": m * hidden * size + every * hidden * out + 2 * table + E * 8,
         "flops": m * topk + (3 * m * hidden if op == "permute_int8" else 0)}
    if case["grad"]:
        n["bytes"] += (rows + m) * hidden * size + table
        n["flops"] += rows * hidden
    return n


def _experts_touched(case: dict) -> float:
    """Expected number of experts that get a token (with replacement where skewed)."""
    E, draws = case["experts"], case["tokens"] * case["topk"]
    if case["zipf"] == 0.0:
        return E * (1.0 - (1.0 - case["topk"] / E) ** case["tokens"])
    p = [1.0 / (e + 1) ** case["zipf"] for e in range(E)]
    return sum(1.0 - (1.0 - q / sum(p)) ** draws for q in p)


def exact(case: dict, seed: int) -> dict | None:
    """The floating outputs from their definitions in 64 bits, expert by expert and row by row.
    What is rounded to 8 bits (and, in the layer, to its type between the operators) is rounded
    here too: that is part of what the operators compute."""
    s = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "quantize":
        scale = s["x"].to(f64).abs().amax(-1).clamp(min=TINY) / 127
        if s["counts"] is not None:
            for e, n in enumerate(s["counts"].tolist()):
                scale[e, n:] = 0
        return {"q": None, "scale": scale}
    E, topk = case["experts"], case["topk"]
    if op == "gemm":
        out = torch.zeros(s["out"].shape, dtype=f64, device=s["out"].device)
        begin = 0
        for e, n in enumerate(s["counts"].tolist()):
            mine = (e, slice(0, n)) if case["padded"] else slice(begin, begin + n)
            begin += n
            out[mine] = _exact_product(s["xq"][mine], s["x_scale"][mine], s["w"][e],
                                       s["w_scale"][e], case["up"])
        return {"out": out}
    # The (token, k) entries that each expert gets, in their order.
    flat = s["indices"].flatten()
    entries = [(flat == e).nonzero().flatten() for e in range(E)]
    if op == "layer":
        x = s["x"].to(f64)
        out = torch.zeros_like(x)
        w = s["weights"].to(f64).flatten()
        xs = x.abs().amax(-1).clamp(min=TINY) / 127
        xq = torch.round(x / xs[:, None])
        for e, mine in enumerate(entries):
            tok = mine // topk
            h = _exact_product(xq[tok], xs[tok], s["w13"][e], s["w13_scale"][e], True)
            h = h.to(s["x"].dtype).to(f64)
            hs = h.abs().amax(-1).clamp(min=TINY) / 127
            hq = torch.round(h / hs[:, None])
            y = _exact_product(hq, hs, s["w2"][e], s["w2_scale"][e], False)
            out.index_add_(0, tok, y.to(s["x"].dtype).to(f64) * w[mine, None])
        return {"out": out}
    cap = case["capacity"]
    if cap:
        entries = [mine[:cap] for mine in entries]
        row_at = torch.cat([e * cap + torch.arange(mine.numel(), device=flat.device)
                            for e, mine in enumerate(entries)])
    else:
        row_at = torch.arange(sum(mine.numel() for mine in entries), device=flat.device)
    entry = torch.cat(entries)  # of every row in row_at
    token = entry // topk
    shape = _rows_shape(case)
    hidden = case["hidden"]
    if op == "unpermute":
        y, w = s["y"].flatten(0, -2).to(f64), s["weights"].to(f64).flatten()
        out = torch.zeros(case["tokens"], hidden, dtype=f64, device=y.device)
        out.index_add_(0, token, y[row_at] * w[entry, None])
        if not case["grad"]:
            return {"out": out}
        g = s["grad_out"].to(f64)
        grad_rows = torch.zeros_like(y)
        grad_rows[row_at] = g[token] * w[entry, None]
        grad_w = torch.zeros(flat.numel(), dtype=f64, device=y.device)
        grad_w[entry] = (y[row_at] * g[token]).sum(-1)
        return {"out": out, "grad_rows": grad_rows.view(s["y"].shape),
                "grad_weights": grad_w.view(s["indices"].shape)}
    result: dict = {"counts": None, "offsets": None, "row_of": None, "rows": None}
    if op == "permute_int8":
        scale = torch.zeros(math.prod(shape), dtype=f64, device=flat.device)
        scale[row_at] = (s["x"].to(f64).abs().amax(-1).clamp(min=TINY) / 127)[token]
        result["scale"] = scale.view(shape)
        return result
    rows = torch.zeros(math.prod(shape), hidden, dtype=f64, device=flat.device)
    rows[row_at] = s["x"].to(f64)[token]
    result["rows"] = rows.view(*shape, hidden)
    if case["grad"]:
        g = s["grad_rows"].flatten(0, -2).to(f64)
        result["grad_x"] = torch.zeros(case["tokens"], hidden, dtype=f64, device=flat.device)
        result["grad_x"].index_add_(0, token, g[row_at])
    return result


def _exact_product(xq, x_scale, w, w_scale, up: bool) -> torch.Tensor:
    f64 = torch.float64
    y = xq.to(f64) @ w.to(f64).t() * x_scale.to(f64)[:, None] * w_scale.to(f64)[None, :]
    if not up:
        return y
    gate, value = y.chunk(2, dim=-1)
    return gate * torch.sigmoid(gate) * value
