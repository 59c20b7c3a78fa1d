"""The operators on 8-bit codes with a scale for each row, and what a user's program does with them.

* ``rows``: ``RowQuantizer.quantize``: int8 codes and one float32 scale for each row;
* ``product``: ``QuantizedMatrix.product``: rows of floats times a matrix that is held as int8 codes with a scale for each output channel;
* ``shared``: rows quantized once and multiplied by two matrices (``QuantizedMatrix.product_of_codes``), as projections of the same input are;
* ``grouped``: the product with one matrix for each group of consecutive rows (experts), group sizes ragged and known to the GPU alone;
* ``gradient``: ``QuantizedMatrix.input_gradient``: what the rows in front of a frozen matrix are trained with, for one matrix or several.

Sizes: 1 .. 16,384 rows, 64 .. 8,192 inputs and outputs, 2 .. 64 groups, odd ones among them; float32, float16 and bfloat16.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MOST_WORK = 8192**3


def listed():
    return [
        # the hidden state of one token: latency only
        {"name": "rows_one", "op": "rows", "n": 1, "inputs": 4096, "type": "bf16"},
        # a prompt's hidden states: bandwidth only
        {"name": "rows_16k", "op": "rows", "n": 16384, "inputs": 4096, "type": "bf16"},
        # rows that begin at any address
        {"name": "rows_odd", "op": "rows", "n": 5001, "inputs": 1001, "type": "f32"},
        # one token of one request: the matrix is read once, nothing else counts
        {"name": "product_token", "op": "product", "n": 1, "inputs": 4096, "outputs": 4096, "bias": False, "type": "bf16"},
        # one token of each of 16 requests
        {"name": "product_batch", "op": "product", "n": 16, "inputs": 4096, "outputs": 14336, "bias": False, "type": "f16"},
        # a short prompt, no size a multiple of a tile
        {"name": "product_odd", "op": "product", "n": 333, "inputs": 1001, "outputs": 1500, "bias": True, "type": "f32"},
        # long prompts
        {"name": "product_prompt", "op": "product", "n": 8192, "inputs": 8192, "outputs": 8192, "bias": False, "type": "bf16"},
        # two projections of the same rows
        {"name": "shared_two", "op": "shared", "n": 2048, "inputs": 4096, "outputs": 4096, "second": 1024, "type": "bf16"},
        # 32 experts, a prompt's rows sorted by expert; some rows go to none
        {"name": "grouped_prompt", "op": "grouped", "n": 8192, "inputs": 2048, "outputs": 1408, "groups": 32, "rest": 57, "type": "bf16"},
        # 64 experts, few rows each: their matrices are read once
        {"name": "grouped_token", "op": "grouped", "n": 128, "inputs": 2048, "outputs": 1024, "groups": 64, "rest": 0, "type": "f16"},
        # training in front of a frozen matrix, and in front of frozen experts
        {"name": "gradient_dense", "op": "gradient", "n": 4096, "inputs": 4096, "outputs": 4096, "groups": 0, "rest": 0, "type": "bf16"},
        {"name": "gradient_grouped", "op": "gradient", "n": 3001, "inputs": 1000, "outputs": 1536, "groups": 8, "rest": 5, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    w = _log(rng, lo, hi)
    return rng.choice([w, max(lo, w // 64 * 64), max(lo, w // 64 * 64)])


def draw(rng):
    op = rng.choice(["rows", "product", "product", "shared", "grouped", "grouped", "gradient"])
    c = {"op": op, "n": _log(rng, 1, 16384), "inputs": _width(rng, 64, 8192)}
    if op == "rows":
        return {**c, "type": rng.choice(["f32", "f16", "bf16"])}
    c["outputs"] = _width(rng, 64, 8192)
    if op == "product":
        c |= {"bias": rng.random() < 0.3, "type": rng.choice(["f32", "f16", "bf16", "bf16"])}
    elif op == "shared":
        c |= {"second": _width(rng, 64, 4096), "type": rng.choice(["f16", "bf16"])}
    else:
        dense = op == "gradient" and rng.random() < 0.5
        c |= {"groups": 0 if dense else rng.randint(2, 64), "rest": 0 if dense else rng.choice([0, rng.randint(0, c["n"] // 4)])}
        c["type"] = rng.choice(["f16", "bf16"])
        if not dense:
            c["inputs"], c["outputs"] = min(c["inputs"], 4096), min(c["outputs"], 4096)
            while c["groups"] * c["inputs"] * c["outputs"] > 1 << 28:
                c["groups"] = max(2, c["groups"] // 2)
                c["inputs"] = c["inputs"] // 2 if c["groups"] == 2 and c["groups"] * c["inputs"] * c["outputs"] > 1 << 28 else c["inputs"]
    while c["n"] * c["inputs"] * (c["outputs"] + c.get("second", 0)) > MOST_WORK // (2 if op == "gradient" else 1):
        c["n"] //= 2
        if "rest" in c:
            c["rest"] = min(c["rest"], c["n"] // 4)
    return c


def _counts(case):
    """How many rows each group has: skewed, as a router's choices are; the smallest groups often have none."""
    groups, n = case["groups"], case["n"] - case["rest"]
    rs = np.random.RandomState(1000 * groups + n)
    return rs.multinomial(n, rs.dirichlet(np.full(groups, 1.5)))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _activations(g, n, width, kind):
    """Rows of different sizes with a few large columns, as hidden states have; one row in 64 is padding."""
    columns = torch.ones(width, device="cuda")
    columns[torch.randperm(width, generator=g, device="cuda")[: max(1, width // 256)]] = 16.0
    x = _normal(g, n, width) * columns * torch.exp(0.5 * _normal(g, n, 1))
    x[37::64] = 0.0
    return x.to(TYPES[kind])


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, inputs, kind = case["n"], case["inputs"], case["type"]
    s = {"case": case}
    gradient = case["op"] == "gradient"
    if gradient:
        s["dy"] = (1e-3 * _normal(g, n, case["outputs"]) * torch.exp(_normal(g, n, 1))).to(TYPES[kind])
    else:
        s["x"] = _activations(g, n, inputs, kind)
    if case["op"] != "rows":
        groups = case.get("groups", 0)
        shapes = [(groups, case["outputs"], inputs) if groups else (case["outputs"], inputs)]
        shapes += [(case["second"], inputs)] if case["op"] == "shared" else []
        s["weights"] = [_normal(g, *shape) * (0.7 + 0.3 * _normal(g, *shape[:-1], 1).abs()) / math.sqrt(inputs) for shape in shapes]
        if groups:
            counts = _counts(case)
            s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
            s["most"] = max(1, int(counts.max()))
        s["bias"] = _normal(g, case["outputs"]) if case.get("bias") else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    # a program holds its matrices quantized, and the handles that keep them laid out
    weights = s.pop("weights", [])
    if own:
        import vq_b200 as vq

        s["rows"] = vq.RowQuantizer.fit()
        s["matrices"] = [vq.QuantizedMatrix.fit(w, gradient=case["op"] == "gradient") for w in weights]
    else:
        s["matrices"] = [_quantize(w) for w in weights]
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------
def _quantize(x):
    x = x.float()
    largest = x.abs().amax(-1, keepdim=True)
    scale = torch.where(largest > 0, (largest.double() / 127.0).float().clamp_min(2.0**-126), torch.ones_like(largest))
    codes = torch.round(x.double() / scale.double()).to(torch.int8)  # (in 64 bits: quotients next to a half)
    return codes, torch.where(largest > 0, scale, torch.zeros_like(scale))[..., 0]


def _by_group(s, rows, matrices):
    """rows[i] @ matrices[group of i]: the groups' rows padded to the largest group's number; 0 for rows of no group."""
    offsets = s["offsets"]
    at = torch.arange(rows.shape[0], device=rows.device)
    group = torch.searchsorted(offsets[1:], at, right=True)
    within = group < matrices.shape[0]
    place = torch.where(within, group, 0) * s["most"] + torch.where(within, at - offsets[torch.where(within, group, 0)], 0)
    padded = rows.new_zeros(matrices.shape[0] * s["most"], rows.shape[1])
    padded = padded.index_add(0, place, rows * within[:, None])
    y = torch.bmm(padded.view(matrices.shape[0], s["most"], -1), matrices)
    return y.flatten(0, 1)[place] * within[:, None], group.clamp(max=matrices.shape[0] - 1), within


def _plain_product(s, codes, scales, matrix):
    w, channel = matrix
    if "offsets" in s:
        y, group, within = _by_group(s, codes.float(), w.float().mT)
        y = y * scales[:, None] * channel[group] * within[:, None]
    else:
        y = (codes.float() @ w.float().T) * scales[:, None] * channel
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[s["case"]["type"]])


def _plain(s):
    op = s["case"]["op"]
    if op == "gradient":
        (w, channel), dy = s["matrices"][0], s["dy"].float()
        if "offsets" in s:
            dx = _by_group(s, dy, w.float() * channel[..., None])[0]
        else:
            dx = (dy * channel) @ w.float()
        return dx.to(s["dy"].dtype)
    codes, scales = _quantize(s["x"])
    if op == "rows":
        return codes, scales
    return [_plain_product(s, codes, scales, m) for m in s["matrices"]]


# ---- the framework's calls --------------------------------------------------------------------------------------
def _own(s):
    op, matrices = s["case"]["op"], s["matrices"]
    if op == "rows":
        return s["rows"].quantize(s["x"])
    if op == "gradient":
        return matrices[0].input_gradient(s["dy"], offsets=s.get("offsets"))
    if op == "shared":
        codes, scales = s["rows"].quantize(s["x"])
        return [m.product_of_codes(codes, scales, dtype=s["x"].dtype) for m in matrices]
    return [matrices[0].product(s["x"], bias=s["bias"], offsets=s.get("offsets"))]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op, n, k, size = case["op"], case["n"], case["inputs"], BYTES[case["type"]]
    if op == "rows":
        return {"bytes": n * k * (size + 1) + 4 * n, "flops": 3 * n * k}
    outputs = case["outputs"] + case.get("second", 0)
    matrices, used = 1, n
    if case.get("groups"):
        matrices, used = int((_counts(case) > 0).sum()), n - case["rest"]
    read, written = (outputs, k) if op == "gradient" else (k, outputs)
    nbytes = used * read * size + matrices * outputs * (k + 4) + n * written * size + (4 * outputs if case.get("bias") else 0)
    nbytes += 8 * (case["groups"] + 1) if case.get("groups") else 0
    return {"bytes": nbytes, "flops": 2 * used * k * outputs}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------
def _codes64(x):
    """(whole numbers, scale that they go with, that scale before its rounding to float32)"""
    x = x.to(torch.float64)
    real = x.abs().max(dim=-1).values / 127
    held = real.to(torch.float32).to(torch.float64)
    quotient = x / torch.where(held == 0, 1.0, held).unsqueeze(-1)
    return torch.round(quotient), held, real


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rows":
        codes, _, real = _codes64(s["x"])
        return codes.to(torch.int8), real
    gradient = case["op"] == "gradient"
    rows = s["dy"].double() if gradient else None
    if not gradient:
        codes, held, _ = _codes64(s["x"])
        rows = codes * held[:, None]
    results = []
    for w in s["weights"]:
        codes, held, _ = _codes64(w)
        matrix = codes * held[..., None]
        if "offsets" not in s:
            results.append(rows @ (matrix if gradient else matrix.t()))
        else:
            ends = s["offsets"].tolist()
            y = torch.zeros(case["n"], case["inputs"] if gradient else case["outputs"], dtype=torch.float64, device="cuda")
            for g, (a, b) in enumerate(zip(ends[:-1], ends[1:])):
                y[a:b] = rows[a:b] @ (matrix[g] if gradient else matrix[g].t())
            results.append(y)
        if s["bias"] is not None:
            results[-1] = results[-1] + s["bias"].double()
    return results[0] if gradient else results
