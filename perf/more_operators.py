"""The operators around 8-bit projections and the choice of tokens: what is measured of them.

Four operators, each in its plain form (elementary torch operations) and as the calls a user makes of libtkcuda:

  norm      tk_add_rmsnorm_fp8  a layer's output added to the residual stream, its RMS norm, and that in 8 bits
  quantise  tk_fp8_quantize     rows in groups of 128, or a weight in blocks of 128 x 128, in 8 bits
  matmul    tk_fp8_matmul       8-bit rows times an 8-bit weight, with a scale for each block of 128
  sample    tk_sample_tokens    a token of each row of logits: temperature, top-k, top-p, min-p, given random numbers

8 bits are e4m3 codes with an f32 scale: value = code * scale, scale = (largest magnitude of the group) / 448.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
CODES = torch.float8_e4m3fn
GROUP, LARGEST, LEAST, EPS = 128, 448.0, 2.0 ** -126, 1e-5


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of the 4096-wide model in the framework's own f32 activations: latency
        dict(name="norm decode 4 f32", op="norm", rows=4, dim=4096, dtype="f32", residual=True),
        # a whole prompt of it
        dict(name="norm prompt 8192 bf16", op="norm", rows=8192, dim=4096, dtype="bf16", residual=True),
        # the intermediate activations of a chunk of a prompt, before the down projection
        dict(name="quantise rows 2048 bf16", op="quantise", rows=2048, dim=14336, block=1, dtype="bf16"),
        # a gate projection when a model is loaded
        dict(name="quantise weight f32", op="quantise", rows=14336, dim=4096, block=128, dtype="f32"),
        # one token through the same projection
        dict(name="matmul 1 x 4096 x 14336", op="matmul", m=1, k=4096, n=14336, dtype="f32"),
        # a decode batch through the down projection
        dict(name="matmul 32 x 14336 x 4096", op="matmul", m=32, k=14336, n=4096, dtype="bf16"),
        # a decode batch through the output head of a large vocabulary, logits in f32
        dict(name="matmul 48 x 4096 x 128256", op="matmul", m=48, k=4096, n=128256, dtype="f32"),
        # odd sizes: the tokens of a few ragged prompts, a k that ends inside a block, an odd number of columns
        dict(name="matmul 777 x 2000 x 5003", op="matmul", m=777, k=2000, n=5003, dtype="f16"),
        # a whole prompt
        dict(name="matmul 8192 x 4096 x 14336", op="matmul", m=8192, k=4096, n=14336, dtype="bf16"),
        # one user's next token: latency
        dict(name="sample 1 x 128256 f32", op="sample", rows=1, vocab=128256, dtype="f32", filters="all"),
        # a decode batch whose users asked for different things, 16-bit logits with many ties
        dict(name="sample 64 x 128256 bf16", op="sample", rows=64, vocab=128256, dtype="bf16", filters="mixed"),
        # a large batch over a smaller vocabulary, plain sampling
        dict(name="sample 256 x 32000 f32", op="sample", rows=256, vocab=32000, dtype="f32", filters="none"),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _width(rng, lo, hi):
    """A width as models have them: mostly a multiple of 128, at times any number."""
    w = _spread(rng, lo, hi)
    return rng.choice([w, max(16, w // 16 * 16), *[max(128, w // 128 * 128)] * 4])


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "quantise", "matmul", "sample")}
    while True:
        op = rng.choice(["norm", "quantise", "matmul", "matmul", "matmul", "sample", "sample"])
        dtype = rng.choice(["f32", "f16", "bf16"])
        if op == "norm":
            case = dict(op=op, rows=_spread(rng, 1, 8192), dim=_width(rng, 256, 16384), dtype=dtype,
                        residual=rng.random() < 0.7)
        elif op == "quantise":
            case = dict(op=op, rows=_spread(rng, 1, 16384), dim=_width(rng, 128, 16384), block=rng.choice([1, 1, 128]),
                        dtype=dtype)
        elif op == "matmul":
            case = dict(op=op, m=_spread(rng, 1, rng.choice([16, 256, 8192])), k=_width(rng, 256, 16384),
                        n=_width(rng, 64, rng.choice([16384, 131072])), dtype=dtype)
        else:
            case = dict(op=op, rows=_spread(rng, 1, 256), vocab=rng.choice([32000, 50257, 128256, _spread(rng, 100, 262144)]),
                        dtype=dtype, filters=rng.choice(["all", "mixed", "mixed", "none"]))
        if _cost(case) <= most[op]:
            return case


def _blocks(n):
    return -(-n // GROUP)


def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["dim"]
        moved = n * SIZE[case["dtype"]] * (3 if case["residual"] else 1) + n
        return {"bytes": moved + 4 * case["dim"] + 4 * case["rows"] * _blocks(case["dim"]), "flops": 8 * n}
    if op == "quantise":
        n = case["rows"] * case["dim"]
        scales = -(-case["rows"] // case["block"]) * _blocks(case["dim"])
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + 4 * scales, "flops": 3 * n}
    if op == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        scales = (m + _blocks(n)) * _blocks(k)
        return {"bytes": m * k + n * k + 4 * scales + m * n * SIZE[case["dtype"]], "flops": 2 * m * n * k}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * SIZE[case["dtype"]] + 28 * case["rows"], "flops": 6 * n}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _activations(gen, rows, dim, dtype):
    """Rows of a trained model: channels of different size, a few of them by much."""
    size = torch.exp(0.5 * _normal(gen, (dim,)))
    size[:: max(1, dim // 5)] *= 12.0
    return (_normal(gen, (rows, dim)) * size).to(dtype)


def _row(dim):
    """Bytes from one row of codes to the next: on the 16-byte boundary that the product asks for."""
    return -(-dim // 16) * 16


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = globals()["_prepare_" + case["op"]](case, gen)
    s["case"] = case
    if own:
        ops, device = _framework()
        s.update(ops=ops, device=device)
    return s


def _prepare_norm(case, gen):
    rows, dim, kind = case["rows"], case["dim"], TYPES[case["dtype"]]
    s = dict(x=_activations(gen, rows, dim, kind), weight=1.0 + 0.1 * _normal(gen, (dim,)),
             codes=torch.empty((rows, _row(dim)), dtype=torch.uint8, device="cuda"),
             scales=torch.empty((rows, _blocks(dim)), dtype=torch.float32, device="cuda"), residual=None, sum=None)
    if case["residual"]:
        s.update(residual=_activations(gen, rows, dim, kind), sum=torch.empty((rows, dim), dtype=kind, device="cuda"))
    return s


def _prepare_quantise(case, gen):
    rows, dim, block = case["rows"], case["dim"], case["block"]
    x = _activations(gen, rows, dim, TYPES[case["dtype"]])
    return dict(x=x, codes=torch.empty((rows, _row(dim)), dtype=torch.uint8, device="cuda"),
                scales=torch.empty((-(-rows // block), _blocks(dim)), dtype=torch.float32, device="cuda"))


def _prepare_matmul(case, gen):
    m, k, n = case["m"], case["k"], case["n"]
    s = {}
    for name, rows, block in (("a", m, 1), ("w", n, GROUP)):
        x = _activations(gen, rows, k, torch.float32)
        codes, s[name + "_scales"] = _in_8_bits(x if name == "a" else x * k ** -0.5, block)
        held = torch.zeros((rows, _row(k)), dtype=torch.uint8, device="cuda")
        held[:, :k] = codes.view(torch.uint8)
        s[name] = held
        del x, codes
    s["out"] = torch.empty((m, n), dtype=TYPES[case["dtype"]], device="cuda")
    return s


def _prepare_sample(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    f32 = dict(generator=gen, device="cuda", dtype=torch.float32)
    # a broad body, some tokens of the context well above it, and tokens that a grammar forbids
    logits = _normal(gen, (rows, vocab)) * (1.0 + 1.5 * torch.rand((rows, 1), **f32)) - 2.0
    near = torch.randint(0, vocab, (rows, min(40, vocab)), generator=gen, device="cuda")
    logits.scatter_add_(1, near, 4.0 + 8.0 * torch.rand(near.shape, **f32))
    logits[:, vocab - vocab // 100:] = -torch.inf
    s = dict(logits=logits.to(TYPES[case["dtype"]]), random=torch.rand((rows,), **f32), temperature=None, top_k=None,
             top_p=None, min_p=None, tokens=torch.zeros((rows,), dtype=torch.int32, device="cuda"),
             kept=torch.zeros((rows,), dtype=torch.int32, device="cuda"))
    if case["filters"] != "none":
        s.update(temperature=0.5 + torch.rand((rows,), **f32), top_p=0.8 + 0.19 * torch.rand((rows,), **f32),
                 top_k=torch.randint(1, 200, (rows,), generator=gen, device="cuda", dtype=torch.int32),
                 min_p=0.1 * torch.rand((rows,), **f32))
    if case["filters"] == "mixed":  # a row's filter is off, or the row is greedy, where its user did not ask
        for name, off, share in (("temperature", 0.0, 0.1), ("top_k", 0, 0.6), ("top_p", 1.0, 0.3), ("min_p", 0.0, 0.7)):
            s[name][torch.rand((rows,), **f32) < share] = off
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    return globals()[("_own_" if own else "_plain_") + s["case"]["op"]](s)


def _in_8_bits(y, block):
    """(codes, scales) of y [rows, dim] in groups of `block` x 128."""
    rows, dim = y.shape
    down, across = -(-rows // block), _blocks(dim)
    padded = torch.nn.functional.pad(y, (0, across * GROUP - dim, 0, down * block - rows))
    tiles = padded.view(down, block, across, GROUP)
    scales = (tiles.abs().amax((1, 3)) / tiles.new_full((), LARGEST)).clamp(min=LEAST)
    codes = (tiles / scales[:, None, :, None]).view(down * block, across * GROUP)[:rows, :dim]
    return codes.to(CODES), scales


def _plain_norm(s):
    y = s["x"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    normed = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * s["weight"]
    codes, scales = _in_8_bits(normed, 1)
    return [codes, scales] if s["residual"] is None else [codes, scales, y.to(s["x"].dtype)]


def _plain_quantise(s):
    return list(_in_8_bits(s["x"].float(), s["case"]["block"]))


def _plain_matmul(s):
    k, n = s["case"]["k"], s["case"]["n"]
    a, w = (s[x][:, :k].view(CODES).float() for x in "aw")
    a = a * s["a_scales"].repeat_interleave(GROUP, 1)[:, :k]
    w = w * s["w_scales"].repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return (a @ w.t()).to(s["out"].dtype)


def _plain_sample(s):
    """In 64 bits: tokens are whole numbers that go by where a sum passes another."""
    l = s["logits"].double()
    rows, vocab = l.shape
    heat = torch.ones(rows, device="cuda") if s["temperature"] is None else s["temperature"]
    greedy = heat <= 0
    heat = torch.where(greedy, torch.ones_like(heat), heat).double()[:, None]
    top, order = l.sort(dim=-1, descending=True, stable=True)  # ties: the lowest index first
    p = torch.exp((top - top[:, :1]) / heat)
    rank = torch.arange(vocab, device="cuda")
    keep = torch.isfinite(top)
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] <= 0, torch.full_like(s["top_k"], vocab), s["top_k"])
        keep = keep & (rank < k[:, None])
    p = torch.where(keep, p, torch.zeros_like(p))
    if s["top_p"] is not None:
        before = p.cumsum(-1) - p
        wanted = s["top_p"].double()[:, None] * p.sum(-1, keepdim=True)
        keep = keep & ((before < wanted) | (s["top_p"] >= 1)[:, None])
    if s["min_p"] is not None:
        keep = keep & (p >= s["min_p"].double()[:, None])
    keep = keep & ((rank == 0) | ~greedy[:, None])
    p = torch.where(keep, p, torch.zeros_like(p))
    weight = torch.zeros_like(p).scatter_(1, order, p)
    passed = weight.cumsum(-1)
    token = (passed <= s["random"].double()[:, None] * passed[:, -1:]).sum(-1)
    return [token.to(torch.int32), keep.sum(-1).to(torch.int32)]


# ---- the framework's calls ---------------------------------------------------------------------------------------

STREAM = 1  # cudaStreamLegacy: the stream that torch works on by default
_kept = {}


def _framework():
    if not _kept:
        path = os.path.join(os.getcwd(), "tiny-kernel_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import tiny_kernel
        from tiny_kernel import ops
        _kept.update(ops=ops, device=tiny_kernel.init(torch.cuda.current_device()))
    return _kept["ops"], _kept["device"]


def _own_norm(s):
    case, codes = s["case"], s["codes"]
    s["ops"].add_rmsnorm_fp8(s["device"], s["x"], s["residual"], s["weight"], s["sum"], codes, s["scales"], case["rows"],
                             case["dim"], EPS, case["dtype"], codes_stride=codes.shape[1], stream=STREAM, sync=False)
    out = [codes[:, : case["dim"]].view(CODES), s["scales"]]
    return out if s["sum"] is None else out + [s["sum"]]


def _own_quantise(s):
    case, codes = s["case"], s["codes"]
    s["ops"].fp8_quantize(s["device"], s["x"], codes, s["scales"], case["rows"], case["dim"], case["block"], case["dtype"],
                          codes_stride=codes.shape[1], stream=STREAM, sync=False)
    return [codes[:, : case["dim"]].view(CODES), s["scales"]]


def _own_matmul(s):
    case = s["case"]
    s["ops"].fp8_matmul(s["device"], s["a"], s["a_scales"], s["w"], s["w_scales"], s["out"], case["m"], case["k"], case["n"],
                        case["dtype"], a_stride=s["a"].shape[1], w_stride=s["w"].shape[1], stream=STREAM, sync=False)
    return s["out"]


def _own_sample(s):
    case = s["case"]
    s["ops"].sample_tokens(s["device"], s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["random"],
                           s["tokens"], s["kept"], case["rows"], case["vocab"], case["dtype"], stream=STREAM, sync=False)
    return [s["tokens"], s["kept"]]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def _exact_8_bits(y, block):
    """What the codes stand for before they are rounded, and the scales, strip by strip of 128 columns."""
    codes, scales = [], []
    for strip in y.split(GROUP, 1):
        largest = torch.cat([rows.abs().max().view(1) for rows in strip.split(block)]) if block > 1 else strip.abs().max(-1).values
        scales.append(torch.maximum(largest / LARGEST, torch.full_like(largest, LEAST)))
        each = scales[-1].repeat_interleave(block)[: len(strip)]
        codes.append(strip / each[:, None])
    return torch.cat(codes, 1), torch.stack(scales, 1)


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "quantise":
        return list(_exact_8_bits(s["x"].to(f64), case["block"]))
    if case["op"] == "norm":
        total = s["x"].to(f64) if s["residual"] is None else s["x"].to(f64).add(s["residual"].to(f64))
        size = torch.linalg.vector_norm(total, dim=-1, keepdim=True)
        y = total * (size * size / case["dim"] + EPS).rsqrt() * s["weight"].to(f64)
        out = list(_exact_8_bits(y, 1))
        return out if s["residual"] is None else out + [total]
    if case["op"] == "matmul":
        # block by block, the scales applied to each block's sums
        m, k, n = case["m"], case["k"], case["n"]
        total = torch.zeros((m, n), dtype=f64, device="cuda")
        column = torch.arange(n, device="cuda") // GROUP
        for b in range(_blocks(k)):
            at = slice(b * GROUP, min(k, (b + 1) * GROUP))
            part = s["a"][:, at].view(CODES).to(f64) @ s["w"][:, at].view(CODES).to(f64).T
            part *= s["a_scales"][:, b, None].to(f64)
            total.addcmul_(part, s["w_scales"][column, b].to(f64).expand(m, n))
        return total
    # tokens, row by row: the filters one after the other over ranked logits
    host = {x: None if s[x] is None else s[x].double().cpu().numpy()
            for x in ("logits", "temperature", "top_k", "top_p", "min_p", "random")}
    tokens, kept = [], []
    for r, l in enumerate(host["logits"]):
        order = np.argsort(-l, kind="stable")
        order = order[np.isfinite(l[order])]
        heat = 1.0 if host["temperature"] is None else host["temperature"][r]
        if heat <= 0:
            order, heat = order[:1], 1.0
        if host["top_k"] is not None and host["top_k"][r] > 0:
            order = order[: int(host["top_k"][r])]
        p = np.exp((l[order] - l[order[0]]) / heat)
        least = 0.0 if host["min_p"] is None else host["min_p"][r]
        count = len(p)
        if host["top_p"] is not None and host["top_p"][r] < 1:
            count = min(count, 1 + int(np.searchsorted(np.cumsum(p), host["top_p"][r] * p.sum())))
        count = min(count, int((p >= least).sum()))
        at = np.sort(order[:count])
        passed = np.cumsum(np.exp((l[at] - l[order[0]]) / heat))
        i = int(np.searchsorted(passed, host["random"][r] * passed[-1], side="right"))
        tokens.append(at[min(i, count - 1)])
        kept.append(count)
    return [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (tokens, kept)]
