"""The serving-step operators over a key/value cache held in 4 bits: what is measured of them.

Four operators, each in its plain form (elementary torch operations) and as the calls a user makes of libtkcuda:

  slots   tk_paged_slots      block tables, positions and slots of a step from the requests' lengths
  qk      tk_qk_norm_rope     per-head RMS norm of queries and keys and the position rotation, in one pass
  write   tk_kv4_append, tk_kv4_gather   keys and values quantised into their slots, and read back
  attend  tk_kv4_attention    attention of 1..n query tokens per sequence over the pages of the 4-bit cache

The cache: codes u8 [block][kv_head][block_size][head_dim/2] (even dimension in the low nibble) and f16 (scale, offset)
pairs [block][kv_head][block_size][head_dim/group][2]; a value is code * scale + offset.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GOLDEN = 0.6180339887498949


# ---- cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of a mid-sized server: one new token for each of 64 requests
        dict(name="slots decode 64", op="slots", batch=64, ctx=4096, new_lo=1, new_hi=1, block=16),
        # prompts of many lengths admitted at once, into larger pages
        dict(name="slots prompts 512", op="slots", batch=512, ctx=0, new_lo=1, new_hi=2048, block=32),
        # a decode step of the 4096-wide, 32-head model in the framework's own f32 activations
        dict(name="qk decode 8 f32", op="qk", tokens=8, q_heads=32, kv_heads=8, dim=128, rot=128, dtype="f32",
             interleaved=False, norm=True),
        # a whole prompt of the same model
        dict(name="qk prompt 8192 bf16", op="qk", tokens=8192, q_heads=32, kv_heads=8, dim=128, rot=128, dtype="bf16",
             interleaved=False, norm=True),
        # small heads, half of each rotated, neighbouring pairs, no norm weights; a ragged number of tokens
        dict(name="qk odd 333 f16", op="qk", tokens=333, q_heads=14, kv_heads=2, dim=64, rot=32, dtype="f16",
             interleaved=True, norm=False),
        # the keys and values of a decode step of 64 requests
        dict(name="write decode 64 bf16", op="write", tokens=64, kv_heads=8, dim=128, group=128, block=16, dtype="bf16"),
        # those of a prompt, with two scales a head
        dict(name="write prompt 8192 f32", op="write", tokens=8192, kv_heads=8, dim=128, group=64, block=16, dtype="f32"),
        # one request with a short context: latency
        dict(name="attend 1 x 500 f32", op="attend", batch=1, ctx_lo=500, ctx_hi=500, queries=1, q_heads=32, kv_heads=8,
             dim=128, group=128, block=16, dtype="f32"),
        # a full decode batch with ragged contexts
        dict(name="attend 48 x 8192 bf16", op="attend", batch=48, ctx_lo=64, ctx_hi=8192, queries=1, q_heads=32,
             kv_heads=8, dim=128, group=128, block=16, dtype="bf16"),
        # one request with a long document
        dict(name="attend 1 x 131072 f16", op="attend", batch=1, ctx_lo=131072, ctx_hi=131072, queries=1, q_heads=32,
             kv_heads=8, dim=128, group=64, block=16, dtype="f16"),
        # five tokens a request (one sampled, four drafted), small heads, larger pages
        dict(name="attend drafts 16 x 5 f32", op="attend", batch=16, ctx_lo=300, ctx_hi=2500, queries=5, q_heads=16,
             kv_heads=4, dim=64, group=64, block=64, dtype="f32"),
        # a chunk of two prompts over what is cached of them; five query heads a key head
        dict(name="attend chunk 2 x 256 bf16", op="attend", batch=2, ctx_lo=1500, ctx_hi=4000, queries=256, q_heads=40,
             kv_heads=8, dim=128, group=128, block=16, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    most = max(max(w["bytes"], w["flops"] / 50) for w in map(work, listed()))
    while True:
        op = rng.choice(["slots", "qk", "write", "attend", "attend", "attend"])
        if op == "slots":
            new = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 17, 2048)])
            case = dict(op=op, batch=_spread(rng, 1, 512), ctx=rng.choice([0, _spread(rng, 1, 8192)]), new_lo=1,
                        new_hi=new, block=rng.choice([16, 32, 64]))
        elif op == "qk":
            dim = rng.choice([64, 80, 96, 128, 128, 256])
            kv = _spread(rng, 1, 16)
            case = dict(op=op, tokens=_spread(rng, 1, 8192), q_heads=kv * rng.choice([1, 2, 4, 5, 7, 8]), kv_heads=kv,
                        dim=dim, rot=rng.choice([dim, dim, dim // 2]), dtype=rng.choice(["f32", "f16", "bf16"]),
                        interleaved=rng.random() < 0.3, norm=rng.random() < 0.7)
        elif op == "write":
            dim, group = rng.choice([(64, 64), (128, 64), (128, 128), (256, 64), (256, 128)])
            case = dict(op=op, tokens=_spread(rng, 1, 8192), kv_heads=_spread(rng, 1, 16), dim=dim, group=group,
                        block=rng.choice([16, 32, 64]), dtype=rng.choice(["f32", "f16", "bf16"]))
        else:
            dim, group = rng.choice([(64, 64), (128, 64), (128, 128), (128, 128), (256, 64), (256, 128)])
            kv, hi = rng.choice([1, 2, 4, 8, 8]), _spread(rng, 1, 131072)
            queries = rng.choice([1, 1, 1, _spread(rng, 2, 16), _spread(rng, 17, 256)])
            case = dict(op=op, batch=_spread(rng, 1, 64), ctx_lo=rng.choice([1, max(1, hi // 2), hi]), ctx_hi=hi,
                        queries=queries, q_heads=kv * rng.choice([1, 2, 4, 5, 7, 8, 16]), kv_heads=kv, dim=dim,
                        group=group, block=rng.choice([16, 32, 64]), dtype=rng.choice(["f32", "f16", "bf16"]))
            if case["batch"] * hi * kv * dim > 48 * 8192 * 8 * 128:  # the padded cache of the plain form
                continue
            if case["batch"] * hi * queries * case["q_heads"] > 2 * 4000 * 256 * 40:  # its scores
                continue
        w = work(case)
        if max(w["bytes"], w["flops"] / 50) <= most:
            return case


def _lengths(n, lo, hi):
    """n whole numbers of lo..hi in no order, the first of them hi."""
    return [hi - int(((i * GOLDEN) % 1.0) * (hi - lo + 1)) for i in range(n)]


def _slot_lengths(case):
    ctx = _lengths(case["batch"], min(1, case["ctx"]), case["ctx"])
    return ctx, _lengths(case["batch"], case["new_lo"], case["new_hi"])


def _attend_lengths(case):
    """Context lengths with the step's own tokens among them: at least the query tokens."""
    return [max(n, case["queries"]) for n in _lengths(case["batch"], case["ctx_lo"], case["ctx_hi"])]


def work(case):
    op = case["op"]
    if op == "slots":
        ctx, new = _slot_lengths(case)
        b, t, bs = len(ctx), sum(new), case["block"]
        taken = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        used = sum(1 for c in ctx if c % bs)  # requests whose last page is read from the table
        return {"bytes": 8 * b + 4 * used + 4 * taken + 4 * taken + 8 * b + 8 * t, "flops": 4 * t}
    if op == "qk":
        n = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + case["tokens"] * (4 + 4 * case["rot"]), "flops": 8 * n}
    if op == "write":
        n = case["tokens"] * 2 * case["kv_heads"] * case["dim"]
        held = n // 2 + 4 * (n // case["group"])
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 2 * held + 8 * case["tokens"], "flops": 8 * n}
    lens, n, hk, hq, d = _attend_lengths(case), case["queries"], case["kv_heads"], case["q_heads"], case["dim"]
    seen = sum(n * l - n * (n - 1) // 2 for l in lens)  # pairs of a query token and a token that it sees
    held = sum(lens) * 2 * hk * (d // 2 + 4 * (d // case["group"]))
    pages = sum(-(-l // case["block"]) for l in lens)
    return {"bytes": held + 2 * len(lens) * n * hq * d * SIZE[case["dtype"]] + 4 * pages, "flops": 4 * d * hq * seen}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _normal(gen, shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantise(x, group, kind=torch.float64):
    """(codes, scale f16, offset f16) of x [..., dim] in groups along the last axis: in 64 bits, since a code is a value
    next to a border and the stored numbers go by the nearest."""
    g = x.to(kind).unflatten(-1, (x.shape[-1] // group, group))
    lo, hi = g.amin(-1), g.amax(-1)
    # a tensor as the divisor: torch multiplies by the reciprocal of a plain number
    scale = ((hi - lo) / lo.new_full((), 15.0)).float().clamp(max=65504.0).half()
    offset = lo.float().clamp(-65504.0, 65504.0).half()
    step = scale.to(kind)[..., None]
    codes = torch.where(step > 0, (g - offset.to(kind)[..., None]) / step, torch.zeros_like(g)).round().clamp(0, 15)
    return codes.flatten(-2).to(torch.uint8), scale, offset


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _values(packed, scales, group, dtype=torch.float32):
    """The values that codes [..., dim/2] and (scale, offset) pairs [..., dim/group, 2] stand for."""
    c = _unpack(packed).unflatten(-1, (-1, group)).to(dtype)
    return (c * scales[..., 0:1].to(dtype) + scales[..., 1:2].to(dtype)).flatten(-2)


def _keys_and_values(gen, shape, dtype=torch.float32):
    """Keys whose channels differ in size, a few by much (as trained models' do), and plain values."""
    size = torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device="cuda"))
    size[..., :: max(1, shape[-1] // 3)] *= 6.0
    return (_normal(gen, shape) * size).to(dtype), _normal(gen, shape, dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = globals()["_prepare_" + case["op"]](case, gen)
    s["case"] = case
    if own:
        s.update(_handles(case, s))
    return s


def _prepare_slots(case, gen):
    ctx, new = _slot_lengths(case)
    bs, b = case["block"], len(ctx)
    have = [-(-c // bs) for c in ctx]
    need = [-(-(c + n) // bs) for c, n in zip(ctx, new)]
    width, blocks = max(need) + 3, sum(need) + 17
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    used = sum(have)
    col, rows = torch.arange(width, device="cuda"), torch.tensor(have, device="cuda")
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    table[col[None, :] < rows[:, None]] = order[:used]
    tokens = sum(new) + 13  # a little more room than there are tokens, as a padded step has
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(context_lens=_ints(ctx), query_lens=_ints(new), free_blocks=order[used:].contiguous(),
                free_range=_ints([0, blocks - used]), table=table, blocks=blocks, tokens=tokens,
                kv_lens=torch.zeros(b, **i32), query_start=torch.zeros(b + 1, **i32),
                positions=torch.zeros(tokens, **i32), slots=torch.zeros(tokens, **i32), counts=torch.zeros(4, **i32))


def _prepare_qk(case, gen):
    t, hq, hk, d, rot = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"], case["rot"]
    kind, far = TYPES[case["dtype"]], 16384
    # the rows of a fused projection: queries, keys and values of a token next to each other
    qkv = _normal(gen, (t, (hq + 2 * hk) * d), kind)
    turn = torch.arange(far, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
        torch.tensor(500000.0, device="cuda", dtype=torch.float64),
        -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    weights = [1.0 + 0.1 * _normal(gen, (d,)) if case["norm"] else None for _ in range(2)]
    return dict(qkv=qkv, q_weight=weights[0], k_weight=weights[1], cos=turn.cos().float(), sin=turn.sin().float(),
                far=far, positions=torch.randint(0, far, (t,), generator=gen, device="cuda", dtype=torch.int32),
                q_out=torch.empty((t, hq, d), dtype=kind, device="cuda"),
                k_out=torch.empty((t, hk, d), dtype=kind, device="cuda"))


def _cache(blocks, hk, bs, d, group):
    u8 = dict(dtype=torch.uint8, device="cuda")
    f16 = dict(dtype=torch.float16, device="cuda")
    return dict(k_codes=torch.zeros((blocks, hk, bs, d // 2), **u8), v_codes=torch.zeros((blocks, hk, bs, d // 2), **u8),
                k_scales=torch.zeros((blocks, hk, bs, d // group, 2), **f16),
                v_scales=torch.zeros((blocks, hk, bs, d // group, 2), **f16))


def _prepare_write(case, gen):
    t, hk, d, bs = case["tokens"], case["kv_heads"], case["dim"], case["block"]
    kind = TYPES[case["dtype"]]
    k, v = _keys_and_values(gen, (t, hk, d), kind)
    blocks = -(-t // bs) + 5
    slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:t].to(torch.int32)
    s = _cache(blocks, hk, bs, d, case["group"])
    s.update(k=k, v=v, slots=slots, blocks=blocks, k_back=torch.empty_like(k), v_back=torch.empty_like(v))
    return s


def _prepare_attend(case, gen):
    lens, n, bs = _attend_lengths(case), case["queries"], case["block"]
    hq, hk, d, kind = case["q_heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
    pages = [-(-l // bs) for l in lens]
    width, blocks = max(pages), sum(pages) + 3
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    col, rows = torch.arange(width, device="cuda"), torch.tensor(pages, device="cuda")
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[col[None, :] < rows[:, None]] = order[: sum(pages)]
    s = {}
    for name, x in zip("kv", _keys_and_values(gen, (blocks, hk, bs, d))):
        codes, scale, offset = _quantise(x, case["group"], torch.float32)
        s[name + "_codes"], s[name + "_scales"] = _pack(codes), torch.stack((scale, offset), -1)
        del x, codes
    t = len(lens) * n
    q = _normal(gen, (t, hq, d), kind)
    s.update(q=q, table=table, kv_lens=_ints(lens), blocks=blocks, width=width, tokens=t, scale=d ** -0.5,
             query_start=_ints([i * n for i in range(len(lens) + 1)]), out=torch.empty_like(q))
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(s):
    return globals()[("_own_" if own else "_plain_") + s["case"]["op"]](s)


def _plain_slots(s):
    bs, t = s["case"]["block"], s["tokens"]
    b, width = s["table"].shape
    ctx, new = s["context_lens"].long(), s["query_lens"].long()
    have, need = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    taken = (need - have).cumsum(0)
    first = taken - (need - have)
    begin, end = s["free_range"].long().unbind(0)
    col = torch.arange(width, device="cuda")[None, :]
    at = begin + first[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    block = s["free_blocks"][at.clamp(0, s["free_blocks"].numel() - 1)]
    block = torch.where((at < end) & (block >= 0) & (block < s["blocks"]), block, torch.full_like(block, -1))
    table = torch.where(fresh, block, s["table"])
    start = torch.cat((new.new_zeros(1), new.cumsum(0)))
    token = torch.arange(t, device="cuda")
    seq = torch.searchsorted(start[1:].contiguous(), token, right=True).clamp(max=b - 1)
    real = token < start[-1]
    pos = torch.where(real, ctx[seq] + token - start[seq], torch.full_like(token, -1))
    page = table[seq, (pos.clamp(min=0) // bs).clamp(max=width - 1)].long()
    slot = torch.where(real & (page >= 0), page * bs + pos % bs, torch.full_like(token, -1))
    counts = torch.stack((start[-1], taken[-1], (real & (slot < 0)).sum(), begin + taken[-1]))
    s["table"].copy_(table)
    return [s["table"]] + [x.to(torch.int32) for x in (ctx + new, start, pos, slot, counts)]


def _turned(x, weight, cos, sin, case, eps):
    """x [tokens, heads, dim] normalised and rotated, in the type of cos."""
    y = x.to(cos.dtype)
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * weight.to(cos.dtype)
    rot, c, n = case["rot"], cos[:, None, :], sin[:, None, :]
    if case["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * c - b * n, b * c + a * n), -1).flatten(-2)
    else:
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        turned = torch.cat((a * c - b * n, b * c + a * n), -1)
    return torch.cat((turned, y[..., rot:]), -1)


def _heads(s):
    case = s["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    return (s["qkv"][:, : hq * d].unflatten(-1, (hq, d)), s["qkv"][:, hq * d: (hq + hk) * d].unflatten(-1, (hk, d)))


EPS = 1e-5


def _plain_qk(s):
    q, k = _heads(s)
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]
    return [_turned(x, w, cos, sin, s["case"], EPS).to(x.dtype) for x, w in ((q, s["q_weight"]), (k, s["k_weight"]))]


def _plain_write(s):
    group, bs = s["case"]["group"], s["case"]["block"]
    page, row = s["slots"].long() // bs, s["slots"].long() % bs
    back = []
    for name in "kv":
        codes, scale, offset = _quantise(s[name], group)
        s[name + "_codes"][page, :, row] = _pack(codes)
        s[name + "_scales"][page, :, row] = torch.stack((scale, offset), -1)
        back.append(_values(s[name + "_codes"][page, :, row], s[name + "_scales"][page, :, row], group).to(s[name].dtype))
    return back


def _attention(s, kind):
    """[batch, kv_heads, queries * heads a group, dim] in `kind`, of sequences with the same number of queries."""
    case = s["case"]
    n, hq, hk, d, group = case["queries"], case["q_heads"], case["kv_heads"], case["dim"], case["group"]
    pages = s["table"].clamp(min=0).long()
    b = pages.shape[0]
    k, v = (_values(s[x + "_codes"][pages], s[x + "_scales"][pages], group, kind).transpose(1, 2).flatten(2, 3) for x in "kv")
    q = s["q"].to(kind).view(b, n, hk, hq // hk, d).transpose(1, 2).flatten(2, 3)
    score = q @ k.transpose(-1, -2) * s["scale"]
    del k
    sees = s["kv_lens"].long()[:, None] - n + 1 + torch.arange(n, device="cuda").repeat_interleave(hq // hk)
    hidden = torch.arange(score.shape[-1], device="cuda") >= sees[:, None, :, None]
    score = score.masked_fill_(hidden, -torch.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.view(b, hk, n, hq // hk, d).transpose(1, 2).reshape(b * n, hq, d)


def _plain_attend(s):
    return _attention(s, torch.float32).to(s["q"].dtype)


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


def _handles(case, s):
    """What a program keeps for its calls: the device, the description of its cache, a workspace."""
    ops, device = _framework()
    kept = {"ops": ops, "device": device}
    if case["op"] in ("write", "attend"):
        kept["cache"] = ops.kv4_cache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], s["blocks"],
                                      case["kv_heads"], case["block"], case["dim"], case["group"])
    if case["op"] == "attend":
        size = ops.kv4_attention_workspace(device, kept["cache"], case["q_heads"])
        kept["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return kept


def _own_slots(s):
    s["ops"].paged_slots(s["device"], s["context_lens"], s["query_lens"], s["free_blocks"], s["free_range"], s["table"],
                         s["kv_lens"], s["query_start"], s["positions"], s["slots"], s["counts"], s["table"].shape[0],
                         s["table"].shape[1], s["case"]["block"], s["blocks"], s["tokens"], stream=STREAM, sync=False)
    return [s[x] for x in ("table", "kv_lens", "query_start", "positions", "slots", "counts")]


def _own_qk(s):
    case, row = s["case"], s["qkv"].shape[1]
    size = s["qkv"].element_size()
    q = s["qkv"].data_ptr()
    s["ops"].qk_norm_rope(s["device"], q, q + case["q_heads"] * case["dim"] * size, s["q_weight"], s["k_weight"],
                          s["cos"], s["sin"], s["positions"], s["q_out"], s["k_out"], case["tokens"], case["q_heads"],
                          case["kv_heads"], case["dim"], case["rot"], s["far"], EPS, case["dtype"],
                          interleaved=case["interleaved"], q_stride=row, k_stride=row, stream=STREAM, sync=False)
    return [s["q_out"], s["k_out"]]


def _own_write(s):
    case = s["case"]
    s["ops"].kv4_append(s["device"], s["cache"], s["k"], s["v"], s["slots"], case["tokens"], case["dtype"],
                        stream=STREAM, sync=False)
    s["ops"].kv4_gather(s["device"], s["cache"], s["slots"], s["k_back"], s["v_back"], case["tokens"], case["dtype"],
                        stream=STREAM, sync=False)
    return [s["k_back"], s["v_back"]]


def _own_attend(s):
    case = s["case"]
    s["ops"].kv4_attention(s["device"], s["cache"], s["q"], s["table"], s["kv_lens"], s["query_start"], s["out"],
                           s["workspace"], s["workspace"].numel(), s["tokens"], s["table"].shape[0], case["q_heads"],
                           s["width"], s["scale"], case["dtype"], stream=STREAM, sync=False)
    return s["out"]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "slots":
        return None  # whole numbers
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "qk":
        at, out = s["positions"].long(), []
        for x, w in zip(_heads(s), (s["q_weight"], s["k_weight"])):
            y = x.to(f64)
            if w is not None:
                y = y * (y.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).pow(-0.5) * w.to(f64)
            # the rotated pairs as complex numbers
            turn = torch.complex(s["cos"].to(f64)[at], s["sin"].to(f64)[at])[:, None, :]
            rot, half = case["rot"], case["rot"] // 2
            pairs = y[..., :rot].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
            pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
            turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            turned = turned if case["interleaved"] else turned.transpose(-1, -2)
            out.append(torch.cat((turned.flatten(-2), y[..., rot:]), -1))
        return out
    if case["op"] == "write":
        out = []
        for name in "kv":  # the stored scale and offset are f16 by definition, and the code goes by them
            g = s[name].to(f64).unflatten(-1, (-1, case["group"]))
            offset = g.min(-1).values.half().to(f64)[..., None]
            scale = ((g.max(-1).values - g.min(-1).values) / 15).float().half().to(f64)[..., None]
            out.append((torch.clamp(torch.round((g - offset) / scale), 0, 15) * scale + offset).flatten(-2))
        return out
    # attention, sequence by sequence, with the softmax as a log-sum
    out, n, per = [], case["queries"], case["q_heads"] // case["kv_heads"]
    for b, l in enumerate(_attend_lengths(case)):
        pages = s["table"][b, : -(-l // case["block"])].long()
        k, v = (_values(s[x + "_codes"][pages], s[x + "_scales"][pages], case["group"], f64)
                .permute(1, 0, 2, 3).flatten(1, 2)[:, :l] for x in "kv")
        q = s["q"][b * n: (b + 1) * n].to(f64).unflatten(1, (-1, per))
        score = torch.einsum("nhgd,htd->hgnt", q, k) * s["scale"]
        late = torch.arange(l, device="cuda")[None, :] > torch.arange(l - n, l, device="cuda")[:, None]
        score = score.masked_fill(late, -torch.inf)
        weight = torch.exp(score - torch.logsumexp(score, -1, keepdim=True))
        out.append(torch.einsum("hgnt,htd->nhgd", weight, v).flatten(1, 2))
    return torch.cat(out)
