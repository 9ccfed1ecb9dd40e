"""The 4-bit microscaled operators and block-sparse attention, as a program uses them, with their plain forms.

``own`` false: elementary torch operations; true: the framework's calls.  A case names its operator in ``"op"``:

quantize  x (rows, cols) -> 4-bit codes and block scales -> the values they stand for
linear    x (rows, k) times a 4-bit weight (n, k): quantise x, product, bias, SiLU, residual
select    for each query the ``topk`` key blocks of the largest score (query . mean key of the block)
attend    the selection and the attention over the selected blocks
"""
import math

import torch

own = False

BLOCK = 32  # values that share one scale
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of e2m1 codes 0..7


def _quant(name, rows, cols, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(name, rows, n, k, dtype, bias, act, res):
    return {"name": name, "op": "linear", "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias, "act": act, "res": res}


def _attn(name, op, batch, nq, nk, heads, kv_heads, dk, dv, block, topk, dtype, masked):
    return {"name": name, "op": op, "batch": batch, "nq": nq, "nk": nk, "heads": heads, "kv_heads": kv_heads, "dk": dk,
            "dv": dv, "block": block, "topk": topk, "dtype": dtype, "masked": masked}


def listed():
    return [
        # one token's activations on their way into a 4-bit layer: launch latency
        _quant("quantize one row", 1, 768, "bf16"),
        # the 160x160 map of a batch of 8 at 1280x1280, 384 channels: streaming
        _quant("quantize 160x160 map", 204800, 384, "bf16"),
        # fp32 values, columns that end inside a block
        _quant("quantize ragged fp32", 4001, 1000, "fp32"),
        # one token through a wide layer: the weight is streamed once
        _linear("linear one row", 1, 4096, 4096, "bf16", True, False, False),
        # a 1x1 conv 768 -> 768 + SiLU on the 40x40 maps of a batch of 8 at 1280x1280
        _linear("linear 40x40 maps", 12800, 768, 768, "bf16", True, True, False),
        # odd sizes in fp16 with a residual (a block's second projection)
        _linear("linear odd fp16", 401, 520, 1000, "fp16", True, False, True),
        # the largest product: matrix rate
        _linear("linear large", 16384, 4096, 4096, "bf16", True, True, True),
        # one query against a long map of keys: latency and the streaming of the keys
        _attn("select one query", "select", 1, 1, 65536, 8, 8, 64, 64, 64, 16, "bf16", False),
        # every token of an 80x80 map selects (key width 32, as the network's attention has it)
        _attn("select 80x80 map", "select", 2, 6400, 6400, 6, 6, 32, 64, 64, 8, "bf16", False),
        # one query per image over 128x128 maps of keys, padded to the largest of the batch
        _attn("attend one query", "attend", 4, 1, 16384, 8, 8, 64, 64, 64, 16, "bf16", True),
        # 40x40 maps of a batch of 8 at 1280x1280: six heads of key width 32 and value width 64, padded maps
        _attn("attend 40x40 maps", "attend", 8, 1600, 1600, 6, 6, 32, 64, 64, 8, "bf16", True),
        # the longest map, four query heads to a key head
        _attn("attend 128x128 map", "attend", 1, 16384, 16384, 8, 2, 64, 64, 64, 16, "bf16", False),
    ]


def _span(rng, lo, hi):
    """A whole number, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "select", "attend"))
    if op == "quantize":
        cols = _span(rng, 1, 8192)
        c = _quant("", _span(rng, 1, max(1, min(204800, 30_000_000 // cols))), cols, rng.choice(("bf16", "fp16", "fp32")))
    elif op == "linear":
        n, k = _span(rng, 1, 8192), _span(rng, 1, 8192)
        rows = _span(rng, 1, max(1, min(32768, int(2.5e11 / (n * k)))))
        c = _linear("", rows, n, k, rng.choice(("bf16", "fp16", "fp32")), rng.random() < 0.7, rng.random() < 0.5, rng.random() < 0.4)
    else:
        kv = rng.choice((1, 2, 3, 4, 6))
        heads = kv * rng.choice((1, 1, 1, 2, 4))
        block, topk = rng.choice((32, 64, 64, 128)), rng.choice((1, 4, 7, 8, 12, 16))
        least = 1
        if op == "select":  # alone it has something to choose from; shorter maps come with "attend"
            topk = max(topk, 4)
            least = 4 * topk * block
        if rng.random() < 0.4:  # a single query per image
            nq, nk, batch = 1, _span(rng, least, 65536), _span(rng, 1, 16)
        else:
            nk = _span(rng, least, max(least, min(16384, math.isqrt(int(1.5e9 / heads)))))
            nq = rng.choice((nk, _span(rng, 1, nk)))
            batch = _span(rng, 1, max(1, min(16, int(1.5e9 / (heads * nq * nk)))))
        dk = rng.choice((16, 32, 32, 64, 64, 80, 128))
        dv = rng.choice((32, 64, 64, 96, 128))
        c = _attn("", op, batch, nq, nk, heads, kv, dk, dv, block, topk, rng.choice(("bf16", "bf16", "fp16")), rng.random() < 0.5)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------------------- inputs
def _field(gen, batch, n, width, heads):
    """Token vectors of a map: neighbours share a part, as neighbours on an image do."""
    run = 48
    part = torch.randn(batch, (n + run - 1) // run, heads, width, generator=gen, device="cuda").repeat_interleave(run, 1)[:, :n]
    return 0.8 * part + 0.6 * torch.randn(batch, n, heads, width, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = dict(case)
    if case["op"] == "quantize":
        x = torch.nn.functional.silu(normal(case["rows"], case["cols"])) * torch.exp(normal(1, case["cols"]))
        s["x"] = x.to(dt)
    elif case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        s["x"] = (torch.nn.functional.silu(normal(rows, k)) * torch.exp(0.5 * normal(1, k))).to(dt)
        # the weight as a program keeps it: codes, two to a byte with the first in the low half, and scales
        s["codes"], s["scales"] = _pack(normal(n, k) * (1.0 / math.sqrt(k)))
        s["bias"] = (0.1 * normal(n)) if case["bias"] else None
        s["res"] = normal(rows, n).to(dt) if case["res"] else None
    else:
        b, nq, nk = case["batch"], case["nq"], case["nk"]
        s["q"] = _field(gen, b, nq, case["dk"], case["heads"]).to(dt)
        s["k"] = _field(gen, b, nk, case["dk"], case["kv_heads"]).to(dt)
        s["v"] = normal(b, nk, case["kv_heads"], case["dv"]).to(dt)
        s["mask"] = None
        if case["masked"]:  # a batch of maps padded to the largest: the last of them may be all padding
            size = torch.randint(nk // 2, nk + 1, (b,), generator=gen, device="cuda")
            size[-1] = 0 if b > 2 and seed % 2 else nk
            s["mask"] = torch.arange(nk, device="cuda")[None] < size[:, None]
    return s


# --------------------------------------------------------------------------------------------------------- plain forms
def _blocks(x):
    """(rows, cols) in 32 bits -> (rows, blocks, 32), zeros behind the last column."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    return torch.nn.functional.pad(x.float(), (0, pad)).view(rows, (cols + pad) // BLOCK, BLOCK)


def _codes(x):
    """Codes 0..15 (sign in bit 3) and scale bytes of every block."""
    v = _blocks(x)
    amax = v.abs().amax(-1)
    s = ((amax.view(torch.int32) >> 23) - 2).clamp(min=0)
    s = torch.where(torch.isfinite(v).all(-1), s, torch.full_like(s, 255))
    # 2^(127 - s) by its bits: the division by the scale is exact
    up = (((254 - s) << 23).clamp(min=0)).view(torch.float32)
    a = v.abs() * up[..., None]
    c = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return c + 8 * torch.signbit(v).int(), s


def _pack(x):
    c, s = _codes(x)
    c = c.view(c.shape[0], -1)
    return (c[:, 0::2] + 16 * c[:, 1::2]).to(torch.uint8), s.to(torch.uint8)


def _values(c, s):
    """What codes (rows, blocks, 32) and scales (rows, blocks) stand for, in 32 bits."""
    levels = torch.tensor(LEVELS, device=c.device)
    mag = levels[(c & 7).long()] * torch.where(c > 7, -1.0, 1.0)
    # 2^(s - 127) in two factors: the smallest are not normal numbers
    scale = (((s + 1) << 23).clamp(max=0x7F000000).view(torch.float32) * 0.5)
    scale = torch.where(s == 255, torch.full_like(scale, float("nan")), scale)
    return (mag * scale[..., None]).flatten(1)


def _unpack(codes, scales):
    c = codes.int()
    c = torch.stack((c & 15, c >> 4), -1).view(codes.shape[0], -1, BLOCK)
    return _values(c, scales.int())


def _plain_linear(s):
    c, sc = _codes(s["x"])
    y = _values(c, sc) @ _unpack(s["codes"], s["scales"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"]:
        y = y * (1.0 / (1.0 + torch.exp(-y)))
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["x"].dtype)


def _visible(s):
    """(batch, blocks, block) in truth values: the keys that may be read."""
    b, nk, block = s["k"].shape[0], s["k"].shape[1], s["block"]
    m = s["mask"] if s["mask"] is not None else torch.ones(b, nk, dtype=torch.bool, device=s["k"].device)
    return torch.nn.functional.pad(m, (0, -nk % block)).view(b, -1, block)


def _plain_select(s):
    """The scores in 64 bits: two blocks next to the border must not change places."""
    q, k, block, topk = s["q"].double(), s["k"].double(), s["block"], s["topk"]
    b, nq, heads, dk = q.shape
    kv = k.shape[2]
    vis = _visible(s)
    nb = vis.shape[1]
    kk = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, -k.shape[1] % block)).view(b, nb, block, kv, dk)
    kk = torch.where(vis[..., None, None], kk, torch.zeros_like(kk))
    mean = kk.sum(2) / vis.sum(2).clamp(min=1)[..., None, None]  # (b, nb, kv, dk)
    qq = q.view(b, nq, kv, heads // kv, dk).sum(3)
    score = qq.permute(0, 2, 1, 3).contiguous() @ mean.permute(0, 2, 3, 1).contiguous()  # (b, kv, nq, nb)
    can = vis.any(2)[:, None, None, :].expand_as(score)
    score = torch.where(can, score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :topk]
    order = torch.where(torch.gather(can, -1, order), order, torch.full_like(order, nb))
    order = torch.sort(order, dim=-1).values
    order = torch.nn.functional.pad(order, (0, topk - order.shape[-1]), value=nb)
    return torch.where(order == nb, torch.full_like(order, -1), order).int()


def _plain_attend(s, picked):
    q, k, v, block = s["q"].float(), s["k"].float(), s["v"].float(), s["block"]
    b, nq, heads, dk = q.shape
    nk, kv = k.shape[1], k.shape[2]
    vis = _visible(s)
    nb, g = vis.shape[1], heads // kv
    hit = torch.zeros(b, kv, nq, nb + 1, dtype=torch.bool, device=q.device)
    hit.scatter_(-1, torch.where(picked < 0, nb, picked).long(), True)
    # (b, kv, nq, nk): the keys of the picked blocks that are not masked
    see = hit[..., :nb].repeat_interleave(block, -1)[..., :nk] & vis.view(b, 1, 1, -1)[..., :nk]
    open_ = vis.view(b, -1)[:, :nk, None, None]
    k, v = torch.where(open_, k, torch.zeros_like(k)), torch.where(open_, v, torch.zeros_like(v))
    qh = q.view(b, nq, kv, g, dk).permute(0, 2, 3, 1, 4).reshape(b, kv, g * nq, dk)
    z = (qh * dk ** -0.5) @ k.permute(0, 2, 3, 1).contiguous()
    z = z.view(b, kv, g, nq, nk).masked_fill_(~see[:, :, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(b, kv, g * nq, nk) @ v.permute(0, 2, 1, 3).contiguous()
    o = o.view(b, kv, g, nq, -1) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4).reshape(b, nq, heads, -1).to(s["q"].dtype)


def run(s):
    op = s["op"]
    if own:
        import yololite_amd as ya

        if op == "quantize":
            return ya.mx4_dequantize(ya.mx4_quantize(s["x"]))
        if op == "linear":
            return ya.mx4_linear(s["x"], ya.Mx4Tensor(s["codes"], s["scales"], s["k"]), bias=s["bias"], act=s["act"], res=s["res"])
        picked = ya.block_select(s["q"], s["k"], block=s["block"], topk=s["topk"], mask=s["mask"])
        if op == "select":
            return picked
        return {"blocks": picked, "out": ya.block_attention(s["q"], s["k"], s["v"], picked, block=s["block"], mask=s["mask"])}
    if op == "quantize":
        return _values(*_codes(s["x"]))[:, : s["cols"]].to(torch.bfloat16)
    if op == "linear":
        return _plain_linear(s)
    picked = _plain_select(s)
    return picked if op == "select" else {"blocks": picked, "out": _plain_attend(s, picked)}


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        packed = rows * ((cols + BLOCK - 1) // BLOCK) * 17
        return {"bytes": rows * cols * (size + 2) + packed, "flops": 0}
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        data = rows * k * size + n * ((k + BLOCK - 1) // BLOCK) * 17 + rows * n * size * (2 if case["res"] else 1) + (4 * n if case["bias"] else 0)
        return {"bytes": data, "flops": 2 * rows * n * k}
    b, nq, nk, heads, kv, dk, dv = (case[x] for x in ("batch", "nq", "nk", "heads", "kv_heads", "dk", "dv"))
    nb = (nk + case["block"] - 1) // case["block"]
    topk = min(case["topk"], nb)
    data = 2 * b * (nq * heads * dk + nk * kv * dk) + 4 * b * kv * nq * case["topk"] + (b * nk if case["masked"] else 0)
    flops = 2 * b * kv * nq * nb * dk
    if case["op"] == "attend":
        # of the values only the selected blocks have to be read
        data += 2 * b * (kv * dv * min(nk, nq * topk * case["block"]) + nq * heads * dv)
        flops += 2 * b * nq * heads * min(nk, topk * case["block"]) * (dk + dv)
    return {"bytes": data, "flops": flops}


# -------------------------------------------------------------------------------------------------------------- exact
def _two_to(e):
    """2^e in 64 bits, by its bits: a power function may be off in the last place, and that decides ties."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_round(x):
    """The 4-bit values of x (rows, cols), in 64 bits, from the definition: scale 2^(floor(log2 amax) - 2), the nearest level,
    ties to the level of even code."""
    rows, cols = x.shape
    n = -(-cols // BLOCK)
    v = torch.zeros(rows, n * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.reshape(rows * n, BLOCK)
    amax = v.abs().max(1).values
    _, e = torch.frexp(amax)  # amax = m 2^e with 1/2 <= m < 1
    e = torch.where(amax > 0, e - 1 - 2, torch.full_like(e, -127)).clamp(min=-127)
    scale = _two_to(e)
    a = v.abs() / scale[:, None]
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    hi = torch.searchsorted(levels, a.clamp(max=6.0)).clamp(max=7)  # the first level at or over a
    lo = (hi - 1).clamp(min=0)
    up, down = levels[hi] - a.clamp(max=6.0), a.clamp(max=6.0) - levels[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    r = levels[pick] * scale[:, None] * torch.sign(v)
    return r.reshape(rows, n * BLOCK)


def _exact_weight(codes, scales, cols):
    table = torch.tensor([*LEVELS, *(-x for x in LEVELS)], dtype=torch.float64, device=codes.device)
    pairs = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    pairs[:, 0::2] = table[(codes % 16).long()]
    pairs[:, 1::2] = table[torch.div(codes, 16, rounding_mode="floor").long()]
    scale = _two_to(scales.int() - 127)
    return (pairs.reshape(*scales.shape, BLOCK) * scale[..., None]).reshape(codes.shape[0], -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_round(s["x"])[:, : case["cols"]]
    if case["op"] == "linear":
        y = torch.matmul(_exact_round(s["x"])[:, : case["k"]], _exact_weight(s["codes"], s["scales"], case["k"]).T)
        y = y + s["bias"].double() if s["bias"] is not None else y
        y = y * torch.sigmoid(y) if s["act"] else y
        return y + s["res"].double() if s["res"] is not None else y
    if case["op"] == "select":
        return None
    # attention row by row of the map, from the selection's definition: a key is seen where fewer than topk visible blocks rank before its own
    b, nq, nk, heads, kv, block = (case[x] for x in ("batch", "nq", "nk", "heads", "kv_heads", "block"))
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    nb = -(-nk // block)
    of = torch.arange(nk, device=q.device) // block
    member = torch.zeros(nb, nk, dtype=torch.float64, device=q.device)
    member[of, torch.arange(nk, device=q.device)] = 1.0
    out = torch.zeros(b, nq, heads, case["dv"], dtype=torch.float64, device=q.device)
    for i in range(b):
        ok = torch.ones(nk, dtype=torch.bool, device=q.device) if s["mask"] is None else s["mask"][i]
        if not bool(ok.any()):
            continue
        weight = member * ok
        count = weight.sum(1)
        for j in range(kv):
            mine = range(j * heads // kv, (j + 1) * heads // kv)
            centre = torch.matmul(weight, k[i, :, j]) / count.clamp(min=1.0)[:, None]
            score = torch.matmul(sum(q[i, :, h] for h in mine), centre.T)
            score[:, count == 0] = -math.inf
            rank = torch.empty(nq, nb, dtype=torch.long, device=q.device)
            place = torch.argsort(-score, dim=1, stable=True)
            rank.scatter_(1, place, torch.arange(nb, device=q.device).expand(nq, nb).contiguous())
            seen = (rank < case["topk"])[:, of] & ok
            for h in mine:
                z = torch.matmul(q[i, :, h], k[i, :, j].T) / math.sqrt(case["dk"])
                z[~seen] = -math.inf
                out[i, :, h] = torch.matmul(torch.softmax(z, 1), v[i, :, j])
    return {"blocks": None, "out": out}
